// Sequences of the 8-bit cache become other ones: in place among the beams of a group, or into another cache.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {
namespace reorder {

constexpr int MAX_BEAMS = 64;

struct Args {
  const int8_t *kc, *vc;
  const float *ks, *vs;
  int8_t *dk, *dv;
  float *dks, *dvs;
  const int *parents, *lens;
  int* new_lens;
  int L, Bs, B, F, H, C, Cd, D;  // F: sequences of a group
};

// What sequence b becomes: -1 where it stays as it is.  Parents and lengths live on the device, where the host cannot refuse them:
// a parent outside the source (of beams: outside the group) leaves the sequence as it is, a length is cut off, and both are recorded.
__device__ __forceinline__ int parent_of(const Args& a, int b, bool record) {
  const int p = a.parents[b], lo = a.dk == a.kc ? b / a.F * a.F : 0, hi = a.dk == a.kc ? lo + a.F : a.Bs;
  if (p < 0) return -1;
  if (p < lo || p >= hi) {
    if (record) atomicOr(&g_status, (unsigned int)ST_KV8_RANGE);
    return -1;
  }
  return p;
}
__device__ __forceinline__ int len_of(const Args& a, int p, bool record) {
  const int len = a.lens[p], in = min(max(len, 0), min(a.C, a.Cd));
  if (in != len && record) atomicOr(&g_status, (unsigned int)ST_KV8_RANGE);
  return in;
}

// Thread = a 16-byte column of a head, or a scale, of all sequences of a group: all are read before the first is written.
__global__ void __launch_bounds__(128) kv8_reorder_kernel(Args a) {
  griddep_wait();
  griddep_launch();
  const int h = blockIdx.y % a.H, layer = blockIdx.y / a.H, b0 = blockIdx.z * a.F;
  const int units = a.Cd * a.D / 16, blocks = a.Cd / BLK;
  const int u = blockIdx.x * 128 + threadIdx.x;
  const bool first = u == 0 && blockIdx.y == 0;
  if (first)
    for (int f = 0; f < a.F; f++) {
      const int p = parent_of(a, b0 + f, true);
      if (p >= 0) len_of(a, p, true);
      if (a.new_lens) {
        const int from = p >= 0 ? p : a.dk == a.kc ? b0 + f : -1;
        if (from >= 0) a.new_lens[b0 + f] = len_of(a, from, false);
      }
    }
  uint4 k[MAX_BEAMS], v[MAX_BEAMS];
  if (u < units) {
    for (int f = 0; f < a.F; f++) {
      const int p = parent_of(a, b0 + f, false);
      if (p < 0 || u * 16 >= len_of(a, p, false) * a.D) continue;
      const size_t at = (((size_t)layer * a.Bs + p) * a.H + h) * a.C * a.D + (size_t)u * 16;
      k[f] = *reinterpret_cast<const uint4*>(a.kc + at), v[f] = *reinterpret_cast<const uint4*>(a.vc + at);
    }
    for (int f = 0; f < a.F; f++) {
      const int p = parent_of(a, b0 + f, false);
      if (p < 0 || u * 16 >= len_of(a, p, false) * a.D) continue;
      const size_t at = (((size_t)layer * a.B + b0 + f) * a.H + h) * a.Cd * a.D + (size_t)u * 16;
      *reinterpret_cast<uint4*>(a.dk + at) = k[f], *reinterpret_cast<uint4*>(a.dv + at) = v[f];
    }
  }
  if (u < blocks) {
    for (int f = 0; f < a.F; f++) {
      const int p = parent_of(a, b0 + f, false);
      if (p < 0 || u * BLK >= len_of(a, p, false)) continue;
      const size_t at = (((size_t)layer * a.Bs + p) * a.H + h) * (a.C / BLK) + u;
      k[f].x = __float_as_uint(a.ks[at]), v[f].x = __float_as_uint(a.vs[at]);
    }
    for (int f = 0; f < a.F; f++) {
      const int p = parent_of(a, b0 + f, false);
      if (p < 0 || u * BLK >= len_of(a, p, false)) continue;
      const size_t at = (((size_t)layer * a.B + b0 + f) * a.H + h) * (a.Cd / BLK) + u;
      a.dks[at] = __uint_as_float(k[f].x), a.dvs[at] = __uint_as_float(v[f].x);
    }
  }
}

}  // namespace reorder
}  // namespace kv8
}  // namespace vt

extern "C" int vt_kv8_reorder(cudaStream_t st, int8_t* kc, int8_t* vc, float* ks, float* vs, int layers, int Bs, int C, int8_t* dst_kc,
                              int8_t* dst_vc, float* dst_ks, float* dst_vs, int dst_C, const int* parents, const int* lens, int B,
                              int beams, int H, int D, int* new_lens) {
  using namespace vt;
  using kv8::overlap;
  const char* what = "vt_kv8_reorder";
  const bool in_place = !dst_kc && !dst_vc && !dst_ks && !dst_vs;
  if (layers < 0 || B < 0 || Bs < 0) return set_error(E_SHAPE, "%s: layers=%d Bs=%d B=%d", what, layers, Bs, B);
  if ((long long)layers * Bs > 0x7fffffffLL || (long long)layers * B > 0x7fffffffLL)
    return set_error(E_SHAPE, "%s: layers * B too large", what);
  int rc = kv8::check_cache(what, kc, vc, ks, vs, layers * Bs, H, C, D);
  if (!rc && !in_place) rc = kv8::check_cache("vt_kv8_reorder (dst)", dst_kc, dst_vc, dst_ks, dst_vs, layers * B, H, dst_C, D);
  if (rc) return rc;
  if (in_place && (beams <= 0 || beams > kv8::reorder::MAX_BEAMS || B % beams || Bs != B))
    return set_error(E_SHAPE, "%s: in place needs groups of 1 .. %d beams that divide the batch (B=%d of %d, beams=%d)", what,
                     kv8::reorder::MAX_BEAMS, B, Bs, beams);
  if (layers == 0 || B == 0) return OK;
  if (!parents || !lens) return set_error(E_SHAPE, "%s: null pointer", what);
  if ((long long)layers * H > 65535 || B / (in_place ? beams : 1) > 65535)
    return set_error(E_SHAPE, "%s: layers * H = %lld or B = %d too large", what, (long long)layers * H, B);
  const long long n = (long long)layers * Bs * H, nd = (long long)layers * B * H;
  const struct { const void* p; long long n; } src[] = {{kc, n * C * D}, {vc, n * C * D}, {ks, n * C / 16}, {vs, n * C / 16}, {parents, B * 4LL}, {lens, Bs * 4LL}},
      dst[] = {{in_place ? kc : dst_kc, in_place ? n * C * D : nd * dst_C * D}, {in_place ? vc : dst_vc, in_place ? n * C * D : nd * dst_C * D},
               {in_place ? ks : dst_ks, in_place ? n * C / 16 : nd * dst_C / 16}, {in_place ? vs : dst_vs, in_place ? n * C / 16 : nd * dst_C / 16},
               {new_lens, new_lens ? B * 4LL : 0}};
  for (int x = 0; x < 6; x++)
    for (int y = 0; y < 5; y++)
      if (dst[y].n && !(in_place && x == y && x < 4) && overlap(src[x].p, src[x].n, dst[y].p, dst[y].n))
        return set_error(E_SHAPE, "%s: the destination overlaps the source", what);
  kv8::reorder::Args a{kc, vc, ks, vs, in_place ? kc : dst_kc, in_place ? vc : dst_vc, in_place ? ks : dst_ks, in_place ? vs : dst_vs,
                       parents, lens, new_lens, layers, Bs, B, in_place ? beams : 1, H, C, in_place ? C : dst_C, D};
  launch_k(kv8::reorder::kv8_reorder_kernel, dim3((a.Cd * D / 16 + 127) / 128, layers * H, B / a.F), 128, 0, st, a);
  return check_launch(what);
}
