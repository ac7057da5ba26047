// Attention over the 8-bit cache for sequences that share a prefix: S prefix caches, F = B / S sequences on each, every
// sequence with a cache of its own behind it.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {
namespace shared {

struct Args {
  const uint16_t* q;
  long long sq_b, sq_t, sq_h;
  const int8_t *pk, *pv;
  const float *pks, *pvs;
  int Cp, F;
  const int* plens;
  const int8_t *kc, *vc;
  const float *ks, *vs;
  int C;
  const int *lens, *counts;
  int n, G, H;
  float scale_log2;
  uint16_t* out;
  long long so_b, so_t, so_h;
};

__device__ __forceinline__ int prefix_len(const int* plens, int s, int Cp, bool record) {
  const int len = plens[s], in = min(max(len, 0), Cp);
  if (in != len && record) atomicOr(&g_status, (unsigned int)ST_KV8_RANGE);
  return in;
}

// One row (b, i, query head) a CTA: 128 keys at a time, thread = key for the scores, thread = dim for the sum.
template <int D>
__global__ void __launch_bounds__(128) attn_kv8_shared_kernel(Args a) {
  __shared__ float sh_q[D], sh_p[128], red[4];
  const int tid = threadIdx.x, hq = blockIdx.x, i = blockIdx.y, b = blockIdx.z, h = hq / a.G;
  griddep_wait();
  griddep_launch();
  const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C);
  const int P = prefix_len(a.plens, b / a.F, a.Cp, tid == 0);
  if (i >= s.cnt) return;
  if (tid < D) sh_q[tid] = bf2f(a.q[b * a.sq_b + i * a.sq_t + hq * a.sq_h + tid]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int part = 0; part < 2; part++) {
    const size_t bh = (size_t)(part ? b : b / a.F) * a.H + h;
    const int T = part ? s.len + i + 1 : P, C = part ? a.C : a.Cp;
    const int8_t *k = (part ? a.kc : a.pk) + bh * C * D, *v = (part ? a.vc : a.pv) + bh * C * D;
    const float *ks = (part ? a.ks : a.pks) + bh * (C / BLK), *vs = (part ? a.vs : a.pvs) + bh * (C / BLK);
    for (int j0 = 0; j0 < T; j0 += 128) {
      const int j = j0 + tid;
      float z = -INFINITY;
      if (j < T) {
        float dot = 0.f;
        for (int d = 0; d < D; d++) dot += sh_q[d] * k[(size_t)j * D + d];
        z = dot * (ks[j / BLK] * a.scale_log2);
      }
      float top = z;
      for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      if (tid % 32 == 0) red[tid / 32] = top;
      __syncthreads();
      top = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
      const float alpha = exp2f(m - top), p = exp2f(z - top);
      m = top;
      sh_p[tid] = j < T ? p * vs[j / BLK] : 0.f;
      float sum = p;
      for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      __syncthreads();
      if (tid % 32 == 0) red[tid / 32] = sum;
      __syncthreads();
      l = l * alpha + (red[0] + red[1] + red[2] + red[3]);
      if (tid < D) {
        o *= alpha;
        for (int x = 0; x < min(128, T - j0); x++) o += sh_p[x] * v[(size_t)(j0 + x) * D + tid];
      }
      __syncthreads();
    }
  }
  if (tid < D) a.out[b * a.so_b + i * a.so_t + hq * a.so_h + tid] = f2bf(o / l);
}

}  // namespace shared
}  // namespace kv8
}  // namespace vt

extern "C" {

long long vt_attn_kv8_shared_ws_bytes(int S, int B, int n, int Hq, int H, int D, int Cp, int C) {
  if (S <= 0 || B <= 0 || B % S || n <= 0 || Hq <= 0 || H <= 0 || Hq % H || Cp <= 0 || C <= 0 || (D != 64 && D != 128)) return 0;
  return 0;
}

int vt_attn_kv8_shared(cudaStream_t st, const uint16_t* q, long long sq_b, long long sq_t, long long sq_h, const int8_t* pk,
                       const int8_t* pv, const float* pks, const float* pvs, int Cp, const int* plens, int S, const int8_t* kc,
                       const int8_t* vc, const float* ks, const float* vs, int C, const int* lens, const int* counts, int B,
                       int n, int Hq, int H, int D, float scale, uint16_t* out, long long so_b, long long so_t, long long so_h,
                       void* ws, long long ws_bytes) {
  using namespace vt;
  const char* what = "vt_attn_kv8_shared";
  int rc = kv8::check_cache("vt_attn_kv8_shared (prefix)", pk, pv, pks, pvs, S, H, Cp, D);
  if (!rc) rc = kv8::check_cache(what, kc, vc, ks, vs, B, H, C, D);
  if (rc) return rc;
  if (n < 0 || Hq <= 0 || Hq % H) return set_error(E_SHAPE, "%s: n=%d Hq=%d H=%d (Hq a multiple of H)", what, n, Hq, H);
  if (B == 0 || n == 0) return OK;
  if (S == 0 || B % S) return set_error(E_SHAPE, "%s: %d sequences over %d prefixes (a multiple of them)", what, B, S);
  if (!q || !lens || !plens || !out || !aligned16(q) || !aligned16(out) || (sq_b | sq_t | sq_h | so_b | so_t | so_h) % 8)
    return set_error(E_SHAPE, "%s: null pointer, or pointers / strides not 16-byte aligned", what);
  if (!(scale >= 0.f && scale < 0x1p100f)) return set_error(E_SHAPE, "%s: scale %g is not 0 .. 2^100", what, scale);
  const long long need = vt_attn_kv8_shared_ws_bytes(S, B, n, Hq, H, D, Cp, C);
  if (need && (!ws || !aligned16(ws) || ws_bytes < need))
    return set_error(E_SHAPE, "%s: workspace of %lld bytes, %lld needed (16-byte aligned)", what, ws ? ws_bytes : 0LL, need);
  if (B > 2048 || n > 65535) return set_error(E_SHAPE, "%s: B=%d (at most 2048) or n=%d too large", what, B, n);
  if (kv8::rows_meet({q, sq_b, sq_t, (Hq - 1) * sq_h + D}, {out, so_b, so_t, (Hq - 1) * so_h + D}, B, n))
    return set_error(E_SHAPE, "%s: out overlaps q", what);
  kv8::shared::Args a{q, sq_b, sq_t, sq_h, pk, pv, pks, pvs, Cp, B / S, plens, kc, vc, ks, vs, C, lens, counts,
                      n, Hq / H, H, scale * kv8::LOG2E, out, so_b, so_t, so_h};
  if (D == 64) launch_k(kv8::shared::attn_kv8_shared_kernel<64>, dim3(Hq, n, B), 128, 0, st, a);
  else launch_k(kv8::shared::attn_kv8_shared_kernel<128>, dim3(Hq, n, B), 128, 0, st, a);
  return check_launch(what);
}

}  // extern "C"
