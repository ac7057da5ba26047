// Sequences of the 8-bit cache become other ones: in place among the beams of a group, or into another cache.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {
namespace reorder {

constexpr int MAX_BEAMS = 64, THREADS = 128;
// Bytes of the sources that are brought in together, of one of them at most.  Of the three calls that are named at the kernel (a served batch's
// beams, a fork, few beams): 16 KB and 8 KB 286, 94, 6.7 us; 8 and 8 KB 286, 93, 8.8; 32 and 16 KB 294, 103, 8.4.
constexpr int STAGE = 16384, MAX_CHUNK = 8192;
constexpr long long kDrainCycles = 200000000LL;

struct Args {
  const int8_t *kc, *vc;
  const float *ks, *vs;
  int8_t *dk, *dv;
  float *dks, *dvs;
  const int *parents, *lens;
  int* new_lens;
  int layers, Bs, B, slots, H, C, Cd, D;  // slots: sequences that are brought in together
  int chunk, ctas;                        // bytes of a sequence's codes at a time; CTAs of a group
};

// What sequence b becomes: -1 where it stays as it is.  Parents and lengths live on the device, where the host cannot refuse them:
// a parent outside the source (of beams: outside the group) leaves the sequence as it is, a length is cut off, and both are recorded.
__device__ __forceinline__ int parent_of(const Args& a, int b, bool record) {
  const int p = a.parents[b], lo = a.dk == a.kc ? b / a.slots * a.slots : 0, hi = a.dk == a.kc ? lo + a.slots : a.Bs;
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

// The sequences that are brought in together are a group: in place its beams, into another cache one source.  A unit is a chunk of the
// codes of one operand (K or V) of one head of a layer, of all sequences of a group; a group's CTAs take its units in turn.  Thread t
// brings in the chunk of the t'th source, if another sequence becomes it; all wait for all of them, then the threads of the sequences
// that become them write it out.  The copies are bulk ones of up to 16 KB, take no registers, and the next unit's loads run beside the
// stores of this one.
// Bound: DRAM, a read of every source that moves and a write of every sequence that changes (24 layers x 8 groups of 8 beams, 32 heads x 64 dims,
// 125 to 250 tokens, 1.76 GB: 286 us, 6.2 TB/s; 64 sequences out of 16 of 2,050 to 4,099 tokens, 8 heads x 128, 515 MB: 94 us, 5.5 TB/s).  Few
// beams of few tokens: latency of the parents, the lengths, one copy in and one out (24 layers x 4 beams of 38 tokens: 6.7 us).
__global__ void __launch_bounds__(THREADS) kv8_reorder_kernel(Args a) {
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ __align__(8) uint64_t full[2];
  __shared__ int sh_abort, need[MAX_BEAMS];
  volatile int* abort_flag = &sh_abort;
  const int tid = threadIdx.x, slots = a.slots;
  const bool in_place = a.dk == a.kc;
  const int p0 = blockIdx.x / a.ctas * slots, cta = blockIdx.x % a.ctas;
  if (tid == 0) {
    mbar_init(&full[0], slots);
    mbar_init(&full[1], slots);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (tid < MAX_BEAMS) need[tid] = 0;
  griddep_wait();
  griddep_launch();
  __syncthreads();
  // the sequences that may become one of the group's sources: b_lo .., a thread each
  const int b_lo = in_place ? p0 : 0, b_n = in_place ? slots : a.B;
  for (int i = tid; i < b_n; i += THREADS) {
    const int p = parent_of(a, b_lo + i, cta == 0);
    const bool moves = p >= p0 && p < p0 + slots && !(in_place && p == b_lo + i);
    const int from = p >= 0 ? p : b_lo + i;
    const bool mine = cta == 0 && (in_place || (p0 == 0 && p >= 0));  // lengths are looked at once
    if (moves || mine) {
      const int len = len_of(a, from, mine);
      if (moves) need[p - p0] = len;
      if (mine && a.new_lens) a.new_lens[b_lo + i] = len;
    }
  }
  __syncthreads();
  int longest = 0;
  for (int i = 0; i < slots; i++) longest = max(longest, need[i]);
  const int chunks = (int)(((long long)longest * a.D + a.chunk - 1) / a.chunk);
  const long long units = 2LL * a.layers * a.H * chunks;  // chunk by chunk, K and V, head by head, layer by layer
  const size_t row = (size_t)a.C * a.D, drow = (size_t)a.Cd * a.D;  // bytes of a head
  const int mine = tid < slots ? need[tid] * a.D : 0;               // bytes of this thread's source
  auto load = [&](long long u, int st) {
    if (tid >= slots) return;
    const int at = (int)(u % chunks) * a.chunk, bytes = min(a.chunk, mine - at);
    const long long x = u / chunks, lh = x >> 1;
    mbar_arrive_expect_tx(&full[st], bytes > 0 ? bytes : 0);
    if (bytes > 0)
      bulk_load(sm + (size_t)(st * slots + tid) * a.chunk,
                (x & 1 ? a.vc : a.kc) + ((lh / a.H * a.Bs + p0 + tid) * a.H + lh % a.H) * row + at, bytes, &full[st]);
  };
  if (cta < units) load(cta, 0);
  // ---- scales, while the first unit arrives
  const int heads2 = 2 * a.layers * a.H, sb = a.C / BLK, db = a.Cd / BLK;
  auto scale_at = [&](int x, int B, int b, int blocks) { return ((size_t)(x >> 1) / a.H * B + b) * a.H * blocks + (size_t)((x >> 1) % a.H) * blocks; };
  if (in_place) {  // columns of one block of all sequences: they are read before the first of them is written
    constexpr int PER = 4;
    const int nb = (longest + BLK - 1) / BLK, cols = THREADS * PER / slots;
    const long long all = (long long)heads2 * nb;
    for (long long c0 = (long long)cta * cols; c0 < all; c0 += (long long)a.ctas * cols) {
      float val[PER];
      float* to[PER];
#pragma unroll
      for (int k = 0; k < PER; k++) {
        const int e = tid + THREADS * k, i = e / cols;
        const long long c = c0 + e % cols;
        to[k] = nullptr;
        if (i >= slots || c >= all) continue;
        const int p = parent_of(a, p0 + i, false), x = (int)(c / nb), blk = (int)(c % nb);
        if (p < 0 || p == p0 + i || blk * BLK >= need[p - p0]) continue;
        val[k] = (x & 1 ? a.vs : a.ks)[scale_at(x, a.Bs, p, sb) + blk];
        to[k] = (x & 1 ? a.dvs : a.dks) + scale_at(x, a.B, p0 + i, db) + blk;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < PER; k++)
        if (to[k]) *to[k] = val[k];
    }
  } else {  // the sequences are dealt out to the groups, whatever they become
    for (int b = p0; b < a.B; b += a.Bs) {
      const int p = parent_of(a, b, false);
      if (p < 0) continue;
      const int nb = (len_of(a, p, false) + BLK - 1) / BLK;
      const long long all = (long long)heads2 * nb;
      for (long long e = (long long)cta * THREADS + tid; e < all; e += (long long)a.ctas * THREADS) {
        const int x = (int)(e / nb), blk = (int)(e % nb);
        (x & 1 ? a.dvs : a.dks)[scale_at(x, a.B, b, db) + blk] = (x & 1 ? a.vs : a.ks)[scale_at(x, a.Bs, p, sb) + blk];
      }
    }
  }
  // ---- codes
  int n = 0;
  for (long long u = cta; u < units; u += a.ctas, n++) {
    const int st = n & 1;
    if (u + a.ctas < units) {  // the other stage: its stores have been read out
      bulk_wait_read<0>();
      __syncthreads();
      load(u + a.ctas, st ^ 1);
    }
    const bool ok = mbar_wait(&full[st], (n >> 1) & 1, abort_flag, ST_KV8_WAIT);
    if (!ok) {  // copies in flight land before the CTA ends
      mbar_wait_drain(&full[st], (n >> 1) & 1, kDrainCycles);
      if (u + a.ctas < units) mbar_wait_drain(&full[st ^ 1], ((n + 1) >> 1) & 1, kDrainCycles);
      break;
    }
    const int at = (int)(u % chunks) * a.chunk;
    const long long x = u / chunks, lh = x >> 1;
    for (int i = tid; i < b_n; i += THREADS) {
      const int p = parent_of(a, b_lo + i, false);
      if (p < p0 || p >= p0 + slots || (in_place && p == b_lo + i)) continue;
      const int bytes = min(a.chunk, need[p - p0] * a.D - at);
      if (bytes > 0)
        bulk_store((x & 1 ? a.dv : a.dk) + ((lh / a.H * a.B + b_lo + i) * a.H + lh % a.H) * drow + at,
                   sm + (size_t)(st * slots + p - p0) * a.chunk, bytes);
    }
    bulk_commit();
  }
  bulk_wait_all<0>();
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
  if (Bs == 0) return set_error(E_SHAPE, "%s: no sequence to take", what);
  if (!parents || !lens) return set_error(E_SHAPE, "%s: null pointer", what);
  if ((long long)layers * H * (Bs > B ? Bs : B) > (1LL << 26) || (long long)(in_place || C > dst_C ? C : dst_C) * D > 0x40000000LL)
    return set_error(E_SHAPE, "%s: layers * B * H or C too large", what);
  const long long n = (long long)layers * Bs * H, nd = (long long)layers * B * H;
  const struct { const void* p; long long n; } src[] = {{kc, n * C * D}, {vc, n * C * D}, {ks, n * C / 16}, {vs, n * C / 16}, {parents, B * 4LL}, {lens, Bs * 4LL}},
      dst[] = {{in_place ? kc : dst_kc, in_place ? n * C * D : nd * dst_C * D}, {in_place ? vc : dst_vc, in_place ? n * C * D : nd * dst_C * D},
               {in_place ? ks : dst_ks, in_place ? n * C / 16 : nd * dst_C / 16}, {in_place ? vs : dst_vs, in_place ? n * C / 16 : nd * dst_C / 16},
               {new_lens, new_lens ? B * 4LL : 0}};
  for (int x = 0; x < 6; x++)
    for (int y = 0; y < 5; y++)
      if (dst[y].n && !(in_place && x == y && x < 4) && overlap(src[x].p, src[x].n, dst[y].p, dst[y].n))
        return set_error(E_SHAPE, "%s: the destination overlaps the source", what);
  const int slots = in_place ? beams : 1, top = (in_place || C < dst_C ? C : dst_C) * D;  // bytes of a head that may move
  int chunk = kv8::reorder::STAGE / slots / 128 * 128;
  if (chunk > kv8::reorder::MAX_CHUNK) chunk = kv8::reorder::MAX_CHUNK;
  if (chunk > top) chunk = top;
  // CTAs for every SM to hold as many as fit, or several times as many where each still has many units (lengths may differ)
  const long long groups = Bs / slots, units = 2LL * layers * H * ((top + chunk - 1) / chunk);
  const int fit = 225 * 1024 / (2 * slots * chunk + 2048), per_sm = fit > 16 ? 16 : fit;
  const long long one = (long long)per_sm * sm_count(), want = units * groups > 16 * one ? 4 * one : one;
  long long ctas = (want + groups - 1) / groups;
  if (ctas > units) ctas = units;
  if (groups * ctas > 0x7fffffffLL) return set_error(E_SHAPE, "%s: grid too large (B=%d)", what, B);
  kv8::reorder::Args a{kc, vc, ks, vs, in_place ? kc : dst_kc, in_place ? vc : dst_vc, in_place ? ks : dst_ks, in_place ? vs : dst_vs,
                       parents, lens, new_lens, layers, Bs, B, slots, H, C, in_place ? C : dst_C, D, chunk, (int)ctas};
  const int smem = (units > ctas ? 2 : 1) * slots * chunk;  // one stage where a CTA has one unit
  rc = smem_attr_once((const void*)kv8::reorder::kv8_reorder_kernel, 2 * kv8::reorder::STAGE, what);
  if (rc) return rc;
  launch_k(kv8::reorder::kv8_reorder_kernel, (unsigned)(groups * ctas), kv8::reorder::THREADS, smem, st, a);
  return check_launch(what);
}
