// Sequences of the 8-bit cache become other ones: in place among the beams of a group, or into another cache.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {
namespace reorder {

constexpr int MAX_BEAMS = 64, THREADS = 128;
constexpr int STAGE = 32768, MAX_CHUNK = 16384;  // bytes of the sources that are brought in together, of one of them at most
constexpr long long kDrainCycles = 200000000LL;

struct Args {
  const int8_t *kc, *vc;
  const float *ks, *vs;
  int8_t *dk, *dv;
  float *dks, *dvs;
  const int *parents, *lens;
  int* new_lens;
  int Bs, B, slots, H, C, Cd, D;  // slots: sequences that are brought in together
  int chunk, splits;              // bytes of a sequence's codes at a time; CTAs that share an item
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

// An item is one operand (K or V codes) of one head of a layer, of the `slots` sequences that are brought in together: in place a group's
// beams, into another cache one source.  A CTA takes every splits'th chunk of an item: thread t brings the chunk of the t'th source in
// if another sequence becomes it, all wait for all of them, then the threads of the sequences that become them write it out.  The
// copies are bulk ones of up to 16 KB and take no registers; a chunk's loads run beside the stores of the one before.
// Bound: DRAM, a read of every source that moves and a write of every sequence that changes (MEASURED).
__global__ void __launch_bounds__(THREADS) kv8_reorder_kernel(Args a) {
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ __align__(8) uint64_t full[2];
  __shared__ int sh_abort, need[MAX_BEAMS];
  volatile int* abort_flag = &sh_abort;
  const int tid = threadIdx.x, slots = a.slots;
  const bool in_place = a.dk == a.kc;
  long long x = blockIdx.x;
  const int split = (int)(x % a.splits);
  x /= a.splits;
  const bool v = x & 1;
  x >>= 1;
  const int h = (int)(x % a.H);
  x /= a.H;
  const int groups = a.Bs / slots, p0 = (int)(x % groups) * slots, layer = (int)(x / groups);
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
  // the sequences that may become one of this item's sources: b_lo .., a thread each
  const int b_lo = in_place ? p0 : 0, b_n = in_place ? slots : a.B;
  const bool record = h == 0 && layer == 0 && !v && split == 0;
  for (int i = tid; i < b_n; i += THREADS) {
    const int p = parent_of(a, b_lo + i, record);
    if (p >= p0 && p < p0 + slots && !(in_place && p == b_lo + i)) need[p - p0] = 1;
    if (record && (in_place || p0 == 0)) {
      const int from = p >= 0 ? p : in_place ? b_lo + i : -1;
      const int len = from >= 0 ? len_of(a, from, true) : 0;
      if (a.new_lens && from >= 0) a.new_lens[b_lo + i] = len;
    }
  }
  __syncthreads();
  const size_t row = (size_t)a.C * a.D, drow = (size_t)a.Cd * a.D;  // bytes of a head
  const int8_t* src = (v ? a.vc : a.kc) + ((size_t)layer * a.Bs * a.H + h) * row;  // of sequence p: + p H row
  int8_t* dst = (v ? a.dv : a.dk) + ((size_t)layer * a.B * a.H + h) * drow;
  // ---- scales, by the first CTA of an item: values of a few columns of all sequences are read before the first is written
  if (split == 0) {
    const float* ss = (v ? a.vs : a.ks) + ((size_t)layer * a.Bs * a.H + h) * (a.C / BLK);
    float* ds = (v ? a.dvs : a.dks) + ((size_t)layer * a.B * a.H + h) * (a.Cd / BLK);
    const int nb = min(a.C, a.Cd) / BLK;
    if (in_place) {
      constexpr int PER = 4;
      const int cols = THREADS * PER / slots;
      for (int c0 = 0; c0 < nb; c0 += cols) {
        float val[PER];
        size_t to[PER];
#pragma unroll
        for (int k = 0; k < PER; k++) {
          const int e = tid + THREADS * k, i = e / cols, c = c0 + e % cols;
          to[k] = (size_t)-1;
          if (i >= slots || c >= nb) continue;
          const int p = parent_of(a, p0 + i, false);
          if (p < 0 || p == p0 + i || c * BLK >= len_of(a, p, false)) continue;
          val[k] = ss[(size_t)p * a.H * (a.C / BLK) + c];
          to[k] = (size_t)(p0 + i) * a.H * (a.C / BLK) + c;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; k++)
          if (to[k] != (size_t)-1) ds[to[k]] = val[k];
      }
    } else {  // shared among the sources' CTAs, whatever they bring in
      for (int b = p0; b < a.B; b += a.Bs) {
        const int p = parent_of(a, b, false);
        if (p < 0) continue;
        const int blocks = (len_of(a, p, false) + BLK - 1) / BLK;
        for (int c = tid; c < blocks; c += THREADS) ds[(size_t)b * a.H * (a.Cd / BLK) + c] = ss[(size_t)p * a.H * (a.C / BLK) + c];
      }
    }
  }
  // ---- codes
  const int mine = tid < slots && need[tid] ? len_of(a, p0 + tid, false) * a.D : 0;  // bytes of this thread's source
  int longest = 0;
  for (int i = 0; i < slots; i++) longest = max(longest, need[i] ? len_of(a, p0 + i, false) : 0);
  const int chunks = (int)(((long long)longest * a.D + a.chunk - 1) / a.chunk);
  auto load = [&](int c, int st) {
    if (tid >= slots) return;
    const int at = c * a.chunk, bytes = min(a.chunk, mine - at);
    mbar_arrive_expect_tx(&full[st], bytes > 0 ? bytes : 0);
    if (bytes > 0) bulk_load(sm + (size_t)(st * slots + tid) * a.chunk, src + (size_t)(p0 + tid) * a.H * row + at, bytes, &full[st]);
  };
  if (split < chunks) load(split, 0);
  for (int c = split, n = 0; c < chunks; c += a.splits, n++) {
    const int st = n & 1;
    if (c + a.splits < chunks) {  // the other stage: its stores have been read out
      bulk_wait_read<0>();
      __syncthreads();
      load(c + a.splits, st ^ 1);
    }
    const bool ok = mbar_wait(&full[st], (n >> 1) & 1, abort_flag, ST_KV8_WAIT);
    if (!ok) {  // copies in flight land before the CTA ends
      mbar_wait_drain(&full[st], (n >> 1) & 1, kDrainCycles);
      if (c + a.splits < chunks) mbar_wait_drain(&full[st ^ 1], ((n + 1) >> 1) & 1, kDrainCycles);
      break;
    }
    for (int i = tid; i < b_n; i += THREADS) {
      const int p = parent_of(a, b_lo + i, false);
      if (p < p0 || p >= p0 + slots || (in_place && p == b_lo + i)) continue;
      const int at = c * a.chunk, bytes = min(a.chunk, len_of(a, p, false) * a.D - at);
      if (bytes > 0) bulk_store(dst + (size_t)(b_lo + i) * a.H * drow + at, sm + (size_t)(st * slots + p - p0) * a.chunk, bytes);
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
  if ((long long)layers * H * (Bs > B ? Bs : B) > (1LL << 26) || (long long)(C > dst_C && !in_place ? C : dst_C) * D > 0x40000000LL)
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
  // items of two operands; split so that there are about eight CTAs for each SM, where the caches are long enough
  const long long items = 2LL * layers * H * (Bs / slots), chunks = (top + chunk - 1) / chunk;
  long long splits = (8LL * sm_count() + items - 1) / items;
  if (splits > chunks) splits = chunks;
  if (items * splits > 0x7fffffffLL) return set_error(E_SHAPE, "%s: grid too large (layers=%d H=%d B=%d)", what, layers, H, B);
  kv8::reorder::Args a{kc, vc, ks, vs, in_place ? kc : dst_kc, in_place ? vc : dst_vc, in_place ? ks : dst_ks, in_place ? vs : dst_vs,
                       parents, lens, new_lens, Bs, B, slots, H, C, in_place ? C : dst_C, D, chunk, (int)splits};
  const int smem = (chunks > splits ? 2 : 1) * slots * chunk;  // one stage where a CTA has one chunk
  rc = smem_attr_once((const void*)kv8::reorder::kv8_reorder_kernel, 2 * kv8::reorder::STAGE, what);
  if (rc) return rc;
  launch_k(kv8::reorder::kv8_reorder_kernel, (unsigned)(items * splits), kv8::reorder::THREADS, smem, st, a);
  return check_launch(what);
}
