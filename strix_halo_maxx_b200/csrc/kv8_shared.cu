// Attention over the 8-bit cache for sequences that share a prefix: S prefix caches, F = B / S sequences on each, every sequence
// with a cache of its own behind it.  A prefix is read once for the rows of all of its sequences.
//
//   few rows on a prefix   F n G <= 32 (16 where heads are 128 wide): one item per head with the prefix's tiles and all own ones (kv8_split.cu)
//   more                   attn_kv8_shared_tc_kernel below.  Where each sequence's own slots are few beside the prefix, or its rows
//                          many, it takes them too; else it takes the prefix alone and leaves each row's output, maximum and sum, and
//                          kv8_split.cu adds the own slots, whose reading then is what costs
//
// The kernel is the one of kv8_tc.cu (its comment says how codes, scales and P are held, and what bounds a tile) with other lists.  A head's
// rows over prefix s are r = t G + g, t numbering the new tokens of all of its sequences without gaps: idle and short sequences cost
// nothing.  An item is ROWS of them; its tiles of 64 keys are the prefix's, then those of each sequence that has rows in it, in order.
//   two M tiles of 128 rows  share every converted tile; own tiles that concern the rows of one M tile are passed over by the other;
//   ALT, up to 128 rows      both M tiles hold the same rows and take the key tiles in turn, so that two are in flight all the same; in
//                            the end each pair of threads puts its row's two halves together.
// 8 x 256 tokens (some fewer), 32/8 heads x 128, over 6,001 + 511 slots, 202 GFLOP: 294 us, 688 TFLOP/s, a tile in 1.6 us; 16 x 1 over
// 131,007 + 65, 271 MB: 136 us, two tiles in 1.8 us.  What bounds a tile is the chain of its scores through TMEM, exponentials and P, about
// 1,400 cycles of a thread's issue and latencies, beside the operands' way through shared memory: without converting anything these two take
// 255 and 111 us; exponentials by a polynomial on the FMA pipe instead of the MUFU, for a fifth of them, 305 and 144.  A call of few tiles:
// launch, lists and shares (3.5 us), the first codes and q (2 to 4), the first tile's cold instructions (2 to 4).
// Items' tiles form one list cut into equal runs, one for each SM; what spans CTAs leaves parts for attn_kv8_shared_join_kernel.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {
namespace shared {

using tc::KEYS;
using tc::kDrainCycles;
using tc::kTinyScale;
using tc::L_LOG2;
using tc::L_SCALE;
using tc::P_MOVE;
using tc::P_TOP;
using tc::P_UP;
using tc::P_UP_SINK;
using tc::THREADS;
using tc::Z_TOP;
constexpr int MAXB = 2048, MAX_CTAS = 512;  // sequences and runs (one for each SM) of a call
constexpr float SINK_SUM = 238.856f;   // 2^P_UP: what the largest term of a row's first tile is
constexpr uint32_t TMEM_COLS = 512;  // S of M tile t, buffer f: columns 128 t + 64 f; O of tile t: 256 + 128 t

template <int D, bool ALT>
struct Smem {
  static constexpr int ROWS = ALT ? 128 : 256, ST = ALT ? 4 : 3;
  static constexpr int QT = 128 * D * 2;   // bytes of one M tile of q
  static constexpr int KT = KEYS * D * 2;  // of a converted K or V tile
  static constexpr int K = (ALT ? 1 : 2) * QT, V = K + ST * KT, RAW = V + ST * KT;
  static constexpr int RAW_TILE = 2 * KEYS * D;  // bytes of a tile's codes, K and V
  static constexpr int BUDGET = (ALT ? 217 : 221) * 1024;  // with the lists behind them, and beside the static arrays
};
constexpr int MAX_RAW = 6;  // tiles of codes in flight
__host__ __device__ inline int list_bytes(int S, int B) { return (3 * B + 2 * S + 3) * 4; }

struct Args {
  const uint16_t* q;
  long long sq_b, sq_t, sq_h;
  const int8_t *pk, *pv;
  const float *pks, *pvs;
  int Cp, S, F;
  const int* plens;
  const int8_t *kc, *vc;
  const float *ks, *vs;
  int C;
  const int *lens, *counts;
  int n, G, H, ctas;
  int items;  // > 0: items of a head, and a CTA for each item (no runs, nothing to join)
  int own;    // whether the sequences' own slots are in the lists
  int raw;    // tiles of codes in flight
  float scale_log2;
  uint16_t* out;
  long long so_b, so_t, so_h;
  float* row_o;      // [B][n][Hq][D] and [B][n][Hq]: where rows go without own slots
  float2* row_ml;
  float* part_o;     // [2 ctas][ROWS][D]
  float2* part_ml;   // [2 ctas][ROWS]
  int4* unfinished;  // [ctas] the item that a CTA begins and others go on with: last CTA (-1: none), slot of the first part, head, first row
  int* row_at;       // [ctas][ROWS] where that item's rows are: b n + i, -1 for none
};

// What every CTA works out for itself.
struct Lists {
  int *tok, *len;  // new tokens before each sequence, [B + 1]; tokens that it held before the call
  int *own, *pre;  // own tiles of the items before each sequence's, [B + 1]; tiles before each prefix's heads, [S + 1]
  int* plen;       // tokens of each prefix
};
__device__ __forceinline__ int seq_of_token(const Args& a, const Lists& l, int s, int t) {  // t: of the prefix's sequences
  return s * a.F + split::find_seq(l.tok + s * a.F, a.F, l.tok[s * a.F] + t);
}
// Own tiles that rows [q ROWS, q ROWS + ROWS) of its prefix need of sequence x, which has rows among them or none at all.
template <int ROWS>
__device__ __forceinline__ int own_tiles(const Args& a, const Lists& l, int s, int x, int q) {
  const int cnt = l.tok[x + 1] - l.tok[x];
  if (!a.own || cnt == 0) return 0;
  const int last = min(cnt - 1, (q * ROWS + ROWS - 1) / a.G - (l.tok[x] - l.tok[s * a.F]));
  return (l.len[x] + last + KEYS) / KEYS;
}
// list[0 .. n] becomes the sums before each of n numbers, count(i) gives them: a warp, 32 at a time.
template <typename Count>
__device__ __forceinline__ void warp_sums(int* list, int n, const Count& count) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int x = i0 + lane < n ? count(i0 + lane) : 0;
    int inc = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    if (i0 + lane < n) list[i0 + lane] = before + inc - x;
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) list[n] = before;
  __syncwarp();
}
// By one warp (block-wide sums took 2 us with their barriers).
template <int ROWS>
__device__ __forceinline__ void make_lists(const Args& a, const Lists& l) {
  const bool record = blockIdx.x == 0;
  const int lane = threadIdx.x & 31, B = a.S * a.F;
  for (int s = lane; s < a.S; s += 32) l.plen[s] = split::prefix_len(a.plens, s, a.Cp, record);
  for (int i0 = 0; i0 < B; i0 += 128) {  // the loads of four at a time side by side
    int len[4], cnt[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int b = i0 + 32 * k + lane;
      len[k] = b < B ? a.lens[b] : 0, cnt[k] = b < B && a.counts ? a.counts[b] : a.n;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int b = i0 + 32 * k + lane;
      if (b >= B) continue;
      const Seq q = clip_seq(len[k], cnt[k], a.n, a.C, record);
      l.len[b] = q.len, l.tok[b] = q.cnt;
    }
  }
  __syncwarp();
  warp_sums(l.tok, B, [&](int b) { return l.tok[b]; });
  if (a.own)
    warp_sums(l.own, B, [&](int x) {
      const int s = x / a.F, first = (l.tok[x] - l.tok[s * a.F]) * a.G, rows = (l.tok[x + 1] - l.tok[x]) * a.G;
      int t = 0;
      if (rows)
        for (int q = first / ROWS; q <= (first + rows - 1) / ROWS; q++) t += own_tiles<ROWS>(a, l, s, x, q);
      return t;
    });
  warp_sums(l.pre, a.S, [&](int s) {
    const int P = l.plen[s], rows = (l.tok[(s + 1) * a.F] - l.tok[s * a.F]) * a.G;
    return ((rows + ROWS - 1) / ROWS * ((P + KEYS - 1) / KEYS) + (a.own ? l.own[(s + 1) * a.F] - l.own[s * a.F] : 0)) * a.H;
  });
}

// A CTA's share of an item: rows q ROWS .. of prefix s, head h; key tiles [ta, tb) of `tiles`, the first pt of them the prefix's.
struct Seg {
  int s, h, q, rows, P, pt, x0, x1, t0, tiles, ta, tb;  // x0, x1: first and last sequence of the item; t0: own tiles of x0
  int last;                                             // the CTA with the item's last tile
  struct Part {
    int oa, ob;  // own tiles that concern the M tile: [oa, ob) of the item's
    bool act;    // whether it has any tile here
  } m0, m1;
  __device__ __forceinline__ Part of(int t) const { return t ? m1 : m0; }
};
// Own tiles of an item before those of sequence x.
__device__ __forceinline__ int own_before(const Args& a, const Lists& l, int x0, int t0, int x) {
  return !a.own || x == x0 ? 0 : t0 + l.own[x] - l.own[x0 + 1];
}
// Tiles of items 0 .. q - 1 of a head.
template <int ROWS>
__device__ __forceinline__ int tiles_before(const Args& a, const Lists& l, int s, int q, int pt) {
  if (q == 0) return 0;
  int t = q * pt;
  if (a.own) {
    const int x = seq_of_token(a, l, s, q * ROWS / a.G), first = (l.tok[x] - l.tok[s * a.F]) * a.G;
    t += l.own[x] - l.own[s * a.F];
    for (int i = first / ROWS; i < q; i++) t += own_tiles<ROWS>(a, l, s, x, i);
  }
  return t;
}
// The largest i < n with value(i) <= u (value(0) is), and its value: the whole warp looks at 32 places at a time.
template <typename Value>
__device__ __forceinline__ int warp_search(int n, int u, int& found, const Value& value) {
  const int lane = threadIdx.x & 31;
  int lo = 0;
  found = 0;
  while (n > 0) {
    const int step = (n + 31) / 32;
    const int v = lane * step < n ? value(lo + lane * step) : 0x7fffffff;
    const int k = 31 - __clz(__ballot_sync(0xffffffffu, v <= u) | 1u);
    found = __shfl_sync(0xffffffffu, v, k);
    lo += k * step, n = step > 1 ? min(step, n - k * step) : 0;
  }
  return lo;
}
// The share that begins at place u of the list (of whole items: this CTA's), worked out by a warp.
template <int D, bool ALT>
__device__ __forceinline__ Seg segment(const Args& a, const Lists& l, int u, int u_end) {
  constexpr int ROWS = Smem<D, ALT>::ROWS;
  const int lane = threadIdx.x & 31;
  Seg g;
  int at = 0;
  if (a.items > 0) {
    const int sh = blockIdx.x / a.items;
    g.s = sh / a.H, g.h = sh % a.H, g.q = blockIdx.x % a.items;
  } else {
    int before = 0;
    g.s = a.S > 1 ? warp_search(a.S, u, before, [&](int s) { return l.pre[s]; }) : 0;
    const int head = (l.pre[g.s + 1] - l.pre[g.s]) / a.H;
    g.h = (u - before) / head, at = (u - before) % head;
  }
  g.rows = (l.tok[(g.s + 1) * a.F] - l.tok[g.s * a.F]) * a.G;
  g.P = l.plen[g.s];
  g.pt = (g.P + KEYS - 1) / KEYS;
  if (a.items == 0) {  // the last item that begins at `at` or before
    int before = 0;
    g.q = warp_search((g.rows + ROWS - 1) / ROWS, at, before, [&](int q) { return tiles_before<ROWS>(a, l, g.s, q, g.pt); });
    at -= before;
  }
  const int r0 = g.q * ROWS;
  g.tiles = 0, g.ta = at, g.x0 = g.x1 = g.t0 = 0;
  int oa1 = 0, ob0 = 0;
  if (r0 < g.rows) {
    // lanes 0 .. 3: the first row of the item, the last one of M tile 0, the first one of M tile 1, the last one of the item
    const int row = min(lane == 0 ? r0 : lane == 1 ? r0 + 127 : lane == 2 ? r0 + 128 : r0 + ROWS - 1, g.rows - 1);
    const int x = seq_of_token(a, l, g.s, row / a.G), own = own_tiles<ROWS>(a, l, g.s, x, g.q);
    g.x0 = __shfl_sync(0xffffffffu, x, 0), g.t0 = __shfl_sync(0xffffffffu, own, 0), g.x1 = __shfl_sync(0xffffffffu, x, 3);
    const int from = g.pt + own_before(a, l, g.x0, g.t0, x), to = from + own;
    ob0 = __shfl_sync(0xffffffffu, to, 1), oa1 = __shfl_sync(0xffffffffu, from, 2), g.tiles = __shfl_sync(0xffffffffu, to, 3);
  }
  g.tb = a.items > 0 ? g.tiles : min(g.tiles, g.ta + (u_end - u));
  const int nt = g.tb - g.ta;
  auto part = [&](int t, int oa, int ob) {
    if (ALT) return Seg::Part{g.pt, g.tiles, nt >= 2 || (nt == 1 && (g.ta & 1) == t)};
    return Seg::Part{oa, ob, nt > 0 && r0 + 128 * t < g.rows && (g.ta < g.pt || max(g.ta, oa) < min(g.tb, ob))};
  };
  g.m0 = part(0, g.pt, ob0), g.m1 = part(1, oa1, g.tiles);
  return g;
}
// The first tile from j on that M tile t takes part in; tb where there is none.
template <bool ALT>
__device__ __forceinline__ int tile_from(const Seg& g, int t, int j) {
  if (ALT) return min(j + ((j ^ t) & 1), g.tb);
  const Seg::Part p = g.of(t);
  if (j >= g.pt) j = max(j, p.oa);
  return j >= g.tb || (j >= g.pt && j >= p.ob) ? g.tb : j;
}

// Where tile j of an item lies: sequence x (-1: the prefix) and block kt of its cache, of n that the item needs.
struct Cursor {
  int x, kt, n;
};
template <int ROWS>
__device__ __forceinline__ Cursor cursor_at(const Args& a, const Lists& l, const Seg& g, int j) {
  if (j < g.pt) return {-1, j, g.pt};
  int lo = g.x0, hi = g.x1 + 1;  // the last sequence whose tiles begin at j or before
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (own_before(a, l, g.x0, g.t0, mid) <= j - g.pt) lo = mid; else hi = mid;
  }
  return {lo, j - g.pt - own_before(a, l, g.x0, g.t0, lo), own_tiles<ROWS>(a, l, g.s, lo, g.q)};
}
template <int ROWS>
__device__ __forceinline__ void advance(const Args& a, const Lists& l, const Seg& g, Cursor& c) {  // there is a next tile
  if (++c.kt < c.n) return;
  c.x = c.x < 0 ? g.x0 : c.x + 1, c.kt = 0;
  while ((c.n = own_tiles<ROWS>(a, l, g.s, c.x, g.q)) == 0) c.x++;
}
// Of the tile's cache: block number among all of its heads and sequences.
__device__ __forceinline__ size_t block_of(const Args& a, const Seg& g, const Cursor& c) {
  return c.x < 0 ? ((size_t)g.s * a.H + g.h) * (a.Cp / BLK) + c.kt : ((size_t)c.x * a.H + g.h) * (a.C / BLK) + c.kt;
}

// A tile as its consumers need it: whose slots (x, -1: the prefix's) from which key on, K's scale times the softmax scale, log2 and inverse
// (times L_SCALE) of V's scale (the approximations err by 2^-22, both in the sum and in O), and how far terms may be above m.
struct Tile {
  int x, key0;
  float c, lvs, ivs, top;
};

// Warps 0-3, 4-7: softmax of M tile 0 / 1, thread = row; 8-11: codes -> operands; 12, 13: MMAs of M tile 0 / 1; 15: works out the CTA's
// shares of items, for all (each warp for itself took 6 us before the first tile); 14: brings in codes and scales,
// `raw` tiles ahead (without that stage, from memory into the converters' registers, the 8 x 256 tokens above take 321 us).
template <int D, bool ALT>
__global__ void __launch_bounds__(THREADS, 1) attn_kv8_shared_tc_kernel(const __grid_constant__ Args a) {
  using L = Smem<D, ALT>;
  constexpr int ROWS = L::ROWS, ST = L::ST;
  extern __shared__ __align__(1024) uint8_t sm[];
  __shared__ Seg segs[2];                       // shares of items, in turn; an empty one ends
  __shared__ int2 row_at[2][256];               // of a thread's row: its sequence and token
  __shared__ Tile tiles[ST];
  __shared__ float2 raw_scale[MAX_RAW];         // K's and V's
  __shared__ int2 raw_at[MAX_RAW];              // x and key0
  __shared__ float2 halves[ALT ? 2 : 1][2][128];  // ALT: (m, l) of a row's two halves
  __shared__ __align__(8) uint64_t bars[2 + 2 * ST + 4 + 4 + 4 + 2 + 2 + 1 + 2 * MAX_RAW + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int sh_abort;
  volatile int* abort_flag = &sh_abort;
  uint64_t *q_full = bars, *kv_full = bars + 2, *kv_empty = kv_full + ST;
  uint64_t *s_full = kv_empty + ST, *p_full = s_full + 4, *o_full = p_full + 4, *o_empty = o_full + 2, *pv_done = o_empty + 2, *drain = pv_done + 2, *halves_full = drain + 2;
  uint64_t *raw_full = halves_full + 1, *raw_empty = raw_full + MAX_RAW, *seg_full = raw_empty + MAX_RAW, *seg_empty = seg_full + 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, B = a.S * a.F;
  int* lists = reinterpret_cast<int*>(sm + L::RAW + a.raw * L::RAW_TILE);
  const Lists l{lists, lists + B + 1, lists + 2 * B + 1, lists + 3 * B + 2, lists + 3 * B + a.S + 3};
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&q_full[i], ALT ? 8 : 4);  // of M tile i; ALT: of every other share, whose q all eight warps bring in
      mbar_init(&o_full[i], 1), mbar_init(&o_empty[i], ALT ? 8 : 4), mbar_init(&pv_done[i], 1), mbar_init(&drain[i], 1);
      mbar_init(&seg_full[i], 1), mbar_init(&seg_empty[i], 15);
    }
    for (int i = 0; i < ST; i++) mbar_init(&kv_full[i], 4), mbar_init(&kv_empty[i], 2);
    for (int i = 0; i < 4; i++) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 4);
    for (int i = 0; i < MAX_RAW; i++) mbar_init(&raw_full[i], 2), mbar_init(&raw_empty[i], 4);  // the bulk copies' bytes, the scales
    mbar_init(halves_full, 8);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  griddep_wait();  // programmatic dependent launch: the previous kernel has completed
  griddep_launch();
  // a wait of the whole warp: every lane gives up when one does
  auto wait = [&](uint64_t* bar, int parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, ST_KV8_WAIT)) != 0;
  };

  // the i'th share: for the warps that work on it
  auto take = [&](int i) { return wait(&seg_full[i & 1], (i >> 1) & 1); };
  auto leave = [&](int i) {
    __syncwarp();
    mbar_arrive_if(&seg_empty[i & 1], lane == 0);
  };

  static_assert(2 * tc::SOFTMAX_REGS + tc::CONVERT_REGS + tc::MMA_REGS <= 4 * 128, "the split must come out of the launch's registers");
  if (warp >= 12) {
    set_regs_down<tc::MMA_REGS>();
    // ---------------- MMA issuer of M tile t, one warp each.  The whole warp walks the loop, one lane issues
    const int t = warp - 12;
    const uint32_t leader = elect_one();
    constexpr uint32_t IDESC_S = idesc_bf16(128, KEYS), IDESC_O = idesc_f16(128, D) | (1u << 16);  // V MN-major
    const uint64_t dq = sdesc_noswz(smem_u32(sm) + (ALT ? 0 : t * L::QT), 2048, 128), dk = sdesc_noswz(smem_u32(sm + L::K), 1024, 128);
    const uint64_t dv = sdesc_noswz(smem_u32(sm + L::V), 128, 1024);
    const uint32_t t_s = tmem + 128 * t, t_o = tmem + 256 + 128 * t;
    bool ok = true;
    int base = 0, js = 0, so = 0, sq = 0;  // tiles of the segments before; tiles and segments that t took part in; q's that came in
    for (int i = 0; t < 2 && ok; i++) {
      ok = take(i);
      const Seg& g = segs[i & 1];
      const int nt = g.tb - g.ta;
      if (!ok || nt == 0) break;
      auto stage = [&](int j) { return (base + j - g.ta) % ST; };
      auto phase = [&](int j) { return ((base + j - g.ta) / ST) & 1; };
      auto pass = [&](int j, int to) {  // tiles [j, to) are the other M tile's: only the barriers
        for (; j < to && ok; j++) {
          ok = wait(&kv_full[stage(j)], phase(j));
          mbar_arrive_if(&kv_empty[stage(j)], leader != 0);
        }
      };
      auto issue_s = [&](int j, int f) {
        ok = ok && wait(&kv_full[stage(j)], phase(j));
        if (!ok) return;
        tc_fence_after();
        if (leader) {
          const uint64_t b = dk + stage(j) * (L::KT >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; k++) umma_f16(t_s + 64 * f, dq + k * (4096 >> 4), b + k * (2048 >> 4), IDESC_S, k > 0 ? 1u : 0u);
          umma_commit(&s_full[2 * t + f]);
        }
        __syncwarp();
      };
      const bool q_here = ALT || g.of(t).act;
      // each q is waited for in turn, without tiles here too: else the next one's phase would be taken for the one before it.  ALT: this
      // warp's lag is bounded by the shares alone, two of them, so their q's have a barrier each
      if (q_here) ok = wait(&q_full[ALT ? i & 1 : t], (ALT ? i >> 1 : sq) & 1);
      if (!g.of(t).act) {
        pass(g.ta, g.tb);
      } else {
        int j = tile_from<ALT>(g, t, g.ta);
        pass(g.ta, j);
        issue_s(j, js & 1);
        bool first = true;
        while (j < g.tb && ok) {
          const int f = js & 1, nx = tile_from<ALT>(g, t, j + 1);
          // S of the next tile goes ahead of this one's P V, unless that needs a stage that is freed by this one
          const bool ahead = nx < g.tb && nx - j < ST;
          if (ahead) pass(j + 1, nx), issue_s(nx, f ^ 1);
          ok = ok && (!first || so == 0 || wait(&o_empty[t], (so - 1) & 1)) && wait(&p_full[2 * t + f], (js >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            const uint64_t b = dv + stage(j) * (L::KT >> 4);
#pragma unroll
            for (int k = 0; k < KEYS / 16; k++) umma_f16_ts(t_o, t_s + 64 * f + k * 8, b + k * (256 >> 4), IDESC_O, !first || k > 0 ? 1u : 0u);
            umma_commit(&kv_empty[stage(j)]);
            umma_commit(&pv_done[t]);
            if (nx >= g.tb) umma_commit(&o_full[t]);
          }
          __syncwarp();
          if (!ahead) {
            pass(j + 1, nx);
            if (nx < g.tb) issue_s(nx, f ^ 1);
          }
          first = false, j = nx, js++;
        }
        so++;
      }
      sq += q_here ? 1 : 0;
      base += nt;
      leave(i);
    }
    if (leader && t < 2) {
      umma_commit(&drain[t]);
      mbar_wait_drain(&drain[t], 0, kDrainCycles);
    }
    if (warp == 14) {
      // ---------------- codes and scales of every tile, in order, as far ahead as there is room
      int j = 0;
      for (int i = 0; ok; i++) {
        ok = take(i);
        const Seg& g = segs[i & 1];
        const int nt = g.tb - g.ta;
        if (!ok || nt == 0) break;
        Cursor c = cursor_at<ROWS>(a, l, g, g.ta);
        for (int k = 0; k < nt; k++, j++) {
          const int st = j % a.raw;
          if (j >= a.raw) ok = wait(&raw_empty[st], (j / a.raw - 1) & 1);
          if (!ok) break;
          if (lane == 0) {
            const size_t blk = block_of(a, g, c);
            uint8_t* to = sm + L::RAW + st * L::RAW_TILE;
            raw_at[st] = make_int2(c.x, c.kt * KEYS);
            mbar_arrive_expect_tx(&raw_full[st], L::RAW_TILE);
            bulk_load(to, (c.x < 0 ? a.pk : a.kc) + blk * (KEYS * D), KEYS * D, &raw_full[st]);
            bulk_load(to + KEYS * D, (c.x < 0 ? a.pv : a.vc) + blk * (KEYS * D), KEYS * D, &raw_full[st]);
            const float *ks = (c.x < 0 ? a.pks : a.ks) + blk, *vs = (c.x < 0 ? a.pvs : a.vs) + blk;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&raw_scale[st].x)), "l"(ks) : "memory");
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&raw_scale[st].y)), "l"(vs) : "memory");
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&raw_full[st])) : "memory");
          }
          __syncwarp();
          if (k + 1 < nt) advance<ROWS>(a, l, g, c);
        }
        leave(i);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      for (int k = max(j - a.raw, 0); k < j; k++) mbar_wait_drain(&raw_full[k % a.raw], (k / a.raw) & 1, kDrainCycles);  // copies in flight land, whatever the others do
    }
    if (warp == 15) {
      // ---------------- the shares
      make_lists<ROWS>(a, l);
      const int total = a.items > 0 ? 1 : l.pre[a.S], run = max((total + a.ctas - 1) / a.ctas, 1), u_begin = a.items > 0 ? 0 : (int)min((long long)blockIdx.x * run, (long long)total);
      const int u_end = (int)min((long long)u_begin + run, (long long)total);
      for (int u = u_begin, i = 0; ok; i++) {
        Seg g;
        g.ta = g.tb = 0;
        if (u < u_end) g = segment<D, ALT>(a, l, u, u_end), g.last = (u - g.ta + g.tiles - 1) / run;
        ok = i < 2 || wait(&seg_empty[i & 1], ((i >> 1) - 1) & 1);
        if (!ok) break;
        const int nt = g.tb - g.ta;
        if (lane == 0) segs[i & 1] = g;
        __syncwarp();
        mbar_arrive_if(&seg_full[i & 1], lane == 0);
        if (nt == 0) break;
        u = a.items > 0 ? u_end : u + nt;
      }
    }
  } else if (warp >= 8) {
    set_regs_down<tc::CONVERT_REGS>();
    // ---------------- converters: warp w rows 16 w .. of a block.  A lane's 16-byte pieces lie on a diagonal: eight lanes read eight
    // pieces of different banks, and write eight rows.  K's and V's codes of the next tile, if they are there, are fetched as soon as
    // this tile's are out of the registers: a tile is mostly waiting, not work
    constexpr int PER = D / 32, PIECES = D / 16;  // pieces of a K or V block that a lane takes, of a row
    const int w = warp - 8;
    int at[PER];  // of a piece in a tile's codes
    uint8_t* to[PER];  // and of its operand
#pragma unroll
    for (int x = 0; x < PER; x++) {
      const int row = 16 * w + 8 * (x & 1) + (lane & 7), p = ((D == 64 ? (lane & 7) >> 1 : lane & 7) + (lane >> 3) + 4 * (x >> 1)) % PIECES;
      at[x] = row * D + 16 * p, to[x] = sm + L::K + (2 * p * KEYS + row) * 16;
    }
    uint4 kr[PER], vr[PER];
    float2 scale, scale_next;
    int2 where, where_next;
    bool ok = true, have = false;  // have: the next tile's codes are in the registers
    for (int j = 0, i = -1, left = 0, rs = 0, rph = 0, st = 0, sph = 0; ok; j++, left--) {
      if (left == 0) {
        if (i >= 0) leave(i);
        ok = take(++i);
        left = segs[i & 1].tb - segs[i & 1].ta;
        if (!ok || left == 0) break;
      }
      auto fetch = [&](uint4 (&r)[PER], int from) {
#pragma unroll
        for (int x = 0; x < PER; x++) r[x] = *reinterpret_cast<const uint4*>(sm + L::RAW + rs * L::RAW_TILE + from + at[x]);
      };
      auto fetched = [&] {  // the stage of codes is free again
        __syncwarp();
        mbar_arrive_if(&raw_empty[rs], lane == 0);
        if (++rs == a.raw) rs = 0, rph ^= 1;
      };
      if (!have) {
        ok = wait(&raw_full[rs], rph);
        if (!ok) break;
        fetch(kr, 0), fetch(vr, KEYS * D);
        scale_next = raw_scale[rs], where_next = raw_at[rs];
        fetched();
      }
      scale = scale_next, where = where_next;
      const bool none = scale.y < kTinyScale;  // V becomes zero
      ok = j < ST || wait(&kv_empty[st], sph ^ 1);
      if (!ok) break;
      if (w == 0 && lane == 0) {
        const float v1 = none ? 1.f : scale.y;
        tiles[st] = {where.x, where.y, scale.x * a.scale_log2, __log2f(v1), __frcp_rn(v1) * L_SCALE, none ? Z_TOP : P_TOP};
      }
      have = left > 1 && __all_sync(0xffffffffu, mbar_try_wait(&raw_full[rs], rph));
#pragma unroll
      for (int x = 0; x < PER; x++) tc::store_codes<KEYS, false>(to[x] + st * L::KT, 0, 0, kr[x]);
      if (have) fetch(kr, 0), scale_next = raw_scale[rs], where_next = raw_at[rs];
#pragma unroll
      for (int x = 0; x < PER; x++) tc::store_codes<KEYS, true>(to[x] + (L::V - L::K) + st * L::KT, 0, 0, none ? make_uint4(0, 0, 0, 0) : vr[x]);
      if (have) fetch(vr, KEYS * D);
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_if(&kv_full[st], lane == 0);
      if (have) fetched();
      if (++st == ST) st = 0, sph ^= 1;
    }
  } else {
    set_regs_up<tc::SOFTMAX_REGS>();
    // ---------------- softmax of M tile t: thread = row.  It brings in its row of q itself (ALT: half of it)
    const int t = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, t_o = tmem + 256 + 128 * t + lanes;
    bool ok = true;
    int base = 0, js = 0, so = 0, so1 = 0, segs_done = 0;  // tiles of the shares before; tiles that t took part in; outputs stored (ALT: of M tile 0 and 1); shares
    int known = -1;  // the last tile whose scores were seen: every one up to it was in place
    int4 open = make_int4(-1, 0, 0, 0);
    const int mine_r = (ALT ? 0 : 128 * t) + (warp & 3) * 32 + lane, me = 128 * t + (warp & 3) * 32 + lane;  // this thread's row of an item
    auto load_q = [&](int i) {  // of the i'th share; every product with the q before it is done: its last scores have been read
      const Seg& g = segs[i & 1];
      const int row = min(g.q * ROWS + mine_r, g.rows - 1);  // rows past the last are copies of it
      const int x = seq_of_token(a, l, g.s, row / a.G), token = row / a.G - (l.tok[x] - l.tok[g.s * a.F]);
      row_at[i & 1][me] = make_int2(x, token);
      if (!ALT && !g.of(t).act) return;
      const uint16_t* mine = a.q + x * a.sq_b + token * a.sq_t + (size_t)(g.h * a.G + row % a.G) * a.sq_h;
      const uint32_t dst = smem_u32(sm + (ALT ? 0 : t * L::QT) + (warp & 3) * 32 * 16);
      // four lanes bring 64 bytes of a row, whole sectors, eight rows at a time (a lane a row took 4 us); rows side by side in a bank line
      constexpr int CH = ALT ? D / 16 : D / 8;  // 16-byte pieces of this M tile's threads
      const int piece = (ALT ? t * CH : 0) + (lane >> 3);
#pragma unroll
      for (int rg = 0; rg < 32; rg += 8) {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), rg + (lane & 7)));
#pragma unroll
        for (int c = 0; c < CH; c += 4)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + (piece + c) * 2048 + (rg + (lane & 7)) * 16), "l"(src + 8 * (piece + c)) : "memory");
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_if(&q_full[ALT ? i & 1 : t], lane == 0);
    };
    ok = take(0);
    if (ok && segs[0].tb > segs[0].ta) load_q(0);
    for (; ok; segs_done++) {
      const Seg& g = segs[segs_done & 1];
      const int nt = g.tb - g.ta, row = g.q * ROWS + mine_r, valid = g.rows;
      if (nt == 0) break;
      const bool whole = g.ta == 0 && g.tb == g.tiles;
      const int2 rat = row_at[segs_done & 1][me];
      const int rx = rat.x, ri = rat.y, own_lim = l.len[rx] + ri + 1;
      const int warp_x0 = __shfl_sync(0xffffffffu, rx, 0), warp_x1 = __shfl_sync(0xffffffffu, rx, 31);
      float m = -INFINITY, sum_l = 0.f;
      if (g.of(t).act) {
        int j = tile_from<ALT>(g, t, g.ta);
        auto announce = [&](int f) {  // P in buffer f is complete
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          mbar_arrive_if(&p_full[2 * t + f], lane == 0);
        };
        bool first = true, fresh = true;  // fresh: a row of the warp has seen no key yet
        while (j < g.tb) {
          const int f = js & 1, at = base + j - g.ta;
          const uint32_t t_s = tmem + 128 * t + 64 * f + lanes;
          uint32_t r0[32], r1[32];
          // what the tile is, before its scores are there; where others lie between, with them: only then is the stage's phase surely its own
          const bool near = at - known < ST;
          ok = (near || wait(&s_full[2 * t + f], (js >> 1) & 1)) && wait(&kv_full[at % ST], (at / ST) & 1);
          if (!ok) break;
          known = at;
          const int x = tiles[at % ST].x, key0 = tiles[at % ST].key0;
          float c = tiles[at % ST].c, lvs = tiles[at % ST].lvs, ivs = tiles[at % ST].ivs;
          const float top = tiles[at % ST].top;
          const bool mine = x < 0 || (x >= warp_x0 && x <= warp_x1);  // whether the warp has rows that see this cache
          const int lim = x < 0 ? g.P : x == rx ? own_lim : 0;
          float mx, sum = 0.f;
          bool look = false;  // whether the row's first keys are in this tile
          auto top32 = [&](const uint32_t (&r)[32]) {
            float y[11];
#pragma unroll
            for (int e = 0; e < 10; e++) y[e] = max3f(__uint_as_float(r[3 * e]), __uint_as_float(r[3 * e + 1]), __uint_as_float(r[3 * e + 2]));
            y[10] = fmaxf(__uint_as_float(r[30]), __uint_as_float(r[31]));
#pragma unroll
            for (int e = 0; e < 3; e++) y[e] = max3f(y[3 * e], y[3 * e + 1], y[3 * e + 2]);
            return max3f(max3f(y[0], y[1], y[2]), y[9], y[10]);
          };
          // P' = 2^(s c + log2 vs - m) of 32 scores into columns `at` of P; returns their sum
          auto exps = [&](const uint32_t (&r)[32], uint32_t at, float mu) {
            const unsigned long long c2 = f2_pack(c, c), sh2 = f2_pack(lvs - mu, lvs - mu);
            unsigned long long sum2[2] = {0ull, 0ull};
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; e++) {
              float x0, x1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), c2, sh2), x0, x1);
              const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
              sum2[e & 1] = f2_add(sum2[e & 1], f2_pack(p0, p1));
              pk[e] = tc::pack_h2_finite(p0, p1);
            }
            tmem_st16(t_s + at, pk);
            float lo, hi;
            f2_unpack(f2_add(sum2[0], sum2[1]), lo, hi);
            return lo + hi;
          };
          ok = !near || wait(&s_full[2 * t + f], (js >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          tmem_ld32(t_s, r0);
          if (!mine) {  // no row of the warp: P is zero
            uint32_t zero[16];
#pragma unroll
            for (int e = 0; e < 16; e++) zero[e] = 0u;
            tmem_ld_wait();
            tmem_st16(t_s, zero);
            tmem_st16(t_s + 16, zero);
            announce(f);
            first = false, js++, j = tile_from<ALT>(g, t, j + 1);
            continue;
          }
          // the fewest keys that a row of this warp sees: tiles up to there need no mask
          const bool edge = key0 + KEYS > (x < 0 ? g.P : __reduce_min_sync(0xffffffffu, lim));
          tmem_ld_wait();
          tmem_ld32(t_s + 32, r1);
          // a tile that every row sees whole, once rows have a maximum: P with the maximum so far, while the second half of
          // the scores arrives and the new maximum is found beside the exponentials; they stand unless it grew too far.  Else the maximum
          // comes first.  One copy of the exponentials for all (the cold instruction cache cost 3 us before the second tile)
          bool guess = !(fresh || edge), sink_looked = false;
          float mu = m;
#pragma unroll 1
          while (true) {
            if (!guess && !sink_looked) {  // the row's maximum, O and the sum brought to it
              tmem_ld_wait();
              const int left = lim - key0;  // keys of the tile that the row sees
              if (edge) {
#pragma unroll
                for (int e = 0; e < 32; e++) {
                  if (e >= left) r0[e] = 0xff800000u;
                  if (32 + e >= left) r1[e] = 0xff800000u;
                }
              }
              const bool begins = m == -INFINITY;  // the row's first keys
              mx = left > 0 ? fmaf(fmaxf(top32(r0), top32(r1)), c, lvs) : -INFINITY;
              const bool need = mx > m + top;
              const float up = top - P_MOVE;
              const float mn = begins ? mx - up : need ? mx - (mx > m + (P_TOP + 12.f) ? fmaxf(up, P_UP_SINK) : up) : m;
              if (!first && __any_sync(0xffffffffu, need && !begins)) {  // O through registers (warp-collective)
                // O must hold every product up to this M tile's last tile; the barrier's next arrival needs P of this row
                ok = wait(&pv_done[t], (js - 1) & 1);
                if (!ok) break;
                tc_fence_after();
                const float half = need && !begins ? ex2_approx(0.5f * (m - mn)) : 1.f, alpha = half * half;
                sum_l = sum_l * half * half;  // what zero blocks put there may be as large as alpha is small
#pragma unroll
                for (int y = 0; y < D / 16; y++) {
                  uint32_t r[16];
                  tmem_ld16(t_o + y * 16, r);
                  tmem_ld_wait();
#pragma unroll
                  for (int e = 0; e < 16; e++) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
                  tmem_st16(t_o + y * 16, r);
                }
              }
              m = mn;
              look = begins && m != -INFINITY;
              // a row that sees nothing of the tile takes no part in its scales, which may be NaN; scores out of sight are -inf,
              // and -inf * 0 of a zero scale must not be NaN
              mu = m == -INFINITY ? 0.f : m;
              if (edge) {
                if (left <= 0) c = 1.f, lvs = 0.f, ivs = 1.f;
                if (c == 0.f) {
#pragma unroll
                  for (int e = 0; e < 32; e++) {
                    r0[e] = e < left ? 0u : r0[e];
                    r1[e] = 32 + e < left ? 0u : r1[e];
                  }
                  c = 1.f;
                }
              }
            }
            sum = exps(r0, 0, mu);
            const float ma = guess ? top32(r0) : 0.f;
            tmem_ld_wait();
            sum += exps(r1, 16, mu);
            if (guess) {
              mx = fmaf(fmaxf(ma, top32(r1)), c, lvs);
              if (!__any_sync(0xffffffffu, mx > m + top)) break;
              guess = false;
              continue;
            }
            const bool sink = look && sum < 1.05f * SINK_SUM;  // a row's first tile whose other keys add up to a twentieth of its largest one
            if (sink_looked || !__any_sync(0xffffffffu, sink)) break;
            m -= sink ? P_UP_SINK - P_UP : 0.f;
            mu = m == -INFINITY ? 0.f : m;
            sink_looked = true;
          }
          if (!ok) break;
          fresh = fresh && __any_sync(0xffffffffu, m == -INFINITY);
          sum_l += sum * ivs;
          announce(f);
          first = false, js++, j = tile_from<ALT>(g, t, j + 1);
        }
        if (!ok) break;
      }
      base += nt;
      // the next item's products start before this one's O is stored (ALT: both M tiles' scores must have been read)
      auto load_next = [&] {
        ok = take(segs_done + 1);
        if (ok && segs[(segs_done + 1) & 1].tb > segs[(segs_done + 1) & 1].ta) load_q(segs_done + 1);
        return ok;
      };
      if (!ALT && !load_next()) break;
      const size_t slot = 2 * (size_t)blockIdx.x + (segs_done ? 1 : 0);
      const int hq = g.h * a.G + min(row, valid - 1) % a.G;
      const size_t out_row = ((size_t)rx * a.n + ri) * (a.G * a.H) + hq;
      uint16_t* op = a.out + rx * a.so_b + ri * a.so_t + hq * a.so_h;
      if (g.ta == 0 && !whole) {
        open = make_int4(g.last, (int)slot, g.h, g.q * ROWS);
        if (!ALT || t == 0) a.row_at[(size_t)blockIdx.x * ROWS + mine_r] = row < valid ? rx * a.n + ri : -1;
      }
      // dims y16 .. y16 + 15 of the row, o = O / l where it is whole.  Parts lie as [dims / 4][row][4]: a warp writes whole lines
      auto put = [&](int y16, const float (&o)[16]) {
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<float4*>(a.part_o + ((slot * (D / 4) + (y16 + e) / 4) * ROWS + mine_r) * 4) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else if (!a.own) {
#pragma unroll
          for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4*>(a.row_o + out_row * D + y16 + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; e += 8)
            *reinterpret_cast<uint4*>(op + y16 + e) = make_uint4(pack_bf2(o[e], o[e + 1]), pack_bf2(o[e + 2], o[e + 3]), pack_bf2(o[e + 4], o[e + 5]), pack_bf2(o[e + 6], o[e + 7]));
        }
      };
      auto put_ml = [&](float mm, float ll) {
        if (!whole) a.part_ml[slot * ROWS + mine_r] = make_float2(mm, ll);
        else if (!a.own) a.row_ml[out_row] = make_float2(mm, ll / L_SCALE);
      };
      if (ALT) {
        float2(&hv)[2][128] = halves[segs_done & 1];
        hv[t][mine_r] = make_float2(m, sum_l);
        __syncwarp();
        mbar_arrive_if(halves_full, lane == 0);
        ok = wait(halves_full, segs_done & 1);
        ok = ok && (!g.m0.act || wait(&o_full[0], so & 1)) && (!g.m1.act || wait(&o_full[1], so1 & 1));
        if (!ok) break;
        tc_fence_after();
        if (!load_next()) break;
        const float2 h0 = hv[0][mine_r], h1 = hv[1][mine_r];
        const float mm = fmaxf(h0.x, h1.x);
        auto weigh = [&](const float2& h, float& w) {  // factor of O; l's is the same, by halves
          const float half = h.x == -INFINITY ? 0.f : ex2_approx(0.5f * (h.x - mm));
          w = half * half;
          return h.y * half * half;
        };
        float w0, w1;
        const float ll = weigh(h0, w0) + weigh(h1, w1), inv = whole ? L_SCALE / ll : 1.f;
        w0 *= inv, w1 *= inv;
#pragma unroll
        for (int y = 0; y < D / 32; y++) {  // this thread's half of the dims
          const int y16 = 16 * (t * (D / 32) + y);
          uint32_t a0[16], a1[16];
          if (g.m0.act) tmem_ld16(tmem + 256 + lanes + y16, a0);
          if (g.m1.act) tmem_ld16(tmem + 384 + lanes + y16, a1);
          tmem_ld_wait();
          float o[16];
#pragma unroll
          for (int e = 0; e < 16; e++) o[e] = (g.m0.act ? __uint_as_float(a0[e]) * w0 : 0.f) + (g.m1.act ? __uint_as_float(a1[e]) * w1 : 0.f);
          if (row < valid) put(y16, o);
        }
        if (t == 0 && row < valid) put_ml(mm, ll);
        tc_fence_before();
        __syncwarp();
        if (g.m0.act) mbar_arrive_if(&o_empty[0], lane == 0), so++;
        if (g.m1.act) mbar_arrive_if(&o_empty[1], lane == 0), so1++;
      } else if (!g.of(t).act) {
        if (row < valid && !whole) a.part_ml[slot * ROWS + mine_r] = make_float2(-INFINITY, 0.f);
      } else {
        ok = wait(&o_full[t], so & 1);
        if (!ok) break;
        tc_fence_after();
        const float inv = whole ? L_SCALE / sum_l : 1.f;
#pragma unroll
        for (int y = 0; y < D / 16; y++) {
          uint32_t x[16];
          tmem_ld16(t_o + y * 16, x);
          tmem_ld_wait();
          float o[16];
#pragma unroll
          for (int e = 0; e < 16; e++) o[e] = __uint_as_float(x[e]) * inv;
          if (row < valid) put(16 * y, o);
        }
        if (row < valid) put_ml(m, sum_l);
        tc_fence_before();
        __syncwarp();
        mbar_arrive_if(&o_empty[t], lane == 0);
        so++;
      }
      leave(segs_done);
    }
    if (a.items == 0 && tid == 0) a.unfinished[blockIdx.x] = open;
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Merges the parts of an item, always in the same order.  blockIdx.x = c: the item that CTA c began and did not finish; blockIdx.y: eight of
// its rows; thread = a row's dims 4 (thread / 8) .. and, where heads are 128 wide, those 64 on.
template <int D, int ROWS>
__global__ void __launch_bounds__(128) attn_kv8_shared_join_kernel(const __grid_constant__ Args a) {
  __shared__ float2 sh_ml[MAX_CTAS][8];
  griddep_wait();
  griddep_launch();
  const int4 open = a.unfinished[blockIdx.x];
  if (open.x < 0) return;
  const int c0 = blockIdx.x, parts = open.x - c0 + 1, r = threadIdx.x & 7, row = blockIdx.y * 8 + r;
  const int at = a.row_at[(size_t)c0 * ROWS + row];
  auto slot = [&](int p) { return (size_t)(p == 0 ? open.y : 2 * (c0 + p)); };
  for (int p = threadIdx.x >> 3; p < parts; p += 16) sh_ml[p][r] = at < 0 ? make_float2(0.f, 1.f) : a.part_ml[slot(p) * ROWS + row];
  __syncthreads();
  if (at < 0) return;
  float mx = -INFINITY, sum = 0.f;
  for (int p = 0; p < parts; p++) mx = fmaxf(mx, sh_ml[p][r].x);
  float4 v[D / 64];
#pragma unroll
  for (int y = 0; y < D / 64; y++) v[y] = make_float4(0.f, 0.f, 0.f, 0.f);
  const int chunk = threadIdx.x >> 3;
#pragma unroll 4
  for (int p = 0; p < parts; p++) {
    const float2 ml = sh_ml[p][r];
    const float half = ml.x == -INFINITY ? 0.f : ex2_approx(0.5f * (ml.x - mx)), f = half * half;
    sum += ml.y * half * half;
#pragma unroll
    for (int y = 0; y < D / 64; y++) {
      const float4 o = *reinterpret_cast<const float4*>(a.part_o + ((slot(p) * (D / 4) + chunk + 16 * y) * ROWS + row) * 4);
      if (ml.x != -INFINITY) v[y].x += o.x * f, v[y].y += o.y * f, v[y].z += o.z * f, v[y].w += o.w * f;  // else the part is empty, or all its scores were NaN
    }
  }
  const float inv = L_SCALE / sum;
  const int hq = open.z * a.G + (open.w + row) % a.G, b = at / a.n, i = at % a.n;
  const size_t out_row = (size_t)at * (a.G * a.H) + hq;
#pragma unroll
  for (int y = 0; y < D / 64; y++) {
    const int d = 4 * chunk + 64 * y;
    if (a.own) *reinterpret_cast<uint2*>(a.out + b * a.so_b + i * a.so_t + hq * a.so_h + d) = make_uint2(pack_bf2(v[y].x * inv, v[y].y * inv), pack_bf2(v[y].z * inv, v[y].w * inv));
    else *reinterpret_cast<float4*>(a.row_o + out_row * D + d) = make_float4(v[y].x * inv, v[y].y * inv, v[y].z * inv, v[y].w * inv);
  }
  if (!a.own && chunk == 0) a.row_ml[out_row] = make_float2(mx, sum / L_SCALE);
}

template <int D, bool ALT>
static int launch(cudaStream_t st, Args a, const char* what) {
  using L = Smem<D, ALT>;
  const int rc = smem_attr_once((const void*)attn_kv8_shared_tc_kernel<D, ALT>, L::BUDGET, what);
  if (rc) return rc;
  const int lists = list_bytes(a.S, a.S * a.F), room = (L::BUDGET - L::RAW - lists) / L::RAW_TILE;
  static_assert((L::BUDGET - L::RAW - (5 * MAXB + 3) * 4) / L::RAW_TILE >= 1, "codes in flight beside the longest lists");
  a.raw = room < MAX_RAW ? room : MAX_RAW;
  launch_k(attn_kv8_shared_tc_kernel<D, ALT>, (unsigned)(a.items > 0 ? a.S * a.H * a.items : a.ctas), THREADS, L::RAW + a.raw * L::RAW_TILE + lists, st, a);
  if (a.items == 0) launch_k(attn_kv8_shared_join_kernel<D, L::ROWS>, dim3(a.ctas, L::ROWS / 8), 128, 0, st, a);
  return check_launch(what);
}

// Fixed on the host from sizes alone.
struct Plan {
  bool few, alt, own;  // one item per head with all rows and keys; rows of an item; whether the tcgen05 kernel takes the own slots too
  bool whole;          // a CTA for each item of it
  int items, ctas;
  split::Plan s;       // of few, or of the sequences' own slots
  long long o_off, ml_off, un_off, at_off, row_off, rml_off, s_off, sun_off, bytes;  // workspace
  static long long up(long long v) { return (v + 255) / 256 * 256; }
  // Lays out what runs of items of so many rows leave for the join; its bytes.
  long long run_bytes(int rows, int D, int sms) {
    ctas = sms < MAX_CTAS ? sms : MAX_CTAS;
    ml_off = up(2LL * ctas * rows * D * 4);
    un_off = ml_off + up(2LL * ctas * rows * 8);
    at_off = un_off + up(ctas * 16LL);
    return at_off + up((long long)ctas * rows * 4);
  }
};
// Rules on sizes alone (capacities stand for lengths), both sides measured; the names are S x F x n, Hq / H heads x D, prefix + own slots.
//   few      up to 32 rows on a prefix (16 of heads 128 wide): against the tcgen05 kernel 1 x 8 x 1, 8/8 x 64, 730 + 60: 7 / 30 us;
//            1 x 32 x 1, 8/8 x 64, 8,191 + 60: 25 / 44; 1 x 4 x 1, 32/8 x 128, 131,000 + 60: 83 / 138
//   whole    a CTA for each item, where the SMs that this leaves idle could do no more than IDLE_TILES tiles each (few: tiles of one
//            warp, eight a CTA): it saves the parts and a kernel.  8 x 32 x 1, 8/8 x 64, 2,000 + 60 (few): 35 / 38 us, 1 x 32 x 1, 8/8 x 64,
//            8,191 + 60 (few): 76 / 25; near where the rule changes 32 rows lose by it (1 x 24 x 1, 8/8 x 64,
//            1,500 + 60: 27 / 18); 8 x 8 x 16, 8/8 x 64, 730 + 32: 25 / 30; 1 x 64 x 1, 32/8 x 128, 8,191 + 60: 215 / 56
//   own      the tcgen05 kernel takes the own slots too: where each sequence has more rows than kv8_split.cu takes, or where an item's own
//            tiles (of a few rows each) are not many.  1 x 32 x 1, 32/8 x 128, 8,191 + 60: 34 / 40 us; 1 x 64 x 1, 32/8 x 128, 8,191 + 60:
//            43 / 56; 1 x 64 x 1, 32/8 x 128, 2,000 + 500: 75 / 53; 1 x 40 x 1, 2/2 x 64, 100 + 10: 42 / 14
//   alt      ALT: up to 128 rows (1 x 32 x 1, 32/8 x 128, 131,000 + 60: 132 / 173 us), and of more where that is little work, whose items
//            otherwise leave SMs idle: 1 x 16 x 32, 32/32 x 64, 730 + 0: 22 / 37; 1 x 32 x 32, the same: 42 / 35; 1 x 8 x 256, 32/8 x 128,
//            6,001 + 511: 402 / 311
constexpr int IDLE_TILES = 24, IDLE_FEW = 80, MOST_TILES = 256, OWN_TILES = 64, ALT_TILES = 24;
static int few_rows(int D) { return D == 64 ? split::FEW_ROWS : 16; }
static bool leave_idle(long long items, long long tiles, long long idle, int sms) {
  return tiles <= MOST_TILES && ((items + sms - 1) / sms * sms - items) * tiles <= idle * sms;
}

static Plan make_plan(int S, int B, int n, int Hq, int H, int D, int Cp, int C, int sms) {
  Plan x{};
  const int F = B / S, G = Hq / H;
  const long long all = (long long)F * n * G, SH = (long long)S * H;
  x.few = all <= few_rows(D);
  if (x.few) {
    const int kt = split::keys_per_tile(D);
    const long long tiles = Cp / kt + (long long)F * (C / kt);
    x.s = split::make_plan(S, F * n, Hq, H, D, Cp, false, sms, tiles, leave_idle(SH, tiles, IDLE_FEW, sms) ? MOST_TILES : 0);
    x.sun_off = x.s.full_off;
    x.bytes = x.sun_off + (x.s.whole ? 0 : Plan::up(x.s.ctas * 16LL));
    return x;
  }
  // own tiles of an item of so many rows: of the sequences that have rows in it
  auto own_of = [&](int rows) {
    const long long seqs = (long long)n * G >= rows ? 2 : rows / ((long long)n * G) + 2;
    return (seqs < F ? seqs : F) * (C / BLK);
  };
  auto tiles_of = [&](int rows) { return Cp / BLK + (x.own ? own_of(rows) : 0); };
  x.own = (long long)n * G > split::FEW_ROWS || own_of(256) <= OWN_TILES || own_of(256) <= Cp / BLK;
  x.alt = all <= 128 || SH * ((all + 127) / 128) * tiles_of(128) <= (long long)ALT_TILES * sms;
  const int rows = x.alt ? 128 : 256;
  x.items = (int)((all + rows - 1) / rows);
  x.whole = leave_idle(SH * x.items, tiles_of(rows), IDLE_TILES, sms);
  const long long runs = x.run_bytes(rows, D, sms);
  x.row_off = x.whole ? 0 : runs;
  x.rml_off = x.row_off + (x.own ? 0 : Plan::up((long long)B * n * Hq * D * 4));
  x.s_off = x.bytes = x.rml_off + (x.own ? 0 : Plan::up((long long)B * n * Hq * 8));
  if (!x.own) x.s = split::make_plan(B, n, Hq, H, D, C, false, sms), x.sun_off = x.s_off + x.s.full_off, x.bytes = x.sun_off + (x.s.whole ? 0 : Plan::up(x.s.ctas * 16LL));
  return x;
}

}  // namespace shared
}  // namespace kv8
}  // namespace vt

extern "C" {

long long vt_attn_kv8_shared_ws_bytes(int S, int B, int n, int Hq, int H, int D, int Cp, int C) {
  using namespace vt::kv8;
  if (S <= 0 || B <= 0 || B % S || n <= 0 || Hq <= 0 || H <= 0 || Hq % H || Cp <= 0 || C <= 0 || (D != 64 && D != 128)) return 0;
  // what n tokens need, and any fewer that may follow with the same workspace: a plan for few rows needs most at its largest n
  const int sms = vt::sm_count();
  long long most = 0;
  for (int m = n < 64 ? n : 64; m > 0; m--) {
    const long long x = shared::make_plan(S, B, m, Hq, H, D, Cp, C, sms).bytes;
    if (x > most) most = x;
  }
  // longer calls take own slots too, and so need parts and rows' places at most: those of runs of 256 rows an item
  const long long runs = shared::Plan().run_bytes(256, D, sms);
  return n > 64 && runs > most ? runs : most;
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
  if (B > kv8::shared::MAXB) return set_error(E_SHAPE, "%s: B=%d (at most %d)", what, B, kv8::shared::MAXB);
  if (kv8::rows_meet({q, sq_b, sq_t, (Hq - 1) * sq_h + D}, {out, so_b, so_t, (Hq - 1) * so_h + D}, B, n))
    return set_error(E_SHAPE, "%s: out overlaps q", what);
  const int G = Hq / H, F = B / S, sms = sm_count();
  const long long most = 0x20000000LL;  // tiles of a list, rows
  if ((long long)B * n * Hq > most / 4 || (long long)S * H * (Cp / kv8::BLK) * ((long long)F * n * G / 128 + 1) > most ||
      (long long)B * H * (C / kv8::BLK) * ((long long)n * G / 8 + 2) > most)
    return set_error(E_SHAPE, "%s: B * Hq * n or B * H * C too large", what);
  const kv8::shared::Plan x = kv8::shared::make_plan(S, B, n, Hq, H, D, Cp, C, sms);
  char* w8 = static_cast<char*>(ws);
  const float c = scale * kv8::LOG2E;
  kv8::split::Args sa{q, sq_b, sq_t, sq_h, kc, vc, ks, vs, lens, counts, x.few ? S : B, n, G, H, C, 1, x.few ? F * n * G : n * G, x.few ? 1 : x.s.rg, x.s.ctas, c,
                      out, so_b, so_t, so_h, (float*)(w8 + x.s_off + x.s.o_off), (float2*)(w8 + x.s_off + x.s.ml_off), nullptr, nullptr, nullptr, nullptr,
                      pk, pv, pks, pvs, plens, Cp, F, (const float*)(w8 + x.row_off), (const float2*)(w8 + x.rml_off), (int4*)(w8 + x.sun_off)};
  if (x.few) return kv8::split::launch_any<kv8::split::SHARED>(st, sa, D, x.s.nt, x.s.whole, what);
  const kv8::shared::Args a{q, sq_b, sq_t, sq_h, pk, pv, pks, pvs, Cp, S, F, plens, kc, vc, ks, vs, C, lens, counts, n, G, H, x.ctas,
                            x.whole ? x.items : 0, x.own, 0, c, out, so_b, so_t, so_h, (float*)(w8 + x.row_off), (float2*)(w8 + x.rml_off), (float*)w8,
                            (float2*)(w8 + x.ml_off), (int4*)(w8 + x.un_off), (int*)(w8 + x.at_off)};
  rc = D == 64 ? (x.alt ? kv8::shared::launch<64, true>(st, a, what) : kv8::shared::launch<64, false>(st, a, what))
               : (x.alt ? kv8::shared::launch<128, true>(st, a, what) : kv8::shared::launch<128, false>(st, a, what));
  if (rc || x.own) return rc;
  return kv8::split::launch_any<kv8::split::OWN>(st, sa, D, x.s.nt, x.s.whole, what);
}

}  // extern "C"
