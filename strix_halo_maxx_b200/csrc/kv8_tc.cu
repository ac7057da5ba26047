// Attention of many rows over the 8-bit cache (a prompt, a chunk of one) on tcgen05, and the weights its slots receive.
//
// A kv head's rows r = i * G + g (token i, query head h G + g of its group) go 256 to an item, two M = 128 tiles that share
// every converted key tile.  The items' tiles of 64 keys (a cache block, so each tile has one K and one V scale) form
// one list that is cut into equal runs, one for each SM, whatever the sequences' lengths and the causal limits; an item
// that spans CTAs leaves its parts (unnormalised O, row max, row sum) for attn_kv8_tc_join_kernel.
//
// CTA = 16 warps (two of them idle):
//   warps 0-3, 4-7   softmax of M tile 0 / 1, thread = row (TMEM lane): q once an item, then P as f16 over the scores;
//   warps 8-11       codes -> operands in shared memory (ST stages), K's as bf16 and V's as f16, one tile's codes ahead in registers;
//   warps 12, 13     tcgen05.mma of M tile 0 / 1: S_(j+1), then O += P_j V_j (P from TMEM, V as an MN-major B operand).
// Codes are exact in both types: in bf16 byte b -> 0x4300 | b, and (that & ~0x80) - (that & 0x80 | 0x4300) = 128 + low bits -
// (128 or 256); in f16 (0x6400 | b ^ 0x80) - 1152.  K and V tiles have the same layout (no-swizzle core matrices, [D/8][64][8]).
// Scales cost nothing per score: K's joins the softmax scale of the tile; V's shifts the exponent, P' = vs P = 2^(s + log2 vs - m),
// and the row sum takes sum(P') / vs before P' is rounded.  P' is at most 2^15.9: m begins P_UP below the row's largest s + log2 vs and
// moves, O through registers, when that has grown by P_MOVE (by 4 instead of 8: 319 against 275 us below).  So P' has f16's 11 bits
// down to 2^-21 of the row's largest term and is off by 2^-32 of it below that; where one key is far above all before it and
// beside it, such as a sink, m goes P_UP_SINK below it and these are 2^-27 and 2^-38.  (In bf16, with its 8 bits, an output's error
// against 64 bits was 1.4 times its own rounding.)  V blocks with a scale below 2^-100 are zeros: their keys, with 1 for
// the scale, count in the sum alone, so m may lie 2^116 below them (with 8 as for others, a sink among them took away the bits of
// all other terms).  The scales of a head's other blocks may differ by 2^64.
// A 2048-token chunk over 6001 slots (32 / 8 heads x 128, 236 GFLOP): 276 us, 853 TFLOP/s (295 us under the power cap).  A tile takes about 2,040 cycles: the
// exponentials occupy the MUFU for 1,024 (16 a clock and SM), the MMAs are issued over about 1,500, and P -> PV -> S of a
// score buffer is a chain of which two are in flight.  128-key tiles with one score buffer were slower (346 us), so were
// four stages (299) and P announced one tile late (294).
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {
namespace tc {

constexpr int ROWS = 256, KEYS = 64, THREADS = 16 * 32, ST = 3, MAXB = 2048;
constexpr uint32_t TMEM_COLS = 512;  // S of M tile t, buffer f: columns 128 t + 64 f; O of tile t: 256 + 128 t
constexpr long long kDrainCycles = 200000000LL;
constexpr float P_TOP = 15.9f, P_MOVE = 8.f, P_UP = P_TOP - P_MOVE, P_UP_SINK = P_TOP - 2.f, Z_TOP = 116.f;  // log2 units
constexpr float L_SCALE = 0x1p-20f, L_LOG2 = -20.f;  // row sums are kept times 2^-20, so that 2^15 / vs does not overflow
constexpr int SOFTMAX_REGS = 168, CONVERT_REGS = 96, MMA_REGS = 80;
constexpr float kTinyScale = 0x1p-100f;
// With caches of up to so many blocks a CTA takes a whole item, however few there are: equal runs for all SMs would cost more in
// parts to write and join than they gain (whole / runs, us: 96 items of 12 tiles 20 / 34; 4 items of 16 22 / 30, 32 of them 23 / 25,
// 128 24 / 41; 2 items of 23 tiles x 128 dims 25 / 54, 32 of them x 64 dims 22 / 24; 1 item of 7 tiles 10 / 16).
constexpr int WHOLE_TILES = 24;

template <int D>
struct Smem {
  static constexpr int QT = 128 * D * 2;   // bytes of one M tile of q
  static constexpr int KT = KEYS * D * 2;  // of a converted K or V tile
  static constexpr int K = 2 * QT, V = K + ST * KT, BYTES = V + ST * KT;
};

struct Args {
  const uint16_t* q;
  long long sq_b, sq_t, sq_h;
  const int8_t *kc, *vc;
  const float *ks, *vs;
  const int *lens, *counts;
  int B, n, G, H, C, causal, rows, ctas;
  int items;  // > 0: items of a head, and a CTA for each item (no runs, nothing to join)
  float scale_log2;
  uint16_t* out;
  long long so_b, so_t, so_h;
  float* part_o;     // [2 ctas][ROWS][D]
  float2* part_ml;   // [2 ctas][ROWS]
  float* lse;        // [B][H][rows] minus log2 of the row's sum, or null
  float* w;
  const float* w_in;
};

struct Plan {
  int rows, ctas;
  bool whole;  // a CTA for each item
  long long ml_off, lse_off, bytes;
};
static Plan make_plan(int B, int n, int Hq, int H, int D, int C, bool weights, int sms) {
  Plan p;
  p.whole = C / BLK <= WHOLE_TILES;
  p.rows = n * (Hq / H);
  p.ctas = sms;
  auto up = [](long long x) { return (x + 255) / 256 * 256; };
  p.ml_off = p.whole ? 0 : up(2LL * sms * ROWS * D * 4);
  p.lse_off = p.ml_off + (p.whole ? 0 : up(2LL * sms * ROWS * 8));
  p.bytes = p.lse_off + (weights ? up((long long)B * H * p.rows * 4) : 0);
  return p;
}

// Key tiles of rows [ROWS qt, ROWS qt + ROWS) of one head: up to the last key that the last of them sees.
__device__ __forceinline__ int item_tiles(const Args& a, const Seq& s, int qt) {
  const int last = min((qt * ROWS + ROWS - 1) / a.G, s.cnt - 1);
  return ((a.causal ? s.len + last + 1 : s.len + s.cnt) + KEYS - 1) / KEYS;
}
__device__ __forceinline__ int seq_items(const Args& a, const Seq& s) { return (s.cnt * a.G + ROWS - 1) / ROWS; }

// The list of all tiles, sequence by sequence, head by head, item by item: pre[b] first tile of sequence b; and the run.
__device__ __forceinline__ int tile_list(const Args& a, int* pre, int* scratch) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + (int)blockDim.x - 1) / (int)blockDim.x, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  int sum = 0;
  for (int b = b0; b < b1; b++) {
    const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C, blockIdx.x == 0 && blockIdx.y == 0);  // those without work are looked at here only
    int t = 0;
    const int items = seq_items(a, s);
    if (a.causal)
      for (int q = 0; q < items; q++) t += item_tiles(a, s, q);
    else if (items)
      t = items * item_tiles(a, s, 0);
    pre[b] = t * a.H;
    sum += t * a.H;
  }
  int inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  int at = inc - sum;
  for (int i = 0; i < warp; i++) at += scratch[i];
  for (int b = b0; b < b1; b++) {
    const int t = pre[b];
    pre[b] = at;
    at += t;
  }
  if (tid == (int)blockDim.x - 1) pre[a.B] = at;
  __syncthreads();
  const int run = max((pre[a.B] + a.ctas - 1) / a.ctas, 1);
  return run;
}

// A CTA's share of one item: rows r0 .. of (b, h), key tiles [ta, tb) of `tiles`.
struct Seg {
  int b, h, r0, ta, tb, tiles;
  Seq s;
};
__device__ __forceinline__ Seg segment(const Args& a, const int* pre, int u, int u_end) {
  Seg g;
  if (a.items > 0) {  // CTA = item
    const int bh = blockIdx.x / a.items, qt = blockIdx.x % a.items;
    g.b = bh / a.H, g.h = bh % a.H, g.r0 = qt * ROWS, g.ta = 0;
    g.s = seq_of(a.lens, a.counts, g.b, a.n, a.C);
    g.tb = g.tiles = g.r0 < g.s.cnt * a.G ? item_tiles(a, g.s, qt) : 0;
    return g;
  }
  g.b = split::find_seq(pre, a.B, u);
  g.s = seq_of(a.lens, a.counts, g.b, a.n, a.C);
  const int head = (pre[g.b + 1] - pre[g.b]) / a.H;  // tiles of one head
  g.h = (u - pre[g.b]) / head;
  int at = (u - pre[g.b]) % head, qt = 0;
  for (g.tiles = item_tiles(a, g.s, 0); at >= g.tiles; g.tiles = item_tiles(a, g.s, ++qt)) at -= g.tiles;
  g.r0 = qt * ROWS, g.ta = at, g.tb = min(g.tiles, at + (u_end - u));
  return g;
}

__device__ __forceinline__ uint32_t sub_bf2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Two codes (bytes lo, lo + 1 of x) as bf16 or f16; x of the latter with its bytes' top bits flipped.
template <int SEL, bool F16>
__device__ __forceinline__ uint32_t two_codes(uint32_t x) {
  if (F16) return split::hsub2(__byte_perm(x, 0x64646464u, SEL), split::H1152);
  const uint32_t w = __byte_perm(x, 0x43434343u, SEL);
  return sub_bf2(w & 0xff7fff7fu, w & 0xff80ff80u);
}
// 16 codes of a row: dims 16 p .. of row `row` into operand chunks 2p, 2p + 1 (CR rows each).
template <int CR, bool F16>
__device__ __forceinline__ void store_codes(uint8_t* tile, int row, int p, uint4 c) {
  uint8_t* at = tile + (2 * p * CR + row) * 16;
  if (F16) c.x ^= 0x80808080u, c.y ^= 0x80808080u, c.z ^= 0x80808080u, c.w ^= 0x80808080u;
  auto lo = [](uint32_t x) { return two_codes<0x4140, F16>(x); };
  auto hi = [](uint32_t x) { return two_codes<0x4342, F16>(x); };
  *reinterpret_cast<uint4*>(at) = make_uint4(lo(c.x), hi(c.x), lo(c.y), hi(c.y));
  *reinterpret_cast<uint4*>(at + CR * 16) = make_uint4(lo(c.z), hi(c.z), lo(c.w), hi(c.w));
}
// Two f16, numbers beyond its range as the largest one (they meet zeros only).
__device__ __forceinline__ uint32_t pack_h2_finite(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// The address of q row r of (b, h).
__device__ __forceinline__ const uint16_t* q_row(const Args& a, int b, int h, int r) {
  return a.q + b * a.sq_b + r / a.G * a.sq_t + (size_t)(h * a.G + r % a.G) * a.sq_h;
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1) attn_kv8_tc_kernel(Args a) {
  using L = Smem<D>;
  extern __shared__ __align__(1024) uint8_t sm[];
  __shared__ int pre[MAXB + 1], scratch[THREADS / 32];
  __shared__ __align__(8) uint64_t bars[2 + 2 * ST + 4 + 4 + 4 + 2];
  __shared__ uint32_t tmem_slot;
  __shared__ int sh_abort;
  volatile int* abort_flag = &sh_abort;
  uint64_t *q_full = bars, *kv_full = bars + 2, *kv_empty = kv_full + ST;
  uint64_t *s_full = kv_empty + ST, *p_full = s_full + 4, *o_full = p_full + 4, *o_empty = o_full + 2, *drain = o_empty + 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&q_full[0], 4);
    mbar_init(&q_full[1], 4);
    for (int i = 0; i < ST; i++) mbar_init(&kv_full[i], 4), mbar_init(&kv_empty[i], 2);
    for (int i = 0; i < 4; i++) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 4);
    for (int i = 0; i < 2; i++) mbar_init(&o_full[i], 1), mbar_init(&o_empty[i], 4);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
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
  int u_begin = 0, u_end;  // this CTA's run of tiles
  if (a.items > 0) {
    u_end = segment(a, pre, 0, 0).tiles;
  } else {
    const int run = tile_list(a, pre, scratch), total = pre[a.B];
    u_begin = (int)min((long long)blockIdx.x * run, (long long)total);
    u_end = (int)min((long long)u_begin + run, (long long)total);
  }
  // a wait of the whole warp: every lane gives up when one does
  auto wait = [&](uint64_t* bar, int parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, ST_KV8_WAIT)) != 0;
  };

  // registers by role: 512 threads are launched with 128 each; the softmax holds 64 scores (2048-token chunk 284 us with this
  // split, 307 with 128 for all; the compiler, which sees 128, still spills 32 bytes a thread)
  static_assert(2 * SOFTMAX_REGS + CONVERT_REGS + MMA_REGS <= 4 * 128, "the split must come out of the launch's registers");
  if (warp >= 12) {
    set_regs_down<MMA_REGS>();  // one instruction for the whole warp group
    // ---------------- MMA issuer of M tile t, one warp each (one thread for both tiles: 435 against 335 us for the 2048-token
    // chunk).  The whole warp walks the loop, one lane issues.  j: key tiles of all segments; js: of those in which t had rows
    const int t = warp - 12, end = t < 2 ? u_end : u_begin;  // warps 14 and 15 are idle
    const uint32_t leader = elect_one();
    constexpr uint32_t IDESC_S = idesc_bf16(128, KEYS), IDESC_O = idesc_f16(128, D) | (1u << 16);  // V MN-major
    const uint64_t dq = sdesc_noswz(smem_u32(sm) + t * L::QT, 2048, 128), dk = sdesc_noswz(smem_u32(sm + L::K), 1024, 128);
    const uint64_t dv = sdesc_noswz(smem_u32(sm + L::V), 128, 1024);
    const uint32_t t_s = tmem + 128 * t, t_o = tmem + 256 + 128 * t;
    bool ok = true;
    int st = 0, ph = 0, js = 0, so = 0;  // stage and phase of the next tile's operands; tiles, segments in which t had rows
    auto next = [](int& x, int& y) { if (++x == ST) x = 0, y ^= 1; };
    for (int u = u_begin; u < end && ok;) {
      const Seg g = segment(a, pre, u, u_end);
      const int nt = g.tb - g.ta;
      u += nt;
      if (g.r0 + 128 * t >= g.s.cnt * a.G) {  // no rows in this M tile: only the barriers
        for (int i = 0; i < nt && ok; i++, next(st, ph)) {
          ok = wait(&kv_full[st], ph);
          mbar_arrive_if(&kv_empty[st], leader != 0);
        }
        continue;
      }
      auto issue_s = [&](int i) {  // S_i of the segment; its operands' stage is st
        if (!wait(&kv_full[st], ph)) return false;
        tc_fence_after();
        const int f = (js + i) & 1;
        if (leader) {
          const uint64_t b = dk + st * (L::KT >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; k++) umma_f16(t_s + 64 * f, dq + k * (4096 >> 4), b + k * (2048 >> 4), IDESC_S, k > 0 ? 1u : 0u);
          umma_commit(&s_full[2 * t + f]);
        }
        __syncwarp();
        next(st, ph);
        return true;
      };
      int sv = st;  // stage of tile i
      ok = wait(&q_full[t], so & 1) && issue_s(0);
      for (int i = 0; i < nt && ok; i++, sv = sv + 1 == ST ? 0 : sv + 1) {
        const int f = (js + i) & 1;
        ok = (i + 1 == nt || issue_s(i + 1)) && (i > 0 || so == 0 || wait(&o_empty[t], (so - 1) & 1)) &&
             wait(&p_full[2 * t + f], ((js + i) >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint64_t b = dv + sv * (L::KT >> 4);
#pragma unroll
          for (int k = 0; k < KEYS / 16; k++) umma_f16_ts(t_o, t_s + 64 * f + k * 8, b + k * (256 >> 4), IDESC_O, i > 0 || k > 0 ? 1u : 0u);
          umma_commit(&kv_empty[sv]);
          if (i == nt - 1) umma_commit(&o_full[t]);
        }
        __syncwarp();
      }
      js += nt, so++;
    }
    if (leader && t < 2) {
      umma_commit(&drain[t]);
      mbar_wait_drain(&drain[t], 0, kDrainCycles);
    }
  } else if (warp >= 8) {
    set_regs_down<CONVERT_REGS>();
    // ---------------- converters: warp w rows 16 w .. of a block, 8 lanes = 8 rows of one 16-byte piece.  K's and V's codes of
    // the next tile are fetched as soon as this tile's are out of the registers
    constexpr int PER = D / 32;  // pieces of a K or V block that a lane takes
    const int w = warp - 8;
    bool ok = true;
    int j = 0;
    for (int u = u_begin; u < u_end && ok;) {
      const Seg g = segment(a, pre, u, u_end);
      const int nt = g.tb - g.ta;
      u += nt;
      const size_t bh = (size_t)g.b * a.H + g.h;
      const int8_t *kp = a.kc + (bh * a.C + (size_t)g.ta * KEYS) * D, *vp = a.vc + (bh * a.C + (size_t)g.ta * KEYS) * D;
      const float* vsp = a.vs + bh * (a.C / BLK) + g.ta;
      const int row = 16 * w + (lane & 7), piece = lane >> 3;
      uint4 kr[PER], vr[PER];
      float vs;
      auto fetch = [&](uint4 (&to)[PER], const int8_t* from) {
#pragma unroll
        for (int x = 0; x < PER; x++)
          to[x] = *reinterpret_cast<const uint4*>(from + (row + 8 * (x & 1)) * D + 16 * (piece + 4 * (x >> 1)));
      };
      fetch(kr, kp);
      fetch(vr, vp);
      vs = vsp[0];
      for (int i = 0; i < nt; i++, j++) {
        const int st = j % ST;
        if (j >= ST) ok = wait(&kv_empty[st], (j / ST - 1) & 1);
        if (!ok) break;
        kp += KEYS * D, vp += KEYS * D;
#pragma unroll
        for (int x = 0; x < PER; x++) store_codes<KEYS, false>(sm + L::K + st * L::KT, row + 8 * (x & 1), piece + 4 * (x >> 1), kr[x]);
        if (i + 1 < nt) fetch(kr, kp);
#pragma unroll
        for (int x = 0; x < PER; x++)
          store_codes<KEYS, true>(sm + L::V + st * L::KT, row + 8 * (x & 1), piece + 4 * (x >> 1), vs < kTinyScale ? make_uint4(0, 0, 0, 0) : vr[x]);
        if (i + 1 < nt) fetch(vr, vp), vs = vsp[i + 1];
        fence_proxy_async_smem();
        __syncwarp();
        mbar_arrive_if(&kv_full[st], lane == 0);
      }
    }
  } else {
    set_regs_up<SOFTMAX_REGS>();
    // ---------------- softmax of M tile t: thread = row.  It brings in its row of q itself
    const int t = warp >> 2;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16, t_o = tmem + 256 + 128 * t + lane_off;
    bool ok = true;
    int j = 0, js = 0, so = 0;
    auto load_q = [&](const Seg& g) {  // every product with the q before it is done: its last scores have been read
      const int r = (warp & 3) * 32 + lane, row = g.r0 + 128 * t + r;
      if (g.r0 + 128 * t >= g.s.cnt * a.G) return;
      const uint16_t* src = q_row(a, g.b, g.h, min(row, g.s.cnt * a.G - 1));  // rows past the last are copies of it
      uint8_t* dst = sm + t * L::QT + r * 16;
#pragma unroll
      for (int c0 = 0; c0 < D / 8; c0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int c = 0; c < 8; c++) v[c] = *reinterpret_cast<const uint4*>(src + 8 * (c0 + c));
#pragma unroll
        for (int c = 0; c < 8; c++) *reinterpret_cast<uint4*>(dst + (c0 + c) * 2048) = v[c];
      }
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_if(&q_full[t], lane == 0);
    };
    Seg g;
    if (u_begin < u_end) load_q(g = segment(a, pre, u_begin, u_end));
    for (int u = u_begin; u < u_end && ok;) {
      const int nt = g.tb - g.ta, row = g.r0 + 128 * t + (warp & 3) * 32 + lane, valid = g.s.cnt * a.G;
      const bool first = u == u_begin;
      u += nt;
      if (g.r0 + 128 * t >= valid) {  // no rows: the MMA issuer skips this M tile too
        j += nt;
        if (u < u_end) load_q(g = segment(a, pre, u, u_end));
        continue;
      }
      const size_t bh = (size_t)g.b * a.H + g.h;
      const float *ksp = a.ks + bh * (a.C / BLK) + g.ta, *vsp = a.vs + bh * (a.C / BLK) + g.ta;
      const int lim = a.causal ? g.s.len + min(row / a.G, g.s.cnt - 1) + 1 : g.s.len + g.s.cnt;
      // the fewest keys that a row of this warp sees: tiles up to there need no mask
      const int lim_min = __reduce_min_sync(0xffffffffu, lim);
      float m = -INFINITY, l = 0.f;
      // of the tile: K's scale times the softmax scale, log2 and inverse (times L_SCALE) of V's scale (the approximations err by
      // 2^-22, both in the sum and in O); the next tile's are worked out while this one's scores arrive
      // and how far terms may be above m
      float c, lvs, ivs, top, ks_next = ksp[0], vs_next = vsp[0], c_next, lvs_next, ivs_next, top_next;
      auto next_scales = [&](int i) {
        const bool none = vs_next < kTinyScale;  // the converters made V zero
        const float v = none ? 1.f : vs_next;
        c_next = ks_next * a.scale_log2, lvs_next = __log2f(v), ivs_next = __frcp_rn(v) * L_SCALE, top_next = none ? Z_TOP : P_TOP;
        if (i + 1 < nt) ks_next = ksp[i + 1], vs_next = vsp[i + 1];
      };
      next_scales(0);
      auto announce = [&](int f) {  // P in buffer f is complete
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_if(&p_full[2 * t + f], lane == 0);
      };
      for (int i = 0; i < nt; i++) {
        const int f = (js + i) & 1, key0 = (g.ta + i) * KEYS;
        const uint32_t t_s = tmem + 128 * t + 64 * f + lane_off;
        c = c_next, lvs = lvs_next, ivs = ivs_next, top = top_next;
        uint32_t r0[32], r1[32];
        float mx, sum;
        auto top32 = [&](const uint32_t (&r)[32]) {
          float x[11];
#pragma unroll
          for (int e = 0; e < 10; e++) x[e] = max3f(__uint_as_float(r[3 * e]), __uint_as_float(r[3 * e + 1]), __uint_as_float(r[3 * e + 2]));
          x[10] = fmaxf(__uint_as_float(r[30]), __uint_as_float(r[31]));
#pragma unroll
          for (int e = 0; e < 3; e++) x[e] = max3f(x[3 * e], x[3 * e + 1], x[3 * e + 2]);
          return max3f(max3f(x[0], x[1], x[2]), x[9], x[10]);
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
            pk[e] = pack_h2_finite(p0, p1);
          }
          tmem_st16(t_s + at, pk);
          float lo, hi;
          f2_unpack(f2_add(sum2[0], sum2[1]), lo, hi);
          return lo + hi;
        };
        ok = wait(&s_full[2 * t + f], ((js + i) >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        tmem_ld32(t_s, r0);
        next_scales(i + 1);
        tmem_ld_wait();
        tmem_ld32(t_s + 32, r1);
        // a tile that every row sees whole, once a row has a maximum: P with the maximum so far, while the second half of
        // the scores arrives and the new maximum is found beside the exponentials; they stand unless it grew too far
        const bool edge = key0 + KEYS > lim_min;
        bool again = i == 0 || edge;
        if (!again) {
          sum = exps(r0, 0, m);
          const float ma = top32(r0);
          tmem_ld_wait();
          sum += exps(r1, 16, m);
          mx = fmaf(fmaxf(ma, top32(r1)), c, lvs);
          again = __any_sync(0xffffffffu, mx > m + top);
        }
        if (again) {
          tmem_ld_wait();
          const int left = lim - key0;  // keys of the tile that the row sees
          if (edge) {
#pragma unroll
            for (int e = 0; e < 32; e++) {
              if (e >= left) r0[e] = 0xff800000u;
              if (32 + e >= left) r1[e] = 0xff800000u;
            }
          }
          mx = left > 0 ? fmaf(fmaxf(top32(r0), top32(r1)), c, lvs) : -INFINITY;
          const bool need = mx > m + top;
          const float up = top - P_MOVE;
          const float mn = i == 0 ? mx - up : need ? mx - (mx > m + (P_TOP + 12.f) ? fmaxf(up, P_UP_SINK) : up) : m;
          if (i > 0 && __any_sync(0xffffffffu, need)) {  // O through registers (warp-collective)
            // O must hold every product up to tile i - 1; the barrier's next arrival, ST tiles on, needs P of this row
            ok = wait(&kv_empty[(j + i - 1) % ST], ((j + i - 1) / ST) & 1);
            if (!ok) break;
            tc_fence_after();
            const float half = need ? ex2_approx(0.5f * (m - mn)) : 1.f, alpha = half * half;
            l = l * half * half;  // what zero blocks put there may be as large as alpha is small
#pragma unroll
            for (int x = 0; x < D / 16; x++) {
              uint32_t r[16];
              tmem_ld16(t_o + x * 16, r);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; e++) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
              tmem_st16(t_o + x * 16, r);
            }
          }
          m = mn;
          // a row that sees nothing of the tile takes no part in its scales, which may be NaN; scores out of sight are -inf,
          // and -inf * 0 of a zero scale must not be NaN
          const float mu = m == -INFINITY ? 0.f : m;
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
          sum = exps(r0, 0, mu) + exps(r1, 16, mu);
          if (i == 0) {  // a tile whose other keys add up to a twentieth of its largest one
            const bool sink = sum < 1.05f * exp2f(P_UP);
            if (__any_sync(0xffffffffu, sink)) {
              m -= sink ? P_UP_SINK - P_UP : 0.f;
              const float ms = m == -INFINITY ? 0.f : m;
              sum = exps(r0, 0, ms) + exps(r1, 16, ms);
            }
          }
        }
        l += sum * ivs;
        announce(f);
      }
      if (!ok) break;
      const Seg done = g;
      if (u < u_end) load_q(g = segment(a, pre, u, u_end));  // the next item's products start before this one's O is stored
      ok = wait(&o_full[t], so & 1);
      if (!ok) break;
      tc_fence_after();
      const bool whole = done.ta == 0 && done.tb == done.tiles;
      const float inv = L_SCALE / l;
      const int at = row - done.r0;
      const size_t slot = (2 * (size_t)blockIdx.x + (first ? 0 : 1)) * ROWS + at;
      uint16_t* op = a.out + done.b * a.so_b + row / a.G * a.so_t + (size_t)(done.h * a.G + row % a.G) * a.so_h;
#pragma unroll
      for (int x16 = 0; x16 < D / 16; x16++) {
        uint32_t r[16];
        tmem_ld16(t_o + x16 * 16, r);
        tmem_ld_wait();
        if (row < valid) {
          if (whole) {
#pragma unroll
            for (int e = 0; e < 16; e += 8)
              *reinterpret_cast<uint4*>(op + 16 * x16 + e) =
                  make_uint4(pack_bf2(__uint_as_float(r[e]) * inv, __uint_as_float(r[e + 1]) * inv),
                             pack_bf2(__uint_as_float(r[e + 2]) * inv, __uint_as_float(r[e + 3]) * inv),
                             pack_bf2(__uint_as_float(r[e + 4]) * inv, __uint_as_float(r[e + 5]) * inv),
                             pack_bf2(__uint_as_float(r[e + 6]) * inv, __uint_as_float(r[e + 7]) * inv));
          } else {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<uint4*>(a.part_o + slot * D + 16 * x16 + e) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
          }
        }
      }
      if (row < valid) {
        if (!whole) a.part_ml[slot] = make_float2(m, l);
        else if (a.lse) a.lse[bh * a.rows + row] = -(m - L_LOG2 + log2f(l));
      }
      tc_fence_before();
      __syncwarp();
      mbar_arrive_if(&o_empty[t], lane == 0);
      j += nt, js += nt, so++;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Merges the parts of an item, in the CTAs' order.  blockIdx.x = c: the item that CTA c left unfinished, if its first part is
// in c's run; blockIdx.y: 16 of its rows; thread = 4 dims of a row.
template <int D>
__global__ void __launch_bounds__(128) attn_kv8_tc_join_kernel(Args a) {
  __shared__ int pre[MAXB + 1], scratch[4];
  constexpr int PER = 128 * 4 / D;
  griddep_wait();
  griddep_launch();
  const int run = tile_list(a, pre, scratch), total = pre[a.B];
  const long long bound = ((long long)blockIdx.x + 1) * run;  // first tile of the next CTA's run
  if (bound >= total) return;
  const Seg g = segment(a, pre, (int)bound, total);
  const int u0 = (int)bound - g.ta, c0 = u0 / run, c1 = (u0 + g.tiles - 1) / run;
  if (g.ta == 0 || c0 != (int)blockIdx.x) return;
  const size_t first = 2 * (size_t)c0 + (u0 == c0 * run ? 0 : 1);
  const int d = threadIdx.x % (D / 4) * 4;
  const size_t bh = (size_t)g.b * a.H + g.h;
  for (int x = threadIdx.x / (D / 4); x < 16; x += PER) {
    const int at = blockIdx.y * 16 + x, row = g.r0 + at;
    if (row >= g.s.cnt * a.G) break;
    float mx = -INFINITY;
    for (int c = c0; c <= c1; c++) mx = fmaxf(mx, a.part_ml[(c == c0 ? first : 2 * (size_t)c) * ROWS + at].x);
    float sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int c = c0; c <= c1; c++) {
      const size_t p = (c == c0 ? first : 2 * (size_t)c) * ROWS + at;
      const float2 ml = a.part_ml[p];
      const float4 o = *reinterpret_cast<const float4*>(a.part_o + p * D + d);
      const float half = ml.x == -INFINITY ? 0.f : ex2_approx(0.5f * (ml.x - mx)), f = half * half;
      sum += ml.y * half * half, v.x += o.x * f, v.y += o.y * f, v.z += o.z * f, v.w += o.w * f;
    }
    const float inv = L_SCALE / sum;
    uint16_t* op = a.out + g.b * a.so_b + row / a.G * a.so_t + (size_t)(g.h * a.G + row % a.G) * a.so_h + d;
    *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf2(v.x * inv, v.y * inv), pack_bf2(v.z * inv, v.w * inv));
    if (d == 0 && a.lse) a.lse[bh * a.rows + row] = -(mx - L_LOG2 + log2f(sum));
  }
}

// ---------------------------------------------------------------- weights
// weights[b][h][j] = (j < len ? weights_in : 0) + sum over rows of 2^(s - lse): S^T = K Q^T with keys as the M dimension, so
// a thread owns a key and adds up along its TMEM lane: no atomics, one order.  CTA = 128 keys of one (sequence, head);
// rows 128 at a time:
//   warps 0-3, 4-7   rows 0-63 / 64-127 of the row tile, thread = key;
//   warps 8-11       K's codes -> the A operand once; q rows and lse of each row tile, ST tiles in flight;
//   warp 12          tcgen05.mma into two S buffers.
// Bound: MUFU, one ex2 a score (730 x 730 x 32 heads: 22 us, most of it on the SMs that have two of the 192 CTAs).
constexpr int WK = 128, WR = 128, WTHREADS = 13 * 32;
template <int D>
struct WSmem {
  static constexpr int ST = D == 64 ? 4 : 2;  // row tiles in flight; two CTAs share an SM
  static constexpr int K = 0, Q = WK * D * 2, QT = WR * D * 2, BYTES = Q + ST * QT;
};
template <int D>
__global__ void __launch_bounds__(WTHREADS, 2) kv8_weights_tc_kernel(Args a) {
  using L = WSmem<D>;
  extern __shared__ __align__(1024) uint8_t sm[];
  constexpr int ST = L::ST;
  __shared__ __align__(16) float sh_lse[ST][WR], half_sum[WK];
  __shared__ __align__(8) uint64_t bars[2 * ST + 2 + 2 + 1];
  __shared__ uint32_t tmem_slot;
  __shared__ int sh_abort;
  volatile int* abort_flag = &sh_abort;
  uint64_t *q_full = bars, *q_empty = bars + ST, *s_full = q_empty + ST, *s_empty = s_full + 2, *drain = s_empty + 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kt = (a.C + WK - 1) / WK, key0 = blockIdx.x % kt * WK;
  const size_t bh = blockIdx.x / kt;
  const int h = (int)(bh % a.H), b = (int)(bh / a.H);
  griddep_wait();
  const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C);
  const int T = s.len + s.cnt, rows = s.cnt * a.G;
  if (key0 >= T) return;
  // the first row that sees a key of this CTA, down to a whole tile
  const int first = a.causal ? max(key0 - s.len, 0) * a.G / WR : 0, nt = (rows + WR - 1) / WR - first;
  if (tid == 0) {
    for (int i = 0; i < ST; i++) mbar_init(&q_full[i], 4), mbar_init(&q_empty[i], 8);
    for (int i = 0; i < 2; i++) mbar_init(&s_full[i], 1), mbar_init(&s_empty[i], 8);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch();  // not before the tensor memory is allocated: the next kernel's CTAs may take theirs while they wait
  const uint32_t tmem = tmem_slot;
  float acc = 0.f;
  bool ok = true;
  // a wait of the whole warp: every lane gives up when one does
  auto wait = [&](uint64_t* bar, int parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, ST_KV8_WAIT)) != 0;
  };
  if (warp == 12) {
    const uint32_t leader = elect_one();
    const uint64_t dk = sdesc_noswz(smem_u32(sm + L::K), 2048, 128), dq = sdesc_noswz(smem_u32(sm + L::Q), 2048, 128);
    for (int i = 0; i < nt; i++) {
      const int f = i & 1, st = i % ST;
      ok = wait(&q_full[st], (i / ST) & 1) && (i < 2 || wait(&s_empty[f], ((i >> 1) - 1) & 1));
      if (!ok) break;
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int k = 0; k < D / 16; k++)
          umma_f16(tmem + 128 * f, dk + k * (4096 >> 4), dq + st * (L::QT >> 4) + k * (4096 >> 4), idesc_bf16(WK, WR), k > 0 ? 1u : 0u);
        umma_commit(&s_full[f]);
      }
      __syncwarp();
    }
    if (leader) {
      umma_commit(drain);
      mbar_wait_drain(drain, 0, kDrainCycles);
    }
  } else if (warp >= 8) {
    const int w = warp - 8, ct = tid - 256;
    const int8_t* kp = a.kc + bh * a.C * D;
    // a warp's copies take 32 bytes of 16 rows at a time: whole sectors, and two lanes to a bank at most
    auto fetch = [&](int i) {
      const int st = i % ST, r0 = (first + i) * WR;
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const int r = 32 * w + 16 * x + (lane >> 1);
        const uint16_t* src = q_row(a, b, h, min(r0 + r, rows - 1)) + 8 * (lane & 1);
        const uint32_t dst = smem_u32(sm + L::Q + st * L::QT + ((lane & 1) * WR + r) * 16);
#pragma unroll
        for (int c = 0; c < D / 16; c++)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 2 * c * WR * 16), "l"(src + 16 * c) : "memory");
      }
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&sh_lse[st][ct])), "l"(a.lse + bh * a.rows + min(r0 + ct, rows - 1))
                   : "memory");
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    for (int i = 0; i < ST - 1; i++) {
      if (i < nt) fetch(i);
      commit();
    }
    for (int x = 0; x < 4 * (D / 64); x++) {  // warp w rows 32 w ..; slots behind the cache's last one are zero
      const int row = 32 * w + 8 * (x & 3) + (lane & 7), p = (lane >> 3) + 4 * (x >> 2);
      uint4 c = make_uint4(0, 0, 0, 0);
      if (key0 + row < a.C) c = *reinterpret_cast<const uint4*>(kp + (size_t)(key0 + row) * D + 16 * p);
      store_codes<WK, false>(sm + L::K, row, p, c);
    }
    for (int i = 0; i < nt; i++) {
      asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_if(&q_full[i % ST], lane == 0);
      const int n = i + ST - 1;  // the next tile to bring in; its stage was tile i - 1's, free when both halves have read its lse
      if (n < nt) {
        if (i > 0) ok = wait(&q_empty[n % ST], ((i - 1) / ST) & 1);
        if (!ok) break;
        fetch(n);
      }
      commit();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    const int half = warp >> 2, key = key0 + (warp & 3) * 32 + lane;
    const uint32_t t_s = tmem + 64 * half + ((uint32_t)((warp & 3) * 32) << 16);
    const float c = key < T ? a.ks[bh * (a.C / BLK) + key / BLK] * a.scale_log2 : 0.f;
    const int r_min = a.causal ? max(key - s.len, 0) * a.G : 0;  // rows before it do not see this key
    const int warp_max = __reduce_max_sync(0xffffffffu, r_min);
    unsigned long long acc2[2] = {0ull, 0ull};
    const unsigned long long c2 = f2_pack(c, c);
    for (int i = 0; i < nt; i++) {
      const int f = i & 1, st = i % ST;
      ok = wait(&q_full[st], (i / ST) & 1) && wait(&s_full[f], (i >> 1) & 1);  // lse, scores
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        uint32_t x[32];
        tmem_ld32(t_s + 128 * f + 32 * hf, x);
        tmem_ld_wait();
        if (hf == 1) {
          tc_fence_before();
          __syncwarp();
          mbar_arrive_if(&s_empty[f], lane == 0);
        }
        const int r0 = (first + i) * WR + 64 * half + 32 * hf;
        const bool edge = r0 < warp_max || r0 + 32 > rows;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 z = *reinterpret_cast<const float4*>(&sh_lse[st][64 * half + 32 * hf + e]);
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const unsigned long long lz = k ? f2_pack(z.z, z.w) : f2_pack(z.x, z.y);
            const unsigned long long y = f2_fma(f2_pack(__uint_as_float(x[e + 2 * k]), __uint_as_float(x[e + 2 * k + 1])), c2, lz);
            float y0, y1;
            f2_unpack(y, y0, y1);
            y0 = ex2_approx(y0), y1 = ex2_approx(y1);
            if (edge) {
              const int ra = r0 + e + 2 * k;
              if (ra < r_min || ra >= rows) y0 = 0.f;
              if (ra + 1 < r_min || ra + 1 >= rows) y1 = 0.f;
            }
            acc2[k] = f2_add(acc2[k], f2_pack(y0, y1));
          }
        }
      }
      __syncwarp();
      mbar_arrive_if(&q_empty[st], lane == 0);
    }
    float lo, hi;
    f2_unpack(f2_add(acc2[0], acc2[1]), lo, hi);
    acc = lo + hi;
    if (half == 1) half_sum[key - key0] = acc;
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp < 4) {
    const int key = key0 + tid;
    if (key < T) {
      const size_t at = bh * a.C + key;
      a.w[at] = (a.w_in && key < s.len ? a.w_in[at] : 0.f) + (acc + half_sum[tid]);
    }
  }
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

template <int D>
static int launch(cudaStream_t st, const Args& a) {
  int rc = smem_attr_once((const void*)attn_kv8_tc_kernel<D>, Smem<D>::BYTES, "vt_attn_kv8");
  if (!rc) rc = smem_attr_once((const void*)kv8_weights_tc_kernel<D>, WSmem<D>::BYTES, "vt_attn_kv8");
  if (rc) return rc;
  if (a.items > 0) {
    launch_k(attn_kv8_tc_kernel<D>, (unsigned)(a.B * a.H * a.items), THREADS, Smem<D>::BYTES, st, a);
  } else {
    launch_k(attn_kv8_tc_kernel<D>, a.ctas, THREADS, Smem<D>::BYTES, st, a);
    launch_k(attn_kv8_tc_join_kernel<D>, dim3(a.ctas, ROWS / 16), 128, 0, st, a);
  }
  if (a.w) launch_k(kv8_weights_tc_kernel<D>, (unsigned)(a.B * a.H * ((a.C + WK - 1) / WK)), WTHREADS, WSmem<D>::BYTES, st, a);
  return check_launch("vt_attn_kv8");
}

}  // namespace tc
}  // namespace kv8
}  // namespace vt
