// Attention of a few rows over the 8-bit cache (one new token, a short question), bound by reading the cache once.
//
// A kv head's rows r = i * G + g (token i, query head h G + g of its group) share every key.  The keys of all heads and
// sequences form one list of tiles (KT keys of one head) that is cut into equal runs, one for each CTA, whatever
// the sequences' lengths: a head's keys may span CTAs, and a CTA may work on several heads.  Partial results
// (unnormalised O, row max, row sum) of heads that span CTAs are merged by attn_kv8_join_kernel, in order.
//
// CTA = 4 warps; each warp has its own ring of ST tiles in shared memory, filled by bulk copies (a tile of K codes and one
// of V codes, 4 KB each and contiguous in the cache), and works on every fourth tile of the CTA's run, so no barrier
// stands between tiles.  The products run on mma.sync (m16n8k16, f16): with at most 32 rows the 128 lanes of a tcgen05
// accumulator would stay mostly empty and every tile's codes would have to be written back to shared memory as 16-bit
// operands; here a code goes from shared memory through two byte permutes and a subtraction into a register of
// the operand.  S^T = K Q^T: keys are the M dimension (16 a step), rows the N dimension (8).
//   codes   byte b -> 0x6400 | (b ^ 0x80) = 1152 + code in f16, minus 1152: exact;
//   q       bf16 -> f16 after scaling each row by a power of two to max 2^15 .. 2^16 (f16 ends there): exact down to 2^-32
//           of the row's largest value, below that off by 2^-40 of it;
//   scores  fp32 accumulators times (row's power of two * scale * log2 e * the block's K scale): the scale is
//           applied to the exact sum of products of codes, so it costs one multiplication a score;
//   P       2^(s - m) in f16, with m 15 below the largest score so far, so that P uses f16's range up to 2^15: 11 bits down to 2^-29
//           of a row's largest weight, below that off by 2^-40 of it at most (the sum takes P before it is rounded; with
//           m at the largest score itself, keys 15 nats below a sink lost 0.5 % and 17.6 nats below it 17 %); S^T's
//           accumulator layout becomes the B operand of O^T = V^T P^T by movmatrix;
//   V^T     needs two keys of one dim in a register: four words of four keys are transposed by byte permutes.  Which
//           of a tile's keys is which row of the MMA is free, so lane t takes keys t, 4 + t, 8 + t, 12 + t: its reads are
//           free of bank conflicts (rows 64 B apart), and K's rows follow the same order;
//   O       a tile's product is accumulated on its own and added as O = O * alpha + vs * (P V): V's scale stays fp32.
// What bounds it: DRAM at long contexts (64 x 8 heads x 128 of 4k-8k slots, 818 MB: 139 us, 5.89 TB/s, issue slots 57 % busy; under
// the power cap, in loops of seconds, 159 us; three CTAs an SM with two stages each: 201 us), else the latency of one tile's chain and of the join.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {
namespace split {

constexpr int ST = 3, FEW_ROWS = 32;                // stages; rows of a kv head that this kernel takes
constexpr int TILE = 4096;                         // bytes of K (or V) codes in a tile
constexpr int RING = 2 * TILE * ST;                // a warp's ring
constexpr int MAXB = 2048;                         // sequences a call takes (their tile counts sit in shared memory)
constexpr int WARPS = 4;                           // of a CTA with a run of tiles
constexpr int MIN_RUN = WARPS;                     // tiles of a run at least
// Where a head has at most so many tiles, and there are at most four items for each SM, a CTA of eight warps takes a whole item:
// no parts, no second kernel, and the weights come from the same CTA (32-token question over 730: 10.0 us, against 8.4 in runs
// and 5.1 to join; one token 6.4 against 5.1 and 4.7; 12 x 32 heads of 800: 13.8 against 17.5 together; but 34 x 32 heads of
// 531 with weights 40.3 against 36.1).
constexpr int WHOLE_WARPS = 8, WHOLE_TILES = 16;
constexpr long long kDrainCycles = 200000000LL;
constexpr float P_UP = 15.f, P_SCALE = 0x1p15f;  // how far m is below the largest score (log2 units); O is kept divided by 2^15, see vc

struct Plan {       // fixed on the host from sizes alone
  int rows, nt, rg;   // rows n G of a kv head, rows / 8 of a row group, row groups
  int ctas;
  bool whole;         // a CTA for each item
  long long o_off, ml_off, full_off, s_off, bytes;  // workspace: partial O, their (m, l), (m, l) of every row, scores
};

__host__ __device__ inline int keys_per_tile(int D) { return TILE / D; }

static Plan make_plan(int B, int n, int Hq, int H, int D, int C, bool weights, int sms) {
  Plan p;
  p.rows = n * (Hq / H);
  // rows of a group: registers hold O [D][rows] of a warp (D rows / 32 a lane) beside q and P: 32 rows for D = 64,
  // 16 for D = 128
  p.nt = p.rows <= 8 ? 1 : (p.rows <= 16 || D == 128) ? 2 : 4;
  p.rg = (p.rows + 8 * p.nt - 1) / (8 * p.nt);
  p.ctas = 2 * sms;
  p.whole = C / keys_per_tile(D) <= WHOLE_TILES && (p.rg == 1 || !weights) && (long long)B * H * p.rg <= 4LL * sms;
  const long long slots = 2LL * p.ctas, gr = 8LL * p.nt;
  auto up = [](long long x) { return (x + 255) / 256 * 256; };
  p.o_off = 0;
  p.ml_off = p.o_off + (p.whole ? 0 : up(slots * gr * D * 4));
  p.full_off = p.ml_off + (p.whole ? 0 : up(slots * gr * 8));
  p.s_off = p.full_off + (p.whole ? 0 : up((long long)B * H * p.rg * gr * 8));
  p.bytes = p.s_off + (weights ? up((long long)B * H * p.rows * C * 4) : 0);
  return p;
}

struct Args {
  const uint16_t* q;
  long long sq_b, sq_t, sq_h;
  const int8_t *kc, *vc;
  const float *ks, *vs;
  const int *lens, *counts;
  int B, n, G, H, C, causal, rows, rg, ctas;
  float scale_log2;
  uint16_t* out;
  long long so_b, so_t, so_h;
  float* part_o;
  float2 *part_ml, *full_ml;
  float* scores;  // [B][H][rows][C], or null
  float* w;
  const float* w_in;
};

// Row groups of gr rows that a sequence's new tokens fill (rg of the plan at most).
__device__ __forceinline__ int row_groups(const Args& a, const Seq& s, int gr) { return (s.cnt * a.G + gr - 1) / gr; }
// First tile of each sequence in the list of all tiles, pre[0 .. B]; a sequence's tiles are those of its (head, row group)
// items one after another.  Every CTA computes it for itself.
__device__ __forceinline__ void tile_list(const Args& a, int kt, int gr, int* pre, int* warp_sum) {
  const int tid = threadIdx.x, nth = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + nth - 1) / nth, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  int sum = 0;
  for (int b = b0; b < b1; b++) {
    const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C, blockIdx.x == 0);  // those without work are looked at here only
    const int t = (s.len + s.cnt + kt - 1) / kt * a.H * row_groups(a, s, gr);
    pre[b] = t;
    sum += t;
  }
  int inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  int at = inc - sum;
  for (int i = 0; i < warp; i++) at += warp_sum[i];
  for (int b = b0; b < b1; b++) {
    const int t = pre[b];
    pre[b] = at;
    at += t;
  }
  if (tid == nth - 1) pre[a.B] = at;
  __syncthreads();
}
__device__ __forceinline__ int find_seq(const int* pre, int B, int u) {  // largest b with pre[b] <= u
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= u) lo = mid; else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ int run_of(int total, int ctas) { return max((total + ctas - 1) / ctas, MIN_RUN); }

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) { return __byte_perm(a, b, s); }
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr uint32_t H1152 = 0x64806480u;  // 1152 in both halves

template <int D, int NT, bool WHOLE>
__global__ void __launch_bounds__((WHOLE ? WHOLE_WARPS : WARPS) * 32, WHOLE ? 1 : 2) attn_kv8_split_kernel(Args a) {
  constexpr int WARPS = WHOLE ? WHOLE_WARPS : split::WARPS;
  constexpr int KT = TILE / D, GR = 8 * NT, WQ = D / 16, MT = KT / 16, OM = D / 16;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int pre[WHOLE ? 1 : MAXB + 1], warp_sum[WARPS];
  __shared__ __align__(8) uint64_t full[WARPS * ST];
  __shared__ float sh_m[WARPS][GR], sh_l[WARPS][GR], sh_lse[WHOLE ? GR : 1];
  __shared__ int sh_abort;
  volatile int* abort_flag = &sh_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = sm + warp * RING;
  uint64_t* bar = full + warp * ST;
  if (tid == 0) {
    for (int i = 0; i < WARPS * ST; i++) mbar_init(&full[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  griddep_wait();  // programmatic dependent launch: the previous kernel has completed
  griddep_launch();
  long long u_begin = 0;
  int total = 1, u_end = 1;  // this CTA's run of tiles (a whole item: one round)
  if (WHOLE) {
    __syncthreads();
  } else {
    tile_list(a, KT, GR, pre, warp_sum);  // its barriers also publish the mbarriers
    total = pre[a.B];
    const int run = run_of(total, a.ctas);
    u_begin = (long long)blockIdx.x * run;
    u_end = (int)min(u_begin + run, (long long)total);
  }
  int consumed = 0;  // tiles this warp has taken from its ring
  bool ok = true;
  for (int u = (int)min(u_begin, (long long)total); u < u_end;) {
    const int b = WHOLE ? blockIdx.x / (a.H * a.rg) : find_seq(pre, a.B, u);
    const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C);
    const int T = s.len + s.cnt, tiles = (T + KT - 1) / KT;
    const int rgs = WHOLE ? a.rg : row_groups(a, s, GR);
    const int item = WHOLE ? blockIdx.x % (a.H * rgs) : (u - pre[b]) / tiles, ta = WHOLE ? 0 : (u - pre[b]) % tiles;
    const int h = item / rgs, rg = item % rgs, r0 = rg * GR;
    // this CTA's tiles of the item: [ta, tb)
    const int tb = WHOLE ? (r0 < s.cnt * a.G ? tiles : 0) : min(tiles, ta + (u_end - u));
    const size_t bh = (size_t)b * a.H + h;
    const int8_t *kp = a.kc + bh * a.C * D, *vp = a.vc + bh * a.C * D;
    const float *ksp = a.ks + bh * (a.C / BLK), *vsp = a.vs + bh * (a.C / BLK);
    const int mine = tb - ta > warp ? (tb - ta - warp + WARPS - 1) / WARPS : 0;  // tiles ta + warp + WARPS j
    const int base = consumed;                        // tile j of them goes to slot (base + j) % ST
    auto load = [&](int j) {
      const int slot = (base + j) % ST;
      const size_t off = (size_t)(ta + warp + WARPS * j) * TILE;
      mbar_arrive_expect_tx(&bar[slot], 2 * TILE);
      bulk_load(ring + slot * 2 * TILE, kp + off, TILE, &bar[slot]);
      bulk_load(ring + slot * 2 * TILE + TILE, vp + off, TILE, &bar[slot]);
    };
    if (lane == 0 && ok)
      for (int j = 0; j < min(mine, ST); j++) load(j);
    float ks_next = 0.f, vs_next = 0.f;  // scales of the next tile
    if (mine > 0) ks_next = ksp[(ta + warp) * KT / BLK], vs_next = vsp[(ta + warp) * KT / BLK];
    // q of rows r0 + 8 nt + g, this lane's dims t D/4 .. as f16 pairs, scaled to a largest value of 2^15 .. 2^16
    uint32_t qf[NT][WQ][2];
    float cq[NT][2];  // scale of columns 2t, 2t + 1: scale * log2 e * the row's power of two
    int lim[NT][2];   // keys that they see
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int r = r0 + 8 * nt + g, i = r / a.G;
      uint32_t x[WQ][2];
      uint32_t top = 0;
      const uint16_t* qp = a.q + b * a.sq_b + i * a.sq_t + (size_t)(h * a.G + r % a.G) * a.sq_h + t * (D / 4);
#pragma unroll
      for (int w = 0; w < WQ; w += 2) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (i < s.cnt) v = *reinterpret_cast<const uint4*>(qp + 4 * w);
        x[w][0] = v.x, x[w][1] = v.y, x[w + 1][0] = v.z, x[w + 1][1] = v.w;
#pragma unroll
        for (int e = 0; e < 2; e++) {
          top = __vmaxu2(top, x[w][e] & 0x7fff7fffu);
          top = __vmaxu2(top, x[w + 1][e] & 0x7fff7fffu);
        }
      }
      top = max(top & 0xffffu, top >> 16);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // exponent e of the row's largest value: 2^(15 - e) as a float (2^126 at most); zero rows and non-finite ones stay as they are
      const int e = (int)(top >> 7), sh = top == 0 || e == 255 ? 0 : max(e - 127 - 15, -126);
      const float f = __uint_as_float((uint32_t)(127 - sh) << 23);
#pragma unroll
      for (int w = 0; w < WQ; w++)
#pragma unroll
        for (int k = 0; k < 2; k++)
          qf[nt][w][k] = pack_h2(__uint_as_float(x[w][k] << 16) * f, __uint_as_float(x[w][k] & 0xffff0000u) * f);
      const float back = __uint_as_float((uint32_t)(127 + sh) << 23) * a.scale_log2;
#pragma unroll
      for (int k = 0; k < 2; k++) {
        cq[nt][k] = __shfl_sync(0xffffffffu, back, (2 * t + k) * 4);  // lane of row 2t + k
        const int ic = (r0 + 8 * nt + 2 * t + k) / a.G;
        lim[nt][k] = ic >= s.cnt ? 0 : a.causal ? s.len + ic + 1 : T;
      }
    }
    const int sees_all = a.causal ? s.len + r0 / a.G + 1 : T;  // keys that every row of the group sees
    const bool all_rows = r0 + GR <= s.cnt * a.G;
    float m[NT][2], l[NT][2], o[OM][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int k = 0; k < 2; k++) m[nt][k] = -INFINITY, l[nt][k] = 0.f;
#pragma unroll
      for (int x = 0; x < OM; x++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[x][nt][e] = 0.f;
    }
    for (int j = 0; j < mine && ok; j++) {
      const int slot = consumed % ST, key0 = (ta + warp + WARPS * j) * KT;
      const float ks = ks_next, vs = vs_next;
      if (j + 1 < mine) ks_next = ksp[(key0 + WARPS * KT) / BLK], vs_next = vsp[(key0 + WARPS * KT) / BLK];
      ok = __all_sync(0xffffffffu, mbar_wait(&bar[slot], (consumed / ST) & 1, abort_flag, ST_KV8_WAIT));
      if (!ok) {
        if (lane == 0)  // the copies in flight land before the CTA ends
          for (int i = j; i < min(mine, j + ST); i++)
            mbar_wait_drain(&bar[(base + i) % ST], ((base + i) / ST) & 1, kDrainCycles);
        break;
      }
      const uint8_t *kt = ring + slot * 2 * TILE, *vt_ = kt + TILE;
      // ---- S^T = K Q^T: row x of an m-tile is key (x even ? x / 2 : 4 + x / 2), rows 8 .. 15 eight keys on
      float sc[MT][NT][4];
#pragma unroll
      for (int x = 0; x < MT; x++) {
        uint32_t kw[2][WQ];
        const int row = 16 * x + (g >> 1) + 4 * (g & 1);
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
          for (int w = 0; w < WQ; w += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(kt + (row + 8 * k) * D + t * (D / 4) + 4 * w);
            kw[k][w] = v.x, kw[k][w + 1] = v.y, kw[k][w + 2] = v.z, kw[k][w + 3] = v.w;
          }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[x][nt][e] = 0.f;
#pragma unroll
        for (int w = 0; w < WQ; w++) {
          const uint32_t c0 = kw[0][w] ^ 0x80808080u, c1 = kw[1][w] ^ 0x80808080u;
          const uint32_t a0 = hsub2(prmt(c0, 0x64646464u, 0x4140), H1152), a1 = hsub2(prmt(c1, 0x64646464u, 0x4140), H1152);
          const uint32_t a2 = hsub2(prmt(c0, 0x64646464u, 0x4342), H1152), a3 = hsub2(prmt(c1, 0x64646464u, 0x4342), H1152);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) mma_f16(sc[x][nt], a0, a1, a2, a3, qf[nt][w][0], qf[nt][w][1]);
        }
      }
      // ---- scores in log2 units; keys out of sight -inf
      const bool edge = !all_rows || key0 + KT > sees_all;
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        const float c[2] = {cq[nt][0] * ks, cq[nt][1] * ks};
#pragma unroll
        for (int x = 0; x < MT; x++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float v = sc[x][nt][e] * c[e & 1];
            if (edge && key0 + 16 * x + (g >> 1) + 4 * (g & 1) + 8 * (e >> 1) >= lim[nt][e & 1]) v = -INFINITY;
            sc[x][nt][e] = v;
          }
      }
      if (a.scores) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const int r = r0 + 8 * nt + 2 * t + k;
            if (r < a.rows) {
              float* sp = a.scores + (bh * a.rows + r) * a.C + key0 + (g >> 1) + 4 * (g & 1);
#pragma unroll
              for (int x = 0; x < MT; x++) {
                sp[16 * x] = sc[x][nt][k];
                sp[16 * x + 8] = sc[x][nt][2 + k];
              }
            }
          }
      }
      // ---- softmax: a column's keys are spread over the eight lanes g
      uint32_t pf[MT][NT][2];
      float al[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        float mu[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          float mx = -INFINITY;
#pragma unroll
          for (int x = 0; x < MT; x++) mx = max3f(mx, sc[x][nt][k], sc[x][nt][2 + k]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(m[nt][k], fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16)) - P_UP);
          mu[k] = mx == -INFINITY ? 0.f : mx;  // no key in sight yet: every exponential below is 0
          al[nt][k] = ex2_approx(m[nt][k] - mu[k]);
          m[nt][k] = mx;
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int x = 0; x < MT; x++) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            p[e] = ex2_approx(sc[x][nt][e] - mu[e & 1]);
            sum[e & 1] += p[e];
          }
          pf[x][nt][0] = transpose8x8(pack_h2(p[0], p[1]));
          pf[x][nt][1] = transpose8x8(pack_h2(p[2], p[3]));
        }
#pragma unroll
        for (int k = 0; k < 2; k++) l[nt][k] = l[nt][k] * al[nt][k] + sum[k];
      }
      // ---- O^T = alpha O^T + vs V^T P^T: word w of lane g is dims g D/8 + 4w .. + 3, two m-tiles.  A row that sees
      // nothing of the tile gets no product with its scale, which may be NaN; P's 2^15 is taken out, so that no scale overflows
      float vc[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int k = 0; k < 2; k++) vc[nt][k] = edge && key0 >= lim[nt][k] ? 0.f : vs * (1.f / P_SCALE);
#pragma unroll
      for (int w = 0; w < D / 32; w++) {
        float acc[2][NT][4];
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[y][nt][e] = 0.f;
#pragma unroll
        for (int x = 0; x < MT; x++) {
          uint32_t v[4];
#pragma unroll
          for (int k = 0; k < 4; k++)
            v[k] = *reinterpret_cast<const uint32_t*>(vt_ + (16 * x + 4 * k + t) * D + g * (D / 8) + 4 * w) ^ 0x80808080u;
          const uint32_t l01 = prmt(v[0], v[1], 0x5140), h01 = prmt(v[0], v[1], 0x7362);
          const uint32_t l23 = prmt(v[2], v[3], 0x5140), h23 = prmt(v[2], v[3], 0x7362);
#pragma unroll
          for (int y = 0; y < 2; y++) {
            const uint32_t p01 = y ? h01 : l01, p23 = y ? h23 : l23;
            const uint32_t a0 = hsub2(prmt(p01, 0x64646464u, 0x4140), H1152), a1 = hsub2(prmt(p01, 0x64646464u, 0x4342), H1152);
            const uint32_t a2 = hsub2(prmt(p23, 0x64646464u, 0x4140), H1152), a3 = hsub2(prmt(p23, 0x64646464u, 0x4342), H1152);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) mma_f16(acc[y][nt], a0, a1, a2, a3, pf[x][nt][0], pf[x][nt][1]);
          }
        }
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              o[2 * w + y][nt][e] = fmaf(vc[nt][e & 1], acc[y][nt][e], o[2 * w + y][nt][e] * al[nt][e & 1]);
      }
      consumed++;
      __syncwarp();  // every lane has read the slot before it is filled again
      if (lane == 0 && j + ST < mine) load(j + ST);
    }
    // ---- the warps' parts of the item, merged over their rings (all their copies have landed)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        float x = l[nt][k];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int r = 8 * nt + 2 * t + k;
        if (g == 0) sh_m[warp][r] = m[nt][k], sh_l[warp][r] = x;
        float* to = reinterpret_cast<float*>(ring) + r * D + g * (D / 8);
#pragma unroll
        for (int w = 0; w < D / 32; w++)
          *reinterpret_cast<float4*>(to + 4 * w) =
              make_float4(o[2 * w][nt][k], o[2 * w][nt][2 + k], o[2 * w + 1][nt][k], o[2 * w + 1][nt][2 + k]);
      }
    __syncthreads();
    const bool whole = WHOLE || (ta == 0 && tb == tiles);
    const int slot = 2 * blockIdx.x + (u == u_begin ? 0 : 1);  // of a part; a run has two at most: its first and its last
    for (int e = tid; e < GR * D / 4; e += WARPS * 32) {
      const int r = e / (D / 4), d = e % (D / 4) * 4, row = r0 + r;
      if (row >= s.cnt * a.G) break;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; w++) mx = fmaxf(mx, sh_m[w][r]);
      float sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        const float f = sh_m[w][r] == -INFINITY ? 0.f : ex2_approx(sh_m[w][r] - mx);
        const float4 x = *reinterpret_cast<const float4*>(sm + w * RING + (r * D + d) * 4);
        // scores that are all NaN leave m at -inf and l at NaN: 0 * NaN carries that on
        sum += sh_l[w][r] * f, v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
      }
      if (whole) {
        const float inv = P_SCALE / sum;
        uint16_t* op = a.out + b * a.so_b + row / a.G * a.so_t + (size_t)(h * a.G + row % a.G) * a.so_h + d;
        *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf2(v.x * inv, v.y * inv), pack_bf2(v.z * inv, v.w * inv));
        if (d == 0 && a.w) {
          if (WHOLE) sh_lse[r] = mx + log2f(sum);
          else a.full_ml[(bh * a.rg + rg) * GR + r] = make_float2(mx, sum);
        }
      } else {
        *reinterpret_cast<float4*>(a.part_o + ((size_t)slot * GR + r) * D + d) = v;
        if (d == 0) a.part_ml[(size_t)slot * GR + r] = make_float2(mx, sum);
      }
    }
    if (WHOLE) {
      if (a.w) {  // one row group: the item's rows are all the rows of (b, h)
        __syncthreads();
        for (int j = tid; j < T; j += WARPS * 32) {
          const size_t at = bh * a.C + j;
          float acc = a.w_in && j < s.len ? a.w_in[at] : 0.f;
          for (int r = 0; r < s.cnt * a.G; r++) acc += ex2_approx(a.scores[(bh * a.rows + r) * a.C + j] - sh_lse[r]);
          a.w[at] = acc;
        }
      }
      return;
    }
    fence_proxy_async_smem();  // these reads and writes come before the next item's copies into the rings
    __syncthreads();
    u += tb - ta;
  }
}

// Merges the parts of items that span CTAs and turns scores into weights.
// CTAs [0, merge_ctas): one row of an item; each of 128 * 4 / D groups of threads (thread = 4 dims) takes every so many'th
// part, the groups' sums are added in order.  The others: 512 keys of one (sequence, head):
// weight = (key before len ? weights_in : 0) + sum over rows of 2^(score - m - log2 l), a row's (m, l) by a warp.
template <int D, int NT>
__global__ void __launch_bounds__(128) attn_kv8_join_kernel(Args a, int merge_ctas) {
  constexpr int KT = TILE / D, GR = 8 * NT, GROUPS = 128 * 4 / D;
  __shared__ int pre[MAXB + 1], warp_sum[4];
  __shared__ float lse[FEW_ROWS];
  __shared__ __align__(16) float4 sh_o[128];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_wait();
  griddep_launch();
  tile_list(a, KT, GR, pre, warp_sum);
  const int run = run_of(pre[a.B], a.ctas);
  // the first and last CTA that hold a part of an item, and the first part's slot (the others begin their CTA's run: 2 c)
  auto parts = [&](const Seq& s, int b, int h, int rg, int tiles, int& c0, int& c1, int& first) {
    const int u0 = pre[b] + (h * row_groups(a, s, GR) + rg) * tiles;
    c0 = u0 / run, c1 = (u0 + tiles - 1) / run;
    first = 2 * c0 + (u0 == c0 * run ? 0 : 1);
  };
  auto slot = [&](int c, int c0, int first) { return (size_t)(c == c0 ? first : 2 * c) * GR; };
  // a row's maximum and sum over its parts, lane c taking part c0 + c and so on: the same in every warp that asks
  auto row_ml = [&](int c0, int c1, int first, int r, float& mx, float& sum) {
    mx = -INFINITY, sum = 0.f;
    for (int c = c0 + lane; c <= c1; c += 32) mx = fmaxf(mx, a.part_ml[slot(c, c0, first) + r].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    for (int c = c0 + lane; c <= c1; c += 32) {
      const float2 ml = a.part_ml[slot(c, c0, first) + r];
      sum += ml.x == -INFINITY ? 0.f * ml.y : ml.y * ex2_approx(ml.x - mx);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  };
  if ((int)blockIdx.x < merge_ctas) {
    const int rows = min(GR, a.rows), item = blockIdx.x / rows, r = blockIdx.x % rows;
    const int rg = item % a.rg, h = item / a.rg % a.H, b = item / a.rg / a.H;
    const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C);
    const int row = rg * GR + r, tiles = (s.len + s.cnt + KT - 1) / KT;
    if (row >= s.cnt * a.G) return;
    int c0, c1, first;
    parts(s, b, h, rg, tiles, c0, c1, first);
    if (c0 == c1) return;
    float mx, sum;
    row_ml(c0, c1, first, r, mx, sum);
    const int grp = tid / (D / 4), d = tid % (D / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = c0 + grp; c <= c1; c += GROUPS) {
      const size_t at = slot(c, c0, first) + r;
      const float m = a.part_ml[at].x;
      const float4 x = *reinterpret_cast<const float4*>(a.part_o + at * D + d);
      const float f = m == -INFINITY ? 0.f : ex2_approx(m - mx);
      v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
    }
    sh_o[tid] = v;
    __syncthreads();
    if (grp == 0) {
      for (int k = 1; k < GROUPS; k++) {
        const float4 x = sh_o[tid + k * (D / 4)];
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      const float inv = P_SCALE / sum;
      uint16_t* op = a.out + b * a.so_b + row / a.G * a.so_t + (size_t)(h * a.G + row % a.G) * a.so_h + d;
      *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf2(v.x * inv, v.y * inv), pack_bf2(v.z * inv, v.w * inv));
    }
    return;
  }
  const int chunks = (a.C + 511) / 512, x = blockIdx.x - merge_ctas;
  const int bh = x / chunks, j = x % chunks * 512 + tid * 4, h = bh % a.H, b = bh / a.H;
  const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C);
  const int T = s.len + s.cnt, rows = s.cnt * a.G, tiles = (T + KT - 1) / KT;
  if (x % chunks * 512 >= T) return;
  for (int r = warp; r < rows; r += 4) {
    int c0, c1, first;
    parts(s, b, h, r / GR, tiles, c0, c1, first);
    float mx, sum;
    if (c0 == c1) {
      const float2 ml = a.full_ml[((size_t)bh * a.rg + r / GR) * GR + r % GR];
      mx = ml.x, sum = ml.y;
    } else {
      row_ml(c0, c1, first, r % GR, mx, sum);
    }
    if (lane == 0) lse[r] = mx + log2f(sum);
  }
  __syncthreads();
  if (j >= T) return;
  float acc[4];
  const size_t at = (size_t)bh * a.C + j;
#pragma unroll
  for (int e = 0; e < 4; e++) acc[e] = a.w_in && j + e < s.len ? a.w_in[at + e] : 0.f;
  for (int r = 0; r < rows; r++) {
    const float4 v = *reinterpret_cast<const float4*>(a.scores + ((size_t)bh * a.rows + r) * a.C + j);
    acc[0] += ex2_approx(v.x - lse[r]);
    acc[1] += ex2_approx(v.y - lse[r]);
    acc[2] += ex2_approx(v.z - lse[r]);
    acc[3] += ex2_approx(v.w - lse[r]);
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (j + e < T) a.w[at + e] = acc[e];
}

template <int D, int NT>
static int launch(cudaStream_t st, const Args& a, bool whole) {
  if (whole) {
    constexpr int SMEM = WHOLE_WARPS * RING;
    const int rc = smem_attr_once((const void*)attn_kv8_split_kernel<D, NT, true>, SMEM, "vt_attn_kv8");
    if (rc) return rc;
    launch_k(attn_kv8_split_kernel<D, NT, true>, (unsigned)(a.B * a.H * a.rg), WHOLE_WARPS * 32, SMEM, st, a);
    return check_launch("vt_attn_kv8");
  }
  constexpr int SMEM = WARPS * RING;
  const int rc = smem_attr_once((const void*)attn_kv8_split_kernel<D, NT, false>, SMEM, "vt_attn_kv8");
  if (rc) return rc;
  launch_k(attn_kv8_split_kernel<D, NT, false>, a.ctas, WARPS * 32, SMEM, st, a);
  const int rows = 8 * NT < a.rows ? 8 * NT : a.rows;
  const int merge = a.B * a.H * a.rg * rows;
  const int chunks = a.w ? a.B * a.H * ((a.C + 511) / 512) : 0;
  launch_k(attn_kv8_join_kernel<D, NT>, merge + chunks, 128, 0, st, a, merge);
  return check_launch("vt_attn_kv8");
}

}  // namespace split
}  // namespace kv8
}  // namespace vt
