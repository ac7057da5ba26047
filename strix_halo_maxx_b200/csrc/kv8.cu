// The 8-bit key / value cache: rotary embedding + quantised cache write, attention over it, eviction from it.
//
// One layer's cache holds int8 codes k, v [B][H][C][D] and one fp32 scale per block of 64 slots and head
// ks, vs [B][H][C / 64]; a value is code * scale.  lens[b] (device memory) counts the tokens sequence b holds
// before a call, counts[b] <= n its new ones, so one captured graph serves every length.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {

constexpr int BLK = 64;    // slots that share a scale
constexpr int ROT = 32;    // rotary dims of a head
constexpr float LOG2E = 1.4426950408889634f;

// What a call does for sequence b: len tokens held, cnt new ones (0: idle).  Lengths live on the device, where the
// host cannot refuse them: what does not fit in the cache is cut off and recorded in the status word.
struct Seq {
  int len, cnt;
};
__device__ __forceinline__ Seq clip_seq(int len, int cnt, int n, int C, bool record) {
  const bool bad = len < 0 || len > C || cnt < 0 || cnt > n || cnt > C - len;
  len = min(max(len, 0), C);
  cnt = min(min(max(cnt, 0), n), C - len);
  if (bad && record) atomicOr(&g_status, (unsigned int)ST_KV8_RANGE);
  return {len, cnt};
}
__device__ __forceinline__ Seq seq_of(const int* lens, const int* counts, int b, int n, int C, bool record) {
  return clip_seq(lens[b], counts ? counts[b] : n, n, C, record);
}
__device__ __forceinline__ Seq seq_of(const int* lens, const int* counts, int b, int n, int C) {
  return seq_of(lens, counts, b, n, C, threadIdx.x == 0);
}

// ---------------------------------------------------------------- append
struct AppendArgs {
  const uint16_t* qkv;
  long long sx_b, sx_t;
  int B, n, Hq, H, C, tab, nb;
  const float *cos_t, *sin_t;
  const int *lens, *pos, *counts;
  uint16_t* q;
  long long sq_b, sq_t, sq_h;
  int8_t *kc, *vc;
  float *ks, *vs;
  long long kv_units;
};

// 8 output dims (chunk c) of a head's row x, as bf16 pairs.  The first 32 dims rotate as pairs (x_i, x_(16+i)) into
// dims 2i, 2i+1; products and differences are rounded one by one (no FMA), so the value that is quantised does
// not depend on how the compiler contracts them.
__device__ __forceinline__ uint4 head_chunk(const uint16_t* x, int c, bool rotate, const float* cs, const float* sn) {
  if (!rotate || c >= ROT / 8) return *reinterpret_cast<const uint4*>(x + 8 * c);
  const uint2 a = *reinterpret_cast<const uint2*>(x + 4 * c), b = *reinterpret_cast<const uint2*>(x + ROT / 2 + 4 * c);
  const float4 co = *reinterpret_cast<const float4*>(cs + 4 * c), si = *reinterpret_cast<const float4*>(sn + 4 * c);
  const float av[4] = {__uint_as_float(a.x << 16), __uint_as_float(a.x & 0xffff0000u), __uint_as_float(a.y << 16),
                       __uint_as_float(a.y & 0xffff0000u)};
  const float bv[4] = {__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16),
                       __uint_as_float(b.y & 0xffff0000u)};
  const float cv[4] = {co.x, co.y, co.z, co.w}, sv[4] = {si.x, si.y, si.z, si.w};
  uint32_t o[4];
#pragma unroll
  for (int e = 0; e < 4; e++)
    o[e] = pack_bf2(__fsub_rn(__fmul_rn(av[e], cv[e]), __fmul_rn(bv[e], sv[e])),
                    __fadd_rn(__fmul_rn(av[e], sv[e]), __fmul_rn(bv[e], cv[e])));
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// rint(x / s) as a byte, s > 0 a block's scale.  The IEEE quotient in five operations (div_rn_by) where that is exact, which
// is for every scale that is not extreme; adding 1.5 * 2^23 rounds it half to even and leaves the integer in the low bits.
// The division itself, with its clamp for subnormal scales, stays out of line: inlined once for each value of a thread it
// filled the instruction cache (eviction's gather 188 us for 268 MB, half of its stalls for want of instructions).
__noinline__ __device__ uint32_t code_div(float x, float s) {
  return (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.f), 127.f);
}
struct Divisor {
  float s, rs;
  bool fast;
  __device__ explicit Divisor(float scale) : s(scale), rs(0.f), fast(scale > 0x1p-80f && scale < 0x1p100f) {
    if (fast) rs = __frcp_rn(s);
  }
};
__device__ __forceinline__ uint32_t code_of(float x, const Divisor& d) {  // in the low byte
  return d.fast ? __float_as_uint(__fadd_rn(div_rn_by(x, d.s, d.rs), 12582912.f)) : code_div(x, d.s);
}
__device__ __forceinline__ uint32_t codes4(float x0, float x1, float x2, float x3, const Divisor& d) {
  return __byte_perm(__byte_perm(code_of(x0, d), code_of(x1, d), 0x0040), __byte_perm(code_of(x2, d), code_of(x3, d), 0x0040), 0x5410);
}

// CTA = one block of 64 slots of one (sequence, head, K or V) that gets new tokens, or a run of q chunks.
// Block scale: max |x| / 127 over the new tokens when the block held none (or only zeros: scale 0); else the old
// scale, doubled until the new tokens fit, the held codes shifted by as many bits (rint(c / 2^j), half to even).
// Doubling keeps a held value within half a step of each scale it went through, 1/2 + 1/4 + ... < 1 step of the
// last, however many tokens arrive one by one; scales that grew just enough would add up to one rounding for
// each token of the block.  A NaN or an infinity among the values makes the block's scale NaN.
// 730 tokens of 32 heads x 64: 6.4 us for 15 MB; one token 2.3 us, a launch and the loads behind its length.
template <int D>
__global__ void __launch_bounds__(128) rope_kv8_kernel(AppendArgs a) {
  constexpr int CH = D / 8, PER = BLK * CH / 128;
  __shared__ unsigned int red[4];
  const int tid = threadIdx.x;
  griddep_wait();  // programmatic dependent launch: the previous kernel has completed
  griddep_launch();
  if ((long long)blockIdx.x >= a.kv_units) {  // q rows: thread = 8 output dims
    const long long total = (long long)a.B * a.n * a.Hq * CH;
    for (long long t = ((long long)blockIdx.x - a.kv_units) * 128 + tid; t < total;
         t += ((long long)gridDim.x - a.kv_units) * 128) {
      const int c = (int)(t % CH), hq = (int)((t / CH) % a.Hq);
      const long long row = t / ((long long)CH * a.Hq);
      const int i = (int)(row % a.n), b = (int)(row / a.n);
      const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C);
      if (i >= s.cnt) continue;
      const int p = min(min(max(a.pos ? a.pos[b] : s.len, 0), a.tab) + i, a.tab - 1);
      const uint16_t* x = a.qkv + b * a.sx_b + i * a.sx_t + (size_t)hq * D;
      *reinterpret_cast<uint4*>(a.q + b * a.sq_b + i * a.sq_t + hq * a.sq_h + 8 * c) =
          head_chunk(x, c, true, a.cos_t + (size_t)p * (ROT / 2), a.sin_t + (size_t)p * (ROT / 2));
    }
    return;
  }
  const int w = blockIdx.x & 1;
  long long u = blockIdx.x >> 1;
  const int h = (int)(u % a.H);
  u /= a.H;
  const int b = (int)(u / a.nb);
  const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C);
  const int blk = s.len / BLK + (int)(u % a.nb);
  const int lo = max(blk * BLK, s.len), hi = min((blk + 1) * BLK, s.len + s.cnt);
  if (lo >= hi) return;
  const int i0 = lo - s.len, m = hi - lo, held = lo - blk * BLK;
  const int p_in = a.pos ? a.pos[b] : s.len, p0 = min(max(p_in, 0), a.tab);
  if (tid == 0 && w == 0 && (p_in != p0 || p0 + i0 + m > a.tab)) atomicOr(&g_status, (unsigned int)ST_KV8_RANGE);
  const size_t bh = (size_t)b * a.H + h;
  int8_t* codes = (w ? a.vc : a.kc) + (bh * a.C + (size_t)blk * BLK) * D;
  float* scale = (w ? a.vs : a.ks) + bh * (a.C / BLK) + blk;
  const float s_old = held ? *scale : 0.f;
  const uint16_t* src = a.qkv + b * a.sx_b + (size_t)(a.Hq + (w ? a.H : 0) + h) * D;
  uint4 v[PER];
  uint32_t top = 0;  // max of |bf16| as bit patterns, two at a time: NaN above infinity above every number
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int t = tid + 128 * k, row = t / CH, c = t % CH;
    v[k] = make_uint4(0, 0, 0, 0);
    if (row < m) {
      const int p = min(p0 + i0 + row, a.tab - 1);
      v[k] = head_chunk(src + (i0 + row) * a.sx_t, c, w == 0, a.cos_t + (size_t)p * (ROT / 2),
                        a.sin_t + (size_t)p * (ROT / 2));
    }
    const uint32_t x[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
    for (int e = 0; e < 4; e++) top = __vmaxu2(top, x[e] & 0x7fff7fffu);
  }
  top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
  top = max(max(red[0], red[1]), max(red[2], red[3]));
  const float need = top >= 0x7f80u ? __uint_as_float(0x7fc00000u) : __fdiv_rn(bf2f((uint16_t)top), 127.f);
  float sc = need;
  if (s_old != 0.f) {
    sc = s_old;
    if (isnan(need) || isnan(s_old)) {
      sc = __uint_as_float(0x7fc00000u);
    } else if (need > s_old) {
      int j = max(ilogbf(need) - ilogbf(s_old), 0);
      if (scalbnf(s_old, j) < need) j++;
      sc = scalbnf(s_old, j);
      const float f = scalbnf(1.f, -j);
      for (int t = tid; t < held * CH; t += 128) {  // the held codes, 8 at a time
        uint2* at = reinterpret_cast<uint2*>(codes) + t;
        const uint2 c = *at;
        uint32_t o[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int x = (int8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3)));
          o[e >> 2] |= ((uint32_t)(int)rintf((float)x * f) & 0xffu) << (8 * (e & 3));
        }
        *at = make_uint2(o[0], o[1]);
      }
    }
  }
  const Divisor div(sc);
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int t = tid + 128 * k, row = t / CH, c = t % CH;
    if (row >= m) continue;
    uint2 o = make_uint2(0, 0);
    if (sc > 0.f) {  // neither zero nor NaN
      auto lo = [](uint32_t x) { return __uint_as_float(x << 16); };
      auto hi = [](uint32_t x) { return __uint_as_float(x & 0xffff0000u); };
      o.x = codes4(lo(v[k].x), hi(v[k].x), lo(v[k].y), hi(v[k].y), div);
      o.y = codes4(lo(v[k].z), hi(v[k].z), lo(v[k].w), hi(v[k].w), div);
    }
    *reinterpret_cast<uint2*>(codes + (size_t)(held + row) * D + 8 * c) = o;
  }
  if (tid == 0) *scale = sc;
}

// ---------------------------------------------------------------- eviction
struct EvictArgs {
  const int8_t *kc, *vc;
  const float *ks, *vs, *w;
  const int* lens;
  int B, H, C, keep, recent, Cd;
  int8_t *dkc, *dvc;
  float *dks, *dvs, *dw;
  int *dlens, *index;
};

constexpr int MAX_EVICT = 8 * 1024 * 32;  // slots of a head that a cluster of 8 CTAs holds in registers

// Order of weights as unsigned numbers: -inf .. +inf, NaN above all, -0 equal to 0.
__device__ __forceinline__ uint32_t order_of(uint32_t u) {
  const uint32_t mag = u & 0x7fffffffu;
  const uint32_t k = u & 0x80000000u && mag ? ~u : mag | 0x80000000u;
  return mag > 0x7f800000u ? 0xffffffffu : k;
}

// The weight with that key (+0 for -0).
__device__ __forceinline__ float weight_of(uint32_t u) {
  return u == 0xffffffffu ? __uint_as_float(0x7fc00000u) : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// Which slots of a head stay: the (keep - recent) largest weights before the recent ones, and the recent ones.  A head is one
// CTA's, or a cluster's of CS CTAs (each a contiguous range of slots), and every weight is read once: a thread keeps the
// order keys of up to KPT slots in registers (warp w of a CTA has 32 kpt consecutive slots, key i of lane l is slot 32 i + l).
// The threshold is found two bits at a time from the top: three counts of keys above a candidate, added up over warps,
// CTAs and the cluster; a candidate with exactly the wanted count ends the search (after about 11 of 16 rounds for
// weights that differ).  Once no more keys share the threshold's leading bits than a CTA has threads, those keys move to
// one register each and a round is little more than its barrier.  Counting by comparison needs no atomics, whose same-address
// conflicts made histograms of these skewed weights (most share an exponent) slow: 397 us for 8 heads of 131k slots,
// 98 us for 256 heads of 16k.  Then positions by ballots and prefix sums: kept slots are written in order, ties to the
// lowest slots.  Bound by instruction issue (six a key and round) and the rounds' barriers.
template <int THREADS, int KPT, int CS>
__global__ void __launch_bounds__(THREADS) kv8_select_kernel(EvictArgs a) {
  constexpr int W = THREADS / 32;
  __shared__ unsigned int sh_warp[2][2][W];
  __shared__ unsigned int sh_cta[2][CS][3];
  __shared__ unsigned int sh_gt[W], sh_eq[W], sh_before[CS][2];
  __shared__ uint32_t sh_key[THREADS];
  __shared__ unsigned int sh_keys;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = CS > 1 ? (int)cluster_ctarank() : 0;
  const long long bh = blockIdx.x / CS;
  const int h = (int)(bh % a.H), b = (int)(bh / a.H);
  if constexpr (CS > 1) cluster_sync();  // every CTA of the cluster has started before another one writes its shared memory
  griddep_wait();
  griddep_launch();
  int len = a.lens[b];
  if ((len < 0 || len > a.C) && tid == 0) atomicOr(&g_status, (unsigned int)ST_KV8_RANGE);
  len = min(max(len, 0), a.C);
  const float* w = a.w + bh * a.C;
  float* dw = a.dw + bh * a.Cd;
  int* idx = a.index + bh * a.keep;
  if (h == 0 && rank == 0 && tid == 0) a.dlens[b] = min(len, a.keep);
  if (len <= a.keep) {  // the whole cluster
    for (int j = rank * THREADS + tid; j < len; j += CS * THREADS) {
      idx[j] = j;
      dw[j] = w[j];
    }
    return;
  }
  const int N = len - a.recent, kpt = (len + CS * THREADS - 1) / (CS * THREADS);
  const unsigned int want = a.keep - a.recent;
  const int j0 = (rank * W + warp) * 32 * kpt + lane;  // slot of key i: j0 + 32 i
  uint32_t key[KPT];  // 0: not a candidate (the key of -inf is 0x007fffff)
#pragma unroll
  for (int i = 0; i < KPT; i++) key[i] = i < kpt && j0 + 32 * i < N ? __float_as_uint(__ldg(w + j0 + 32 * i)) : 0u;  // all on their way
#pragma unroll
  for (int i = 0; i < KPT; i++) key[i] = i < kpt && j0 + 32 * i < N ? order_of(key[i]) : 0u;
  // sums over the warps of a CTA of what lane i < W of each warp holds
  auto over_warps = [&](unsigned int x) { return W > 1 ? __reduce_add_sync(0xffffffffu, lane < W ? x : 0u) : x; };
  int round = 0;
  // sums over the head of three counts (at most 1024 in a warp: two to a register)
  auto total3 = [&](unsigned int c1, unsigned int c2, unsigned int c3, unsigned int (&sum)[3]) {
    const int f = round++ & 1;
    const unsigned int p12 = __reduce_add_sync(0xffffffffu, c1 | (c2 << 16));
    const unsigned int p3 = __reduce_add_sync(0xffffffffu, c3);
    if (lane == 0) sh_warp[f][0][warp] = p12, sh_warp[f][1][warp] = p3;
    __syncthreads();
    if constexpr (W == 2) {
      const unsigned int x = sh_warp[f][0][0], y = sh_warp[f][0][1];
      sum[0] = (x & 0xffffu) + (y & 0xffffu), sum[1] = (x >> 16) + (y >> 16), sum[2] = sh_warp[f][1][0] + sh_warp[f][1][1];
    } else {
      const unsigned int x = lane < W ? sh_warp[f][0][lane] : 0u, y = lane < W ? sh_warp[f][1][lane] : 0u;
      sum[0] = over_warps(x & 0xffffu), sum[1] = over_warps(x >> 16), sum[2] = over_warps(y);
    }
    if constexpr (CS > 1) {
      if (tid < CS * 3) {  // this CTA's sums to every CTA of the cluster
        const uint32_t to = mapa_shared(smem_u32(&sh_cta[f][rank][tid % 3]), tid / 3);
        const unsigned int v = tid % 3 == 0 ? sum[0] : tid % 3 == 1 ? sum[1] : sum[2];
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(v) : "memory");
      }
      __syncwarp();  // the barrier below is one for whole warps
      cluster_sync();
#pragma unroll
      for (int k = 0; k < 3; k++) {
        sum[k] = 0;
#pragma unroll
        for (int r = 0; r < CS; r++) sum[k] += sh_cta[f][r][k];
      }
    }
  };
  // T: the largest key with at least `want` keys >= T; above: how many are > T; upto: how many are >= T
  unsigned int T = want ? 0u : 0xffffffffu, above = 0, upto = 0xffffffffu;
  bool few = false;
  uint32_t one = 0;  // this thread's key among the few that are left
#pragma unroll 1
  for (int shift = 30; shift >= 0 && want > 0; shift -= 2) {
    unsigned int c1 = 0, c2 = 0, c3 = 0, sum[3];
    const uint32_t t1 = T + (1u << shift), t2 = T + (2u << shift), t3 = T + (3u << shift);
    if (few) {
      c1 = one >= t1, c2 = one >= t2, c3 = one >= t3;
    } else {
#pragma unroll
      for (int i = 0; i < KPT; i += 4)
        if (i < kpt) {
#pragma unroll
          for (int e = i; e < i + 4; e++) c1 += key[e] >= t1, c2 += key[e] >= t2, c3 += key[e] >= t3;
        }
    }
    total3(c1, c2, c3, sum);
    if (few) sum[0] += above, sum[1] += above, sum[2] += above;  // the larger keys are not among the few
    const int d = sum[2] >= want ? 3 : sum[1] >= want ? 2 : sum[0] >= want ? 1 : 0;
    above = d == 3 ? above : d == 2 ? sum[2] : d == 1 ? sum[1] : sum[0];
    if (d > 0) upto = d == 3 ? sum[2] : d == 2 ? sum[1] : sum[0];
    T += (unsigned int)d << shift;
    if (d > 0 && upto == want) {  // exactly the keys >= T
      T--, above = want;
      break;
    }
    const uint32_t top = T + ((1u << shift) - 1u);  // keys T .. top share the leading bits
    if (few) {
      if (one < T || one > top) one = 0;
    } else if (upto - above <= THREADS) {  // their number over the head (not known, and large, while T is 0)
      if (tid == 0) sh_keys = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < KPT; i += 4)
        if (i < kpt) {
#pragma unroll
          for (int e = i; e < i + 4; e++)
            if (key[e] >= T && key[e] <= top && key[e] != 0u) sh_key[atomicAdd(&sh_keys, 1u)] = key[e];
        }
      __syncthreads();
      one = tid < (int)sh_keys ? sh_key[tid] : 0u;
      few = true;
    }
  }
  const unsigned int ties = want - above;  // of the keys equal to T
  // positions: kept (key > T, or recent) and equal keys before each slot, over CTAs, warps, rows of 32 and lanes
  unsigned int gt = 0, eq = 0;
#pragma unroll
  for (int i = 0; i < KPT; i++)
    if (i < kpt) {
      const int j = j0 + 32 * i;
      gt += __popc(__ballot_sync(0xffffffffu, key[i] > T || (j >= N && j < len)));
      eq += __popc(__ballot_sync(0xffffffffu, key[i] == T && key[i] != 0u));
    }
  if (lane == 0) sh_gt[warp] = gt, sh_eq[warp] = eq;
  __syncthreads();
  const unsigned int xg = lane < W ? sh_gt[lane] : 0u, xe = lane < W ? sh_eq[lane] : 0u;
  unsigned int bg = __reduce_add_sync(0xffffffffu, lane < warp ? xg : 0u), be = __reduce_add_sync(0xffffffffu, lane < warp ? xe : 0u);
  if constexpr (CS > 1) {
    const unsigned int tg = __reduce_add_sync(0xffffffffu, xg), te = __reduce_add_sync(0xffffffffu, xe);
    if (tid < CS * 2) {
      const uint32_t to = mapa_shared(smem_u32(&sh_before[rank][tid & 1]), tid / 2);
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(tid & 1 ? te : tg) : "memory");
    }
    __syncwarp();
    cluster_sync();  // the last access to another CTA's shared memory is before it
    for (int r = 0; r < rank; r++) bg += sh_before[r][0], be += sh_before[r][1];
  }
  const unsigned int below = (1u << lane) - 1u;
#pragma unroll
  for (int i = 0; i < KPT; i++)
    if (i < kpt) {
      const int j = j0 + 32 * i;
      const bool sure = key[i] > T || (j >= N && j < len), even = key[i] == T && key[i] != 0u;
      const unsigned int mg = __ballot_sync(0xffffffffu, sure), me = __ballot_sync(0xffffffffu, even);
      const unsigned int e = be + __popc(me & below);
      if (sure || (even && e < ties)) {
        const unsigned int at = bg + __popc(mg & below) + min(e, ties);
        idx[at] = j;
        dw[at] = j < N ? weight_of(key[i]) : __ldg(w + j);  // from the register: a load behind each store costs its latency
      }
      bg += __popc(mg), be += __popc(me);
    }
}

// Largest |code| of 16, as a number.
__device__ __forceinline__ int top_code(uint4 c) {
  uint32_t m = __vmaxu4(__vmaxu4(__vabsdiffs4(c.x, 0), __vabsdiffs4(c.y, 0)), __vmaxu4(__vabsdiffs4(c.z, 0), __vabsdiffs4(c.w, 0)));
  m = __vmaxu2(m & 0x00ff00ffu, (m >> 8) & 0x00ff00ffu);
  return (int)max(m & 0xffffu, m >> 16);
}
// Four codes c times `s` (rounded), each divided by the new scale and rounded half to even: codes again.
__noinline__ __device__ uint32_t recode4(uint32_t c, float s, float scale) {
  const Divisor d(scale);
  c ^= 0x80808080u;
  // byte into the mantissa of 2^23: 2^23 + 128 + code
  auto value = [&](uint32_t sel) { return __fmul_rn(__uint_as_float(__byte_perm(c, 0x4b000000u, sel)) - 8388736.f, s); };
  return codes4(value(0x7440), value(0x7441), value(0x7442), value(0x7443), d);
}
// The same from the rounded ratio of the scales: code * ratio is within 127.1 * 4 * 2^-24 < 2^-15 of the quotient above, so it
// rounds to the same integer unless it lies that near to a half; `worst` collects the distance from the integer.
__device__ __forceinline__ uint32_t recode4_near(uint32_t c, unsigned long long ratio2, float& worst) {
  const unsigned long long off = f2_pack(-8388736.f, -8388736.f), magic = f2_pack(12582912.f, 12582912.f),
                           unmagic = f2_pack(-12582912.f, -12582912.f), minus = f2_pack(-1.f, -1.f);
  c ^= 0x80808080u;
  uint32_t o[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const unsigned long long x = f2_add(f2_pack(__uint_as_float(__byte_perm(c, 0x4b000000u, 0x7440 + 2 * k)),
                                                __uint_as_float(__byte_perm(c, 0x4b000000u, 0x7441 + 2 * k))), off);
    const unsigned long long q = f2_mul(x, ratio2), r = f2_add(q, magic);
    float r0, r1, t0, t1;
    f2_unpack(r, r0, r1);
    f2_unpack(f2_fma(f2_add(r, unmagic), minus, q), t0, t1);
    worst = max3f(worst, fabsf(t0), fabsf(t1));
    o[k] = __byte_perm(__float_as_uint(r0), __float_as_uint(r1), 0x0040);
  }
  return __byte_perm(o[0], o[1], 0x5410);
}

// CTA = one block of 64 kept tokens of one (sequence, head), K and V: values code * scale (rounded to fp32), the block's
// scale max |value| / 127 and codes rint(value / scale).  Rows come by 16-byte asynchronous copies, all on their way at once,
// and the passes over them are short loops (unrolled over registers, they ran out of instruction cache).  Most pieces
// of 16 codes need only a multiplication by the ratio of the scales; one in 500 has a value near a half and takes the
// quotients.  Sequences that lost nothing are copied.  Bound: DRAM, rows of 64 or 128 bytes apart.
template <int D>
__global__ void __launch_bounds__(128) kv8_gather_kernel(EvictArgs a) {
  constexpr int PC = D / 16, PIECES = BLK * PC;  // 16-byte pieces of a row, of a block
  __shared__ __align__(16) uint4 code[2][PIECES];
  __shared__ float scale[2][BLK], ratio[2][BLK], red[2][4];
  __shared__ int slot[BLK];
  const int tid = threadIdx.x;
  griddep_wait();
  griddep_launch();
  const int nb = a.keep / BLK, blk = (int)(blockIdx.x % nb);
  const size_t bh = blockIdx.x / nb;
  const int len = min(max(a.lens[bh / a.H], 0), a.C);
  const int rows = min(min(len, a.keep) - blk * BLK, BLK);
  if (rows <= 0) return;
  const bool copy = len <= a.keep;
  const int v = tid / BLK, r = tid % BLK;  // this thread's row of scales: K's or V's
  if (r < rows) {
    const int j = copy ? blk * BLK + r : a.index[bh * a.keep + blk * BLK + r];
    if (v == 0) slot[r] = j;
    scale[v][r] = (v ? a.vs : a.ks)[bh * (a.C / BLK) + j / BLK];
  }
  __syncthreads();
  for (int p = tid; p < rows * PC; p += 128) {
    const size_t at = (bh * a.C + slot[p / PC]) * D + 16 * (p % PC);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&code[0][p])), "l"(a.kc + at) : "memory");
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&code[1][p])), "l"(a.vc + at) : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  int8_t* dst[2] = {a.dkc + (bh * a.Cd + (size_t)blk * BLK) * D, a.dvc + (bh * a.Cd + (size_t)blk * BLK) * D};
  float* ds[2] = {a.dks + bh * (a.Cd / BLK) + blk, a.dvs + bh * (a.Cd / BLK) + blk};
  if (copy) {
    for (int k = 0; k < 2; k++) {
      for (int p = tid; p < rows * PC; p += 128) reinterpret_cast<uint4*>(dst[k])[p] = code[k][p];  // this thread's own copies
      if (tid == 0) *ds[k] = scale[k][0];
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 2; k++) {
    float top = 0.f;  // rounding is monotonic: the largest rounded product is that of the largest code
#pragma unroll 2
    for (int p = tid; p < PIECES; p += 128) {  // a sequence that lost tokens fills its blocks
      const float s = scale[k][p / PC];
      top = isnan(s) ? INFINITY : fmaxf(top, __fmul_rn((float)top_code(code[k][p]), fabsf(s)));
    }
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    if ((tid & 31) == 0) red[k][tid >> 5] = top;
  }
  __syncthreads();
  float s[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const float top = fmaxf(fmaxf(red[k][0], red[k][1]), fmaxf(red[k][2], red[k][3]));
    s[k] = isinf(top) ? __uint_as_float(0x7fc00000u) : __fdiv_rn(top, 127.f);
  }
  // above 2^100 every code of the row is 0 (its value would be the block's largest); an infinite ratio would make them NaN
  ratio[v][r] = fminf(__fdiv_rn(scale[v][r], v ? s[1] : s[0]), 0x1p100f);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; k++) {
    if (tid == 0) *ds[k] = s[k];
    const bool fast = s[k] > 0x1p-80f && s[k] < 0x1p100f;
#pragma unroll 1
    for (int p = tid; p < PIECES; p += 128) {
      const uint4 c = code[k][p];
      uint4 o = make_uint4(0, 0, 0, 0);
      if (s[k] > 0.f) {  // neither zero nor NaN
        const float f = ratio[k][p / PC];
        const unsigned long long f2 = f2_pack(f, f);
        float worst = 0.f;
        o = make_uint4(recode4_near(c.x, f2, worst), recode4_near(c.y, f2, worst), recode4_near(c.z, f2, worst), recode4_near(c.w, f2, worst));
        if (!fast || !(worst < 0.5f - 0x1p-14f)) {
          const float sp = scale[k][p / PC];
          o = make_uint4(recode4(c.x, sp, s[k]), recode4(c.y, sp, s[k]), recode4(c.z, sp, s[k]), recode4(c.w, sp, s[k]));
        }
      }
      reinterpret_cast<uint4*>(dst[k])[p] = o;
    }
  }
}

template <int THREADS, int KPT, int CS>
static int launch_select(cudaStream_t st, const EvictArgs& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * a.H * CS));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CS, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kv8_select_kernel<THREADS, KPT, CS>, a);
  return check_launch("vt_kv8_evict");
}

static bool overlap(const void* p, long long n, const void* q, long long m) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return a < b + (uintptr_t)m && b < a + (uintptr_t)n;
}

// Rows (b, t) of `w` elements at p + b sb + t st.
struct Rows {
  const uint16_t* p;
  long long sb, st, w;
};
// Whether rows of x and y may share an element: by columns where both have the same strides, else by where they begin and end.
static bool rows_meet(const Rows& x, const Rows& y, int B, int n) {
  auto span = [&](const Rows& r, const uint16_t*& lo, const uint16_t*& hi) {
    const long long b = (B - 1) * r.sb, t = (n - 1) * r.st;
    lo = r.p + (b < 0 ? b : 0) + (t < 0 ? t : 0), hi = r.p + (b > 0 ? b : 0) + (t > 0 ? t : 0) + r.w;
  };
  const uint16_t *x0, *x1, *y0, *y1;
  span(x, x0, x1), span(y, y0, y1);
  if (x0 >= y1 || y0 >= x1) return false;
  const long long pitch = n > 1 ? x.st : B > 1 ? x.sb : 0;
  if (pitch <= 0 || (n > 1 && x.st != y.st) || (B > 1 && (x.sb != y.sb || x.sb % pitch))) return true;
  const long long d = ((y.p - x.p) % pitch + pitch) % pitch;  // y's first column in x's rows
  return d < x.w || d + y.w > pitch;
}

// Shared checks of a cache: C slots a multiple of 64, heads 64 or 128 wide, aligned pointers.
static int check_cache(const char* what, const void* kc, const void* vc, const void* ks, const void* vs, int B, int H,
                       int C, int D) {
  if (D != 64 && D != 128) return set_error(E_VARIANT, "%s: head_dim %d unsupported (64 or 128)", what, D);
  if (B < 0 || H <= 0 || C <= 0 || C % BLK)
    return set_error(E_SHAPE, "%s: B=%d H=%d C=%d (C a multiple of %d)", what, B, H, C, BLK);
  if ((long long)B * H > (1LL << 31) / 2) return set_error(E_SHAPE, "%s: B * H = %lld too large", what, (long long)B * H);
  if (B == 0) return OK;  // nothing is read: the pointers of an empty batch may be null
  if (!kc || !vc || !ks || !vs || !aligned16(kc) || !aligned16(vc) || (reinterpret_cast<uintptr_t>(ks) & 3) ||
      (reinterpret_cast<uintptr_t>(vs) & 3))
    return set_error(E_SHAPE, "%s: null or unaligned cache pointer (codes 16 bytes, scales 4)", what);
  return OK;
}

}  // namespace kv8
}  // namespace vt

extern "C" {

int vt_rope_kv8(cudaStream_t st, const uint16_t* qkv, long long sx_b, long long sx_t, int B, int n, int Hq, int H, int D,
                const float* cos_t, const float* sin_t, int tab, const int* lens, const int* pos, const int* counts,
                uint16_t* q, long long sq_b, long long sq_t, long long sq_h, int8_t* kc, int8_t* vc, float* ks, float* vs,
                int C) {
  using namespace vt;
  const int rc = kv8::check_cache("vt_rope_kv8", kc, vc, ks, vs, B, H, C, D);
  if (rc) return rc;
  if (n < 0 || Hq <= 0 || Hq % H || tab <= 0)
    return set_error(E_SHAPE, "vt_rope_kv8: n=%d Hq=%d H=%d tab=%d (Hq a multiple of H)", n, Hq, H, tab);
  if (B == 0 || n == 0) return OK;
  if (!qkv || !cos_t || !sin_t || !lens || !q || !aligned16(qkv) || !aligned16(q) || !aligned16(cos_t) || !aligned16(sin_t) ||
      (sx_b | sx_t | sq_b | sq_t | sq_h) % 8)
    return set_error(E_SHAPE, "vt_rope_kv8: null pointer, or pointers / strides not 16-byte aligned");
  const int nb = (n - 1) / kv8::BLK + 2 < C / kv8::BLK ? (n - 1) / kv8::BLK + 2 : C / kv8::BLK;
  const long long kv_units = 2LL * B * H * nb;
  long long qc = ((long long)B * n * Hq * (D / 8) + 127) / 128;
  if (qc > (1 << 20)) qc = 1 << 20;
  if (kv_units + qc > 0x7fffffffLL) return set_error(E_SHAPE, "vt_rope_kv8: grid too large (B=%d H=%d n=%d)", B, H, n);
  if (kv8::rows_meet({qkv, sx_b, sx_t, (Hq + 2LL * H) * D}, {q, sq_b, sq_t, (Hq - 1) * sq_h + D}, B, n))
    return set_error(E_SHAPE, "vt_rope_kv8: q overlaps qkv");
  kv8::AppendArgs a{qkv, sx_b, sx_t, B, n, Hq, H, C, tab, nb, cos_t, sin_t, lens, pos, counts, q, sq_b, sq_t, sq_h,
                    kc, vc, ks, vs, kv_units};
  if (D == 64) launch_k(kv8::rope_kv8_kernel<64>, (unsigned)(kv_units + qc), 128, 0, st, a);
  else launch_k(kv8::rope_kv8_kernel<128>, (unsigned)(kv_units + qc), 128, 0, st, a);
  return check_launch("vt_rope_kv8");
}

int vt_kv8_evict(cudaStream_t st, const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, int C,
                 const float* weights, const int* lens, int B, int H, int D, int keep, int recent, int8_t* dst_kc,
                 int8_t* dst_vc, float* dst_ks, float* dst_vs, int dst_C, float* dst_weights, int* dst_lens, int* index) {
  using namespace vt;
  int rc = kv8::check_cache("vt_kv8_evict", kc, vc, ks, vs, B, H, C, D);
  if (!rc) rc = kv8::check_cache("vt_kv8_evict (dst)", dst_kc, dst_vc, dst_ks, dst_vs, B, H, dst_C, D);
  if (rc) return rc;
  if (keep <= 0 || keep % kv8::BLK || keep > dst_C || recent < 0 || recent > keep)
    return set_error(E_SHAPE, "vt_kv8_evict: keep=%d (a multiple of %d, at most the destination's %d slots), recent=%d", keep,
                     kv8::BLK, dst_C, recent);
  if (C > kv8::MAX_EVICT) return set_error(E_SHAPE, "vt_kv8_evict: C=%d (at most %d)", C, kv8::MAX_EVICT);
  if (B == 0) return OK;
  if (!weights || !lens || !dst_weights || !dst_lens || !index) return set_error(E_SHAPE, "vt_kv8_evict: null pointer");
  const long long n = (long long)B * H, nc = n * C * D, nd = n * dst_C * D;
  const struct { const void* p; long long n; } src[] = {{kc, nc}, {vc, nc}, {ks, n * C / 16}, {vs, n * C / 16}, {weights, n * C * 4}, {lens, B * 4LL}},
      dst[] = {{dst_kc, nd}, {dst_vc, nd}, {dst_ks, n * dst_C / 16}, {dst_vs, n * dst_C / 16}, {dst_weights, n * dst_C * 4}, {dst_lens, B * 4LL}, {index, n * keep * 4}};
  for (const auto& s : src)
    for (const auto& d : dst)
      if (kv8::overlap(s.p, s.n, d.p, d.n)) return set_error(E_SHAPE, "vt_kv8_evict: the destination overlaps the source");
  const long long units = n * (keep / kv8::BLK);
  if (units > 0x7fffffffLL || n > 0x07ffffffLL)
    return set_error(E_SHAPE, "vt_kv8_evict: grid too large (B=%d H=%d keep=%d)", B, H, keep);
  kv8::EvictArgs a{kc, vc, ks, vs, weights, lens, B, H, C, keep, recent, dst_C, dst_kc, dst_vc, dst_ks, dst_vs, dst_weights, dst_lens, index};
  // Two warps for up to 2048 slots: a warp's share of a round is mostly not its keys.  Beyond, 1024 threads, and as many CTAs a
  // head as leave each thread at most 16 slots when there are fewer heads than SMs (8 heads of 131k slots, clusters of 8:
  // 39 us; clusters of 16 with half the threads 52 us, their barriers cost more than the keys), 32 otherwise
  const int most = n < sm_count() ? 16 : 32;
  if (C <= 2048) rc = kv8::launch_select<64, 32, 1>(st, a);
  else if (C <= most * 1024) rc = kv8::launch_select<1024, 32, 1>(st, a);
  else if (C <= most * 2048) rc = kv8::launch_select<1024, 32, 2>(st, a);
  else if (C <= most * 4096) rc = kv8::launch_select<1024, 32, 4>(st, a);
  else rc = kv8::launch_select<1024, 32, 8>(st, a);
  if (rc) return rc;
  if (D == 64) launch_k(kv8::kv8_gather_kernel<64>, (unsigned)units, 128, 0, st, a);
  else launch_k(kv8::kv8_gather_kernel<128>, (unsigned)units, 128, 0, st, a);
  return check_launch("vt_kv8_evict");
}

}  // extern "C"
