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
__device__ __forceinline__ Seq seq_of(const int* lens, const int* counts, int b, int n, int C) {
  int len = lens[b], cnt = counts ? counts[b] : n;
  const bool bad = len < 0 || len > C || cnt < 0 || cnt > n || cnt > C - len;
  len = min(max(len, 0), C);
  cnt = min(min(max(cnt, 0), n), C - len);
  if (bad && threadIdx.x == 0) atomicOr(&g_status, (unsigned int)ST_KV8_RANGE);
  return {len, cnt};
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

// rint(x / s) clamped to +-127 (s > 0), as a byte.
__device__ __forceinline__ uint32_t code_of(float x, float s) {
  const float r = fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.f), 127.f);
  return (uint32_t)(int)r & 0xffu;
}
__device__ __forceinline__ uint2 codes8(const float* x, float s) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; e++) w[e >> 2] |= code_of(x[e], s) << (8 * (e & 3));
  return make_uint2(w[0], w[1]);
}

// CTA = one block of 64 slots of one (sequence, head, K or V) that gets new tokens, or a run of q chunks.
// Block scale: max |x| / 127 over the new tokens when the block held none (or only zeros: scale 0); else the old
// scale, doubled until the new tokens fit, the held codes shifted by as many bits (rint(c / 2^j), half to even).
// Doubling keeps a held value within half a step of each scale it went through, 1/2 + 1/4 + ... < 1 step of the
// last, however many tokens arrive one by one; scales that grew just enough would add up to one rounding for
// each token of the block.  A NaN or an infinity among the values makes the block's scale NaN.
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
      const int p = min(max((a.pos ? a.pos[b] : s.len) + i, 0), a.tab - 1);
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
  const int p0 = a.pos ? a.pos[b] : s.len;
  if (tid == 0 && w == 0 && (p0 < 0 || p0 + i0 + m > a.tab)) atomicOr(&g_status, (unsigned int)ST_KV8_RANGE);
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
      const int p = min(max(p0 + i0 + row, 0), a.tab - 1);
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
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int t = tid + 128 * k, row = t / CH, c = t % CH;
    if (row >= m) continue;
    uint2 o = make_uint2(0, 0);
    if (sc > 0.f) {  // neither zero nor NaN
      const uint32_t x[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        f[2 * e] = __uint_as_float(x[e] << 16);
        f[2 * e + 1] = __uint_as_float(x[e] & 0xffff0000u);
      }
      o = codes8(f, sc);
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

// Order of weights as unsigned numbers: -inf .. +inf, NaN above all, -0 equal to 0.
__device__ __forceinline__ uint32_t order_of(float f) {
  if (isnan(f)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f == 0.f ? 0.f : f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// CTA = one head: the (keep - recent) largest of the slots before the recent ones, by radix selection on 8 bits a
// pass, then their slots in order (ties: the lowest slots), the recent ones behind them.
constexpr int SEL = 1024;
__global__ void __launch_bounds__(SEL) kv8_select_kernel(EvictArgs a) {
  __shared__ unsigned int hist[256], warp_cnt[32];
  __shared__ unsigned int sh_prefix, sh_left;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.x, b = blockIdx.y;
  griddep_wait();
  griddep_launch();
  int len = a.lens[b];
  if ((len < 0 || len > a.C) && tid == 0) atomicOr(&g_status, (unsigned int)ST_KV8_RANGE);
  len = min(max(len, 0), a.C);
  const size_t bh = (size_t)b * a.H + h;
  const float* w = a.w + bh * a.C;
  float* dw = a.dw + bh * a.Cd;
  int* idx = a.index + bh * a.keep;
  if (h == 0 && tid == 0) a.dlens[b] = min(len, a.keep);
  if (len <= a.keep) {
    for (int j = tid; j < len; j += SEL) {
      idx[j] = j;
      dw[j] = w[j];
    }
    return;
  }
  const int N = len - a.recent, want = a.keep - a.recent;
  unsigned int prefix = 0, left = want;  // the want-th largest key's leading bits, and its rank among those that share them
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int j = tid; j < N; j += SEL) {
      const uint32_t u = order_of(w[j]);
      if (shift == 24 || (u >> (shift + 8)) == prefix) atomicAdd(&hist[(u >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      unsigned int acc = 0;
      int d = 255;
      for (; d > 0 && acc + hist[d] < left; d--) acc += hist[d];
      sh_prefix = (prefix << 8) | (unsigned int)d;
      sh_left = left - acc;
    }
    __syncthreads();
    prefix = sh_prefix;
    left = sh_left;
  }
  unsigned int base = 0, ties = 0;  // slots kept and ties seen so far
  for (int j0 = 0; j0 < N && want > 0; j0 += SEL) {
    const int j = j0 + tid;
    const uint32_t u = j < N ? order_of(w[j]) : 0u;
    const bool gt = j < N && u > prefix, eq = j < N && u == prefix;
    const unsigned int bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    const unsigned int below = (1u << lane) - 1u;
    if (lane == 0) warp_cnt[warp] = __popc(bg) | (__popc(be) << 16);
    __syncthreads();
    unsigned int cg = 0, ce = 0, tg = 0, te = 0;
    for (int i = 0; i < 32; i++) {
      const unsigned int c = warp_cnt[i];
      if (i < warp) {
        cg += c & 0xffffu;
        ce += c >> 16;
      }
      tg += c & 0xffffu;
      te += c >> 16;
    }
    cg += __popc(bg & below);
    ce += __popc(be & below);
    const unsigned int eq_before = min(ties + ce, left);  // ties kept before this slot
    if (gt || (eq && ties + ce < left)) {
      const unsigned int at = base + cg + (eq_before - min(ties, left));
      idx[at] = j;
      dw[at] = w[j];
    }
    base += tg + (min(ties + te, left) - min(ties, left));
    ties += te;
    __syncthreads();
  }
  for (int r = tid; r < a.recent; r += SEL) {
    idx[want + r] = len - a.recent + r;
    dw[want + r] = w[len - a.recent + r];
  }
}

// CTA = one block of 64 kept tokens of one (sequence, head, K or V): their values code * scale (rounded to fp32), the
// scale max |value| / 127 and the codes rint(value / scale).  Sequences that lost nothing are copied.
template <int D>
__global__ void __launch_bounds__(128) kv8_gather_kernel(EvictArgs a) {
  constexpr int CH = D / 8, PER = BLK * CH / 128;
  __shared__ float red[4];
  const int tid = threadIdx.x, w = blockIdx.x & 1;
  griddep_wait();
  griddep_launch();
  long long u = blockIdx.x >> 1;
  const int nb = a.keep / BLK, blk = (int)(u % nb);
  u /= nb;
  const int h = (int)(u % a.H), b = (int)(u / a.H);
  const int len = min(max(a.lens[b], 0), a.C);
  const int rows = min(len, a.keep) - blk * BLK;
  if (rows <= 0) return;
  const size_t bh = (size_t)b * a.H + h;
  const int8_t* src = (w ? a.vc : a.kc) + bh * a.C * D;
  const float* ss = (w ? a.vs : a.ks) + bh * (a.C / BLK);
  int8_t* dst = (w ? a.dvc : a.dkc) + (bh * a.Cd + (size_t)blk * BLK) * D;
  float* ds = (w ? a.dvs : a.dks) + bh * (a.Cd / BLK) + blk;
  const int* idx = a.index + bh * a.keep + blk * BLK;
  const bool copy = len <= a.keep;
  uint2 c[PER];
  float sc[PER], top = 0.f;
  bool odd = false;
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int t = tid + 128 * k, row = t / CH;
    c[k] = make_uint2(0, 0);
    sc[k] = 0.f;
    if (row >= rows) continue;
    const int j = copy ? blk * BLK + row : idx[row];
    c[k] = *reinterpret_cast<const uint2*>(src + (size_t)j * D + 8 * (t % CH));
    sc[k] = ss[j / BLK];
    odd |= isnan(sc[k]);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int x = (int8_t)((e < 4 ? c[k].x : c[k].y) >> (8 * (e & 3)));
      top = fmaxf(top, fabsf(__fmul_rn((float)x, sc[k])));
    }
  }
  if (copy) {
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int t = tid + 128 * k, row = t / CH;
      if (row < rows) *reinterpret_cast<uint2*>(dst + (size_t)row * D + 8 * (t % CH)) = c[k];
    }
    if (tid == 0) *ds = ss[blk];
    return;
  }
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(odd ? INFINITY : top)));
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float s = isinf(top) ? __uint_as_float(0x7fc00000u) : __fdiv_rn(top, 127.f);
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int t = tid + 128 * k, row = t / CH;
    if (row >= rows) continue;
    uint2 o = make_uint2(0, 0);
    if (s > 0.f) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; e++)
        f[e] = __fmul_rn((float)(int8_t)((e < 4 ? c[k].x : c[k].y) >> (8 * (e & 3))), sc[k]);
      o = codes8(f, s);
    }
    *reinterpret_cast<uint2*>(dst + (size_t)row * D + 8 * (t % CH)) = o;
  }
  if (tid == 0) *ds = s;
}

static bool overlap(const void* p, long long n, const void* q, long long m) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return a < b + (uintptr_t)m && b < a + (uintptr_t)n;
}

// Shared checks of a cache: C slots a multiple of 64, heads 64 or 128 wide, aligned pointers.
static int check_cache(const char* what, const void* kc, const void* vc, const void* ks, const void* vs, int B, int H,
                       int C, int D) {
  if (D != 64 && D != 128) return set_error(E_VARIANT, "%s: head_dim %d unsupported (64 or 128)", what, D);
  if (B < 0 || H <= 0 || C <= 0 || C % BLK)
    return set_error(E_SHAPE, "%s: B=%d H=%d C=%d (C a multiple of %d)", what, B, H, C, BLK);
  if ((long long)B * H > (1LL << 31) / 2) return set_error(E_SHAPE, "%s: B * H = %lld too large", what, (long long)B * H);
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
  if (B == 0) return OK;
  if (!weights || !lens || !dst_weights || !dst_lens || !index) return set_error(E_SHAPE, "vt_kv8_evict: null pointer");
  const long long n = (long long)B * H, nc = n * C * D, nd = n * dst_C * D;
  const struct { const void* p; long long n; } src[] = {{kc, nc}, {vc, nc}, {ks, n * C / 16}, {vs, n * C / 16}, {weights, n * C * 4}, {lens, B * 4LL}},
      dst[] = {{dst_kc, nd}, {dst_vc, nd}, {dst_ks, n * dst_C / 16}, {dst_vs, n * dst_C / 16}, {dst_weights, n * dst_C * 4}, {dst_lens, B * 4LL}, {index, n * keep * 4}};
  for (const auto& s : src)
    for (const auto& d : dst)
      if (kv8::overlap(s.p, s.n, d.p, d.n)) return set_error(E_SHAPE, "vt_kv8_evict: the destination overlaps the source");
  const long long units = 2LL * B * H * (keep / kv8::BLK);
  if (B > 65535 || units > 0x7fffffffLL) return set_error(E_SHAPE, "vt_kv8_evict: grid too large (B=%d H=%d keep=%d)", B, H, keep);
  kv8::EvictArgs a{kc, vc, ks, vs, weights, lens, B, H, C, keep, recent, dst_C, dst_kc, dst_vc, dst_ks, dst_vs, dst_weights, dst_lens, index};
  launch_k(kv8::kv8_select_kernel, dim3(H, B), kv8::SEL, 0, st, a);
  if (D == 64) launch_k(kv8::kv8_gather_kernel<64>, (unsigned)units, 128, 0, st, a);
  else launch_k(kv8::kv8_gather_kernel<128>, (unsigned)units, 128, 0, st, a);
  return check_launch("vt_kv8_evict");
}

}  // extern "C"
