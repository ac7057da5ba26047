// Attention over the 8-bit cache: the entry point, and kernels for many rows.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {

// Rows of a kv head that the split kernel takes.
constexpr int FEW_ROWS = 32;
static bool few_rows(int n, int Hq, int H) { return (long long)n * (Hq / H) <= FEW_ROWS; }

// ---------------------------------------------------------------- attention
struct AttnArgs {
  const uint16_t* q;
  long long sq_b, sq_t, sq_h;
  const int8_t *kc, *vc;
  const float *ks, *vs;
  const int *lens, *counts;
  int B, n, Hq, H, C, causal;
  float scale_log2;
  uint16_t* out;
  long long so_b, so_t, so_h;
  float* w;
  const float* w_in;
  float* lse;  // [B][Hq][n]
};

__device__ __forceinline__ float dot16(const int8_t* k, const float* q) {
  const uint4 u = *reinterpret_cast<const uint4*>(k);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  float t = 0.f;
#pragma unroll
  for (int e = 0; e < 16; e++) t = fmaf((float)(int8_t)(w[e >> 2] >> (8 * (e & 3))), q[e], t);
  return t;
}

// CTA = one row and query head: 128 keys at a time, a running max and sum.
template <int D>
__global__ void __launch_bounds__(128) attn_kv8_row_kernel(AttnArgs a) {
  __shared__ float qs[D], ps[128], red[4];
  const int tid = threadIdx.x, i = blockIdx.x, hq = blockIdx.y, b = blockIdx.z;
  griddep_wait();
  griddep_launch();
  const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C);
  if (i >= s.cnt) return;
  const int T = a.causal ? s.len + i + 1 : s.len + s.cnt;
  const size_t bh = (size_t)b * a.H + hq / (a.Hq / a.H);
  const int8_t *k = a.kc + bh * a.C * D, *v = a.vc + bh * a.C * D;
  const float *ks = a.ks + bh * (a.C / BLK), *vs = a.vs + bh * (a.C / BLK);
  if (tid < D) qs[tid] = bf2f(a.q[b * a.sq_b + i * a.sq_t + hq * a.sq_h + tid]) * a.scale_log2;
  __syncthreads();
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int j0 = 0; j0 < T; j0 += 128) {
    const int j = j0 + tid;
    float x = -INFINITY;
    if (j < T) {
      x = 0.f;
      for (int d = 0; d < D; d += 16) x += dot16(k + (size_t)j * D + d, qs + d);
      x *= ks[j / BLK];
    }
    float mx = x;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
    const float alpha = exp2f(m - mn);
    ps[tid] = j < T ? exp2f(x - mn) : 0.f;
    m = mn;
    __syncthreads();
    l *= alpha;
    o *= alpha;
    for (int jj = 0; jj < min(128, T - j0); jj++) {
      l += ps[jj];
      if (tid < D) o = fmaf(ps[jj] * vs[(j0 + jj) / BLK], (float)v[(size_t)(j0 + jj) * D + tid], o);
    }
    __syncthreads();
  }
  if (tid < D) a.out[b * a.so_b + i * a.so_t + hq * a.so_h + tid] = f2bf(o / l);
  if (a.lse && tid == 0) a.lse[((size_t)b * a.Hq + hq) * a.n + i] = m + log2f(l);
}

// weights[b][h][j] = (j < len ? weights_in : 0) + sum over rows and the group's heads of 2^(score - lse); thread = key.
template <int D>
__global__ void __launch_bounds__(128) kv8_weights_row_kernel(AttnArgs a) {
  const int j = blockIdx.x * 128 + threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  griddep_wait();
  griddep_launch();
  const Seq s = seq_of(a.lens, a.counts, b, a.n, a.C);
  if (j >= s.len + s.cnt) return;
  const size_t bh = (size_t)b * a.H + h;
  const int8_t* k = a.kc + (bh * a.C + j) * D;
  const float ks = a.ks[bh * (a.C / BLK) + j / BLK];
  float kv[D];
  for (int d = 0; d < D; d++) kv[d] = (float)k[d];
  const int G = a.Hq / a.H;
  float acc = a.w_in && j < s.len ? a.w_in[bh * a.C + j] : 0.f;
  for (int i = a.causal ? max(j - s.len, 0) : 0; i < s.cnt; i++)
    for (int g = 0; g < G; g++) {
      const uint16_t* q = a.q + b * a.sq_b + i * a.sq_t + (h * G + g) * a.sq_h;
      float x = 0.f;
      for (int d = 0; d < D; d++) x = fmaf(bf2f(q[d]) * a.scale_log2, kv[d], x);
      acc += exp2f(x * ks - a.lse[((size_t)b * a.Hq + h * G + g) * a.n + i]);
    }
  a.w[bh * a.C + j] = acc;
}

}  // namespace kv8
}  // namespace vt

extern "C" {

long long vt_attn_kv8_ws_bytes(int B, int n, int Hq, int H, int D, int C, int weights) {
  if (B <= 0 || n <= 0 || Hq <= 0 || H <= 0 || Hq % H || C <= 0 || (D != 64 && D != 128)) return 0;
  // what n tokens need, and any fewer that may follow with the same workspace
  const int few = vt::kv8::FEW_ROWS / (Hq / H), nf = n < few ? n : few;
  const long long split = nf ? vt::kv8::split::make_plan(B, nf, Hq, H, D, C, weights != 0, vt::sm_count()).bytes : 0;
  const long long many = n > few && weights ? (long long)B * n * Hq * 4 : 0;
  return split > many ? split : many;
}

int vt_attn_kv8(cudaStream_t st, const uint16_t* q, long long sq_b, long long sq_t, long long sq_h, const int8_t* kc,
                const int8_t* vc, const float* ks, const float* vs, int C, const int* lens, const int* counts, int B,
                int n, int Hq, int H, int D, int causal, float scale, uint16_t* out, long long so_b, long long so_t,
                long long so_h, float* weights, const float* weights_in, void* ws, long long ws_bytes) {
  using namespace vt;
  const int rc = kv8::check_cache("vt_attn_kv8", kc, vc, ks, vs, B, H, C, D);
  if (rc) return rc;
  if (n < 0 || Hq <= 0 || Hq % H) return set_error(E_SHAPE, "vt_attn_kv8: n=%d Hq=%d H=%d (Hq a multiple of H)", n, Hq, H);
  if (B == 0 || n == 0) return OK;
  if (!q || !lens || !out || !aligned16(q) || !aligned16(out) || (sq_b | sq_t | sq_h | so_b | so_t | so_h) % 8)
    return set_error(E_SHAPE, "vt_attn_kv8: null pointer, or pointers / strides not 16-byte aligned");
  if (weights_in && !weights) return set_error(E_SHAPE, "vt_attn_kv8: weights_in without weights");
  const long long need = vt_attn_kv8_ws_bytes(B, n, Hq, H, D, C, weights != nullptr);
  if (need && (!ws || !aligned16(ws) || ws_bytes < need))
    return set_error(E_SHAPE, "vt_attn_kv8: workspace of %lld bytes, %lld needed (16-byte aligned)", ws ? ws_bytes : 0LL, need);
  if (B > 65535 || Hq > 65535) return set_error(E_SHAPE, "vt_attn_kv8: B=%d or Hq=%d too large", B, Hq);
  if (kv8::few_rows(n, Hq, H)) {
    const kv8::split::Plan p = kv8::split::make_plan(B, n, Hq, H, D, C, weights != nullptr, sm_count());
    if (B > kv8::split::MAXB || (long long)B * H * p.rg * (C / kv8::split::keys_per_tile(D)) > 0x40000000LL)
      return set_error(E_SHAPE, "vt_attn_kv8: B=%d (at most %d) or B * H * C too large", B, kv8::split::MAXB);
    char* w8 = static_cast<char*>(ws);
    kv8::split::Args a{q, sq_b, sq_t, sq_h, kc, vc, ks, vs, lens, counts, B, n, Hq / H, H, C, causal, p.rows, p.rg, p.ctas,
                       scale * kv8::LOG2E, out, so_b, so_t, so_h, (float*)(w8 + p.o_off), (float2*)(w8 + p.ml_off),
                       (float2*)(w8 + p.full_off), weights ? (float*)(w8 + p.s_off) : nullptr, weights, weights_in};
    if (D == 64) return p.nt == 1 ? kv8::split::launch<64, 1>(st, a) : p.nt == 2 ? kv8::split::launch<64, 2>(st, a) : kv8::split::launch<64, 4>(st, a);
    return p.nt == 1 ? kv8::split::launch<128, 1>(st, a) : kv8::split::launch<128, 2>(st, a);
  }
  kv8::AttnArgs a{q, sq_b, sq_t, sq_h, kc, vc, ks, vs, lens, counts, B, n, Hq, H, C, causal,
                  scale * kv8::LOG2E, out, so_b, so_t, so_h, weights, weights_in, weights ? (float*)ws : nullptr};
  const dim3 grid(n, Hq, B), wgrid((C + 127) / 128, H, B);
  if (D == 64) launch_k(kv8::attn_kv8_row_kernel<64>, grid, 128, 0, st, a);
  else launch_k(kv8::attn_kv8_row_kernel<128>, grid, 128, 0, st, a);
  if (weights) {
    if (D == 64) launch_k(kv8::kv8_weights_row_kernel<64>, wgrid, 128, 0, st, a);
    else launch_k(kv8::kv8_weights_row_kernel<128>, wgrid, 128, 0, st, a);
  }
  return check_launch("vt_attn_kv8");
}

}  // extern "C"
