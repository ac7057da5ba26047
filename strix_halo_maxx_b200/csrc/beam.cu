// The choice of a beam search: of a group of F beams the k continuations with the largest
//   total(f, v) = score[f] + logit[f, v] - log sum_w exp(logit[f, w]),
// in order, the lowest f V + v first where totals are equal.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace beam {

constexpr int MAX_BEAMS = 64, MAX_K = 128;

struct Args {
  const void* logits;
  long long ld;
  int f32;
  const float* scores;
  const uint8_t* done;
  int F, V, k, eos;
  float* out_scores;
  int *out_parents, *out_tokens;
  uint8_t* out_done;
  double2* lse;  // of each row its largest logit and the log of the sum of exponentials above it
};

__device__ __forceinline__ float logit(const Args& a, long long row, int v) {
  return a.f32 ? static_cast<const float*>(a.logits)[row * a.ld + v] : bf2f(static_cast<const uint16_t*>(a.logits)[row * a.ld + v]);
}

__global__ void __launch_bounds__(256) beam_lse_kernel(Args a) {
  __shared__ float red[8];
  __shared__ double sum[8];
  const int tid = threadIdx.x, lane = tid & 31;
  griddep_wait();
  griddep_launch();
  float mx = -INFINITY;
  for (int v = tid; v < a.V; v += 256) mx = fmaxf(mx, logit(a, blockIdx.x, v));
  for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
  if (lane == 0) red[tid / 32] = mx;
  __syncthreads();
  for (int w = 0; w < 8; w++) mx = fmaxf(mx, red[w]);
  double s = 0.;
  for (int v = tid; v < a.V; v += 256) s += expf(logit(a, blockIdx.x, v) - mx);
  for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
  if (lane == 0) sum[tid / 32] = s;
  __syncthreads();
  if (tid) return;
  for (int w = 1; w < 8; w++) s += sum[w];
  a.lse[blockIdx.x] = make_double2(mx, log(s));
}

// One group a CTA; round j takes the best candidate behind the one of round j - 1.
__global__ void __launch_bounds__(256) beam_pick_kernel(Args a) {
  __shared__ double top[8];
  __shared__ long long top_at[8];
  const int tid = threadIdx.x, g = blockIdx.x;
  griddep_wait();
  griddep_launch();
  double last = INFINITY;
  long long last_at = -1;
  for (int j = 0; j < a.k; j++) {
    double best = -INFINITY;
    long long at = -1;
    for (int f = 0; f < a.F; f++) {
      const long long row = (long long)g * a.F + f;
      const bool held = a.done && a.done[row];
      for (int v = held ? a.eos + (tid ? a.V : 0) : tid; v < (held ? a.eos + 1 : a.V); v += 256) {
        const double t = held ? a.scores[row] : a.scores[row] + (((double)logit(a, row, v) - a.lse[row].x) - a.lse[row].y);
        const long long c = (long long)f * a.V + v;
        if ((t < last || (t == last && c > last_at)) && t > best) best = t, at = c;
      }
    }
    for (int x = 16; x > 0; x >>= 1) {
      const double t = __shfl_xor_sync(0xffffffffu, best, x);
      const long long c = __shfl_xor_sync(0xffffffffu, at, x);
      if (t > best || (t == best && t > -INFINITY && c < at)) best = t, at = c;
    }
    if (tid % 32 == 0) top[tid / 32] = best, top_at[tid / 32] = at;
    __syncthreads();
    for (int w = 0; w < 8; w++)
      if (top[w] > best || (top[w] == best && best > -INFINITY && top_at[w] < at)) best = top[w], at = top_at[w];
    __syncthreads();
    if (tid == 0) {
      const long long o = (long long)g * a.k + j;
      const int f = at < 0 ? j % a.F : (int)(at / a.V), v = at < 0 ? -1 : (int)(at % a.V);
      a.out_scores[o] = (float)best;
      a.out_parents[o] = g * a.F + f;
      a.out_tokens[o] = v;
      a.out_done[o] = at < 0 || v == a.eos || (a.done && a.done[(long long)g * a.F + f]);
    }
    if (at >= 0) last = best, last_at = at;
    else last = -INFINITY;
  }
}

}  // namespace beam
}  // namespace vt

extern "C" {

long long vt_beam_select_ws_bytes(int S, int F, int V, int k) {
  if (S <= 0 || F <= 0 || F > vt::beam::MAX_BEAMS || V <= 0 || k <= 0 || k > vt::beam::MAX_K) return 0;
  return 16LL * S * F;
}

int vt_beam_select(cudaStream_t st, const void* logits, long long ld, int f32, const float* scores, const uint8_t* done, int S, int F,
                   int V, int k, int eos, float* out_scores, int* out_parents, int* out_tokens, uint8_t* out_done, void* ws,
                   long long ws_bytes) {
  using namespace vt;
  const char* what = "vt_beam_select";
  if (S < 0 || F <= 0 || F > beam::MAX_BEAMS || V <= 0 || k <= 0 || k > beam::MAX_K)
    return set_error(E_SHAPE, "%s: S=%d F=%d V=%d k=%d (1 .. %d beams, 1 .. %d candidates)", what, S, F, V, k, beam::MAX_BEAMS, beam::MAX_K);
  if (ld < V) return set_error(E_SHAPE, "%s: a pitch of %lld for %d logits", what, ld, V);
  if (eos >= V || (done && eos < 0)) return set_error(E_SHAPE, "%s: eos=%d of %d words", what, eos, V);
  if (S == 0) return OK;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !out_done || (reinterpret_cast<uintptr_t>(logits) & (f32 ? 3 : 1)))
    return set_error(E_SHAPE, "%s: null or unaligned pointer", what);
  const long long need = vt_beam_select_ws_bytes(S, F, V, k);
  if (!ws || !aligned16(ws) || ws_bytes < need)
    return set_error(E_SHAPE, "%s: workspace of %lld bytes, %lld needed (16-byte aligned)", what, ws ? ws_bytes : 0LL, need);
  if ((long long)S * F > 0xffffffLL) return set_error(E_SHAPE, "%s: S=%d too large", what, S);
  const long long rows = (long long)S * F, n = (long long)S * k, es = f32 ? 4 : 2;
  const struct { const void* p; long long n; } in[] = {{logits, ((rows - 1) * ld + V) * es}, {scores, rows * 4}, {done, done ? rows : 0}, {ws, need}},
      outs[] = {{out_scores, n * 4}, {out_parents, n * 4}, {out_tokens, n * 4}, {out_done, n}};
  for (const auto& x : in)
    for (const auto& y : outs)
      if (x.n && kv8::overlap(x.p, x.n, y.p, y.n)) return set_error(E_SHAPE, "%s: an output overlaps an input", what);
  beam::Args a{logits, ld, f32, scores, done, F, V, k, eos, out_scores, out_parents, out_tokens, out_done, (double2*)ws};
  launch_k(beam::beam_lse_kernel, S * F, 256, 0, st, a);
  launch_k(beam::beam_pick_kernel, S, 256, 0, st, a);
  return check_launch(what);
}

}  // extern "C"
