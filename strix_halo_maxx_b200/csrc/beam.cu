// The choice of a beam search: of a group of F beams the k continuations with the largest
//   total(f, v) = score[f] + logit[f, v] - log sum_w exp(logit[f, w]),
// in order, the lowest f V + v first where totals are equal.  Within a row totals follow its logits, so a row's k best words are found
// without its sum, and the logits are read once:
//   beam_words_kernel   a chunk of a row stays in registers: its largest logit, its sum of exponentials, and its k best words in order;
//   beam_pick_kernel    a group: the rows' sums, the totals of the chunks' words, the k best of them.
// The k best of many, in both: maxima of parts, more than k of them; the k'th largest of these maxima is a bound that k values
// reach, and few others; those that reach it are gathered and each counts the ones ahead of it.  The gathered are compared
// as (value, place), no two of them equal, so no order of arrival shows; fewer than k parts have any above the bound.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace beam {

constexpr int MAX_BEAMS = 64, MAX_K = 128, T = 256, TP = 512;  // threads of a CTA of the two kernels
// Words of a thread: with 8 or 16 for calls of few rows, to fill the GPU, their lists cost the second kernel more (32 x 8 rows of 51,200 bf16:
// 24 us with 32, 29 with 16, 37 with 8; 4 x 8 rows: 14, 17, 21; 1 x 4 rows fp32: 8.7, 9.1, 8.8).
constexpr int E = 32;
constexpr int CAP = 2048;                            // totals that beam_pick_kernel gathers; beyond, one by one

struct Args {
  const void* logits;
  long long ld;
  const float* scores;
  const uint8_t* done;
  int F, V, k, eos, chunks;
  float* out_scores;
  int *out_parents, *out_tokens;
  uint8_t* out_done;
  double2* sums;             // [rows][chunks] largest logit, sum of exponentials of the differences to it
  unsigned long long* words; // [rows][chunks][k] (logit, place), best first; 0: none
};

// Parts of a chunk whose maxima are compared, T / parts threads each: 2 k or more.  The best k of 2 k parts leave about 1.4 k words to
// gather, and there are as many comparisons as parts squared (16 x 32 rows of 100,003 fp32, k = 32: 69 us, with 4 k parts 75).
__host__ __device__ inline int parts_of(int k) { return k <= 16 ? 32 : k <= 32 ? 64 : k <= 64 ? 128 : 256; }

// Numbers in the order of floats (zeros of both signs are one), and back.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
// A logit and its word as one number: larger logits first, of equal ones the lowest word; never 0.
__device__ __forceinline__ unsigned long long key_of(float x, int v) { return (unsigned long long)ordered(x) << 32 | (uint32_t)~v; }
__device__ __forceinline__ float key_logit(unsigned long long key) { return unordered((uint32_t)(key >> 32)); }

template <typename Word>
__device__ __forceinline__ float load_word(const Word* p) {
  if constexpr (sizeof(Word) == 4) return __ldg(p);
  else return bf2f(__ldg(p));
}
// Words v0 + (r T + thread) VEC ..; -inf behind the row's end.
template <typename Word, int VEC>
__device__ __forceinline__ void load_chunk(const Word* row, int v0, int V, float (&x)[E]) {
  const Word* p = row + v0 + (int)threadIdx.x * VEC;
  const bool whole = v0 + T * E <= V;
  const int left = V - v0 - (int)threadIdx.x * VEC;
  if (VEC == 1 && whole) {
#pragma unroll
    for (int r = 0; r < E; r++) x[r] = load_word(p + r * T);
    return;
  }
#pragma unroll
  for (int r = 0; r < E / VEC; r++) {
    if (VEC > 1 && (whole || r * T * VEC + VEC <= left)) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(p + r * T * VEC));
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < VEC; e++)
        x[r * VEC + e] = sizeof(Word) == 4 ? __uint_as_float(u[e % 4]) : __uint_as_float(e & 1 ? u[e / 2 % 4] & 0xffff0000u : u[e / 2 % 4] << 16);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++) x[r * VEC + e] = r * T * VEC + e < left ? load_word(p + r * T * VEC + e) : -INFINITY;
    }
  }
}

// CTA = T E words of a row.  Bound with many rows: a chunk's rounds of barriers, of which four CTAs an SM hide part (16 x 32 rows of 100,003
// fp32: 53 us, 3.9 TB/s; 57 % of the cycles issue, 20 instructions a word), with few the latency of one chunk.
template <typename Word, int VEC>
__global__ void __launch_bounds__(T) beam_words_kernel(Args a) {
  constexpr int FOUND = T * E / 2;  // words above the bound are of at most k of 2 k parts or more
  __shared__ float sh_max[T / 32];
  __shared__ double sh_sum[T / 32];
  __shared__ __align__(16) uint32_t part[T];
  __shared__ unsigned long long found[FOUND];
  __shared__ float bound;
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.k;
  const long long row = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x % a.chunks, v0 = chunk * (T * E);
  griddep_wait();
  griddep_launch();
  if (a.done && a.done[row]) return;  // its words are not looked at
  float x[E];
  const Word* words = static_cast<const Word*>(a.logits) + row * a.ld;
  load_chunk<Word, VEC>(words, v0, a.V, x);
  auto word = [&](int e) { return v0 + ((e / VEC) * T + tid) * VEC + e % VEC; };
  // ---- the largest logit of the thread, its part and the chunk
  float mx = x[0];
#pragma unroll
  for (int e = 1; e + 1 < E; e += 2) mx = max3f(mx, x[e], x[e + 1]);
  mx = fmaxf(fmaxf(mx, x[E - 1]), -INFINITY);  // NaN only where the thread has nothing else
  const int parts = parts_of(k), per = T / parts;
  float top = mx, best = mx;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (2 * d == per) best = top;
  }
  if (lane == 0) sh_max[warp] = top;
  // a part's maximum with its number in the lowest bits: no two are equal, and the bound is at most 2^-15 of a value low
  const uint32_t number = parts - 1, mine = (ordered(best) & ~number) | (number - tid / per);
  if (tid % per == 0) part[tid / per] = mine;
  if (tid == 0) count = 0, bound = -INFINITY;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < T / 32; w++) top = fmaxf(top, sh_max[w]);
  // ---- a part's rank among the maxima, its threads taking a share of them each; the k'th is the bound
  {
    int ahead = 0;
    for (int i = tid % per; i < parts / 4; i += per) {
      const uint4 y = reinterpret_cast<const uint4*>(part)[i];
      ahead += (y.x > mine) + (y.y > mine) + (y.z > mine) + (y.w > mine);
    }
    for (int d = 1; d < per; d <<= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, d);
    if (tid % per == 0 && ahead == k - 1 && best > -INFINITY) bound = unordered(mine & ~number);  // -inf where fewer than k parts have a word
  }
  // ---- sum of exponentials: fp32 within the 64 words of two lanes, 64 bits from there on (a sum in fp32 throughout lost what many unlikely
  // words add to a likely one).  A chunk of -inf adds nothing, a NaN or +inf makes it NaN
  {
    const float ref = top == -INFINITY ? 0.f : top;
    const unsigned long long ref2 = f2_pack(-ref, -ref), log2e = f2_pack(1.4426950408889634f, 1.4426950408889634f);
    unsigned long long s2 = 0ull;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      float y0, y1;
      f2_unpack(f2_mul(f2_add(f2_pack(x[e], x[e + 1]), ref2), log2e), y0, y1);
      s2 = f2_add(s2, f2_pack(ex2_approx(y0), ex2_approx(y1)));
    }
    float s, s_odd;
    f2_unpack(s2, s, s_odd);
    s += s_odd;
    double sum = s + __shfl_xor_sync(0xffffffffu, s, 16);
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) sh_sum[warp] = sum;
  }
  __syncthreads();
  // ---- gather the words that reach the bound.  They are few: the others' only cost is a bit
  const float lim = bound == -INFINITY ? -3.402823466e38f : bound;
  uint32_t hits = 0;
  if (__any_sync(0xffffffffu, mx >= lim))
#pragma unroll
  for (int e = 0; e < E; e++)
    asm("{\n\t.reg .pred p;\n\tsetp.ge.f32 p, %1, %2;\n\t@p or.b32 %0, %0, %3;\n\t}" : "+r"(hits) : "f"(x[e]), "f"(lim), "r"(1u << e));
  for (; hits; hits &= hits - 1) {
    const int v = word(__ffs(hits) - 1), n = atomicAdd(&count, 1);
    if (n < FOUND) found[n] = key_of(load_word(words + v), v);
  }
  if (tid == 0) {
    double s = 0.;
#pragma unroll
    for (int w = 0; w < T / 32; w++) s += sh_sum[w];
    a.sums[blockIdx.x] = make_double2(top, s);
  }
  __syncthreads();
  int n = count;
  if (n > FOUND) {  // equal logits in crowds (words banned by the lowest value): the exact bound, what is above it, then its first words
    if (tid % per == 0) part[tid / per] = __float_as_uint(best);
    __syncthreads();
    if (tid == 0) count = 0;
    int ahead = 0;
    for (int i = tid % per; i < parts; i += per) {
      const float y = __uint_as_float(part[i]);
      ahead += y > best || (y == best && i < tid / per);
    }
    for (int d = 1; d < per; d <<= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, d);
    if (tid % per == 0 && ahead == k - 1) bound = best;
    __syncthreads();
    const float lim = bound;  // of fewer than k parts there are words above it
#pragma unroll
    for (int e = 0; e < E; e++)
      if (x[e] > lim) found[atomicAdd(&count, 1)] = key_of(x[e], word(e));
    __syncthreads();
    n = count;
    if (warp == 0) {
      int got = n;
      for (int v = v0 + lane; got < k; v += 32) {
        const bool is = v < a.V && load_word(words + v) == lim;
        const uint32_t all = __ballot_sync(0xffffffffu, is);
        const int at = got + __popc(all & ((1u << lane) - 1));
        if (is && at < k) found[at] = key_of(lim, v);
        got += __popc(all);
        if (__all_sync(0xffffffffu, v >= min(a.V, v0 + T * E))) break;
      }
    }
    n = max(n, k);  // few parts may hold more than k words above it
    __syncthreads();
  }
  unsigned long long* to = a.words + (long long)blockIdx.x * k;
  for (int i = tid; i < n; i += T) {
    const unsigned long long key = found[i];
    int ahead = 0;
    for (int j = 0; j < n; j++) ahead += found[j] > key;
    if (ahead < k) to[ahead] = key;
  }
  for (int i = n + tid; i < k; i += T) to[i] = 0;
}

// A continuation: its total, beam, and logit with word; a total of -inf for none.  Equal totals go by beam, then by logit (which a total of
// 64 bits may have lost) and word.
struct Total {
  double t;
  unsigned long long key;
  int f;
};
__device__ __forceinline__ bool ahead_of(const Total& x, const Total& y) {
  return x.t > y.t || (x.t == y.t && (x.f < y.f || (x.f == y.f && x.key > y.key)));
}
__device__ __forceinline__ Total shfl_xor(const Total& x, int d) {
  return {__shfl_xor_sync(0xffffffffu, x.t, d), __shfl_xor_sync(0xffffffffu, x.key, d), __shfl_xor_sync(0xffffffffu, x.f, d)};
}

// CTA = a group.  Bound: latency, of two trips to L2 and the rounds of comparisons (1 x 4 rows: 4 us of 8.7, 16 x 32 rows of 13 chunks: 15 of 69).
__global__ void __launch_bounds__(TP) beam_pick_kernel(Args a) {
  __shared__ double sh_top[MAX_BEAMS], sh_log[MAX_BEAMS], sh_score[MAX_BEAMS];
  __shared__ double part_t[TP], found_t[CAP];
  __shared__ unsigned long long part_key[TP], found_key[CAP];
  __shared__ uint8_t part_f[TP], found_f[CAP];
  __shared__ uint8_t sh_done[MAX_BEAMS];
  __shared__ Total bound;
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.k, F = a.F;
  const long long row0 = (long long)blockIdx.x * F;
  griddep_wait();
  griddep_launch();
  // every list is dealt out to `deal` runs (entries j, j + deal, ..: in order too); run r is of list r % lists, thread t takes runs
  // t, t + TP, .., and threads p, p + parts, .. are a part: the best words of one beam stand in many parts
  const int lists = F * a.chunks, parts = k <= 16 ? 64 : k <= 32 ? 128 : 256, per = TP / parts;
  int deal = 1;
  while (lists * deal < 2 * TP && deal < k) deal <<= 1;
  const int runs = lists * deal;
  // the first entries of a thread's first runs are fetched while the sums are worked out
  constexpr int AHEAD = 4;
  unsigned long long head[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; i++) {
    const int r = tid + i * TP;
    head[i] = r < runs && r / lists < k ? a.words[(row0 * a.chunks + r % lists) * k + r / lists] : 0;
  }
  // ---- of each row the largest logit and the log of its sum, a warp a row
  for (int f = warp; f < F; f += TP / 32) {
    const bool done = a.done && a.done[row0 + f];
    double top = -INFINITY, sum = 0.;
    if (!done) {
      const double2* s = a.sums + (row0 + f) * a.chunks;
      const double2 mine = lane < a.chunks ? s[lane] : make_double2(-INFINITY, 0.);  // of the first 32 chunks, mostly all
      float m = (float)mine.x;
      for (int c = lane + 32; c < a.chunks; c += 32) m = fmaxf(m, (float)s[c].x);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      if (mine.y != 0.) sum = mine.y * exp(mine.x - m);
      for (int c = lane + 32; c < a.chunks; c += 32) sum += s[c].y == 0. ? 0. : s[c].y * exp(s[c].x - m);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      top = m;
    }
    if (lane == 0) sh_top[f] = top, sh_log[f] = log(sum), sh_score[f] = a.scores[row0 + f], sh_done[f] = done;
  }
  if (tid == 0) count = 0, bound = {-INFINITY, 0, MAX_BEAMS};
  __syncthreads();
  const Total none{-INFINITY, 0, MAX_BEAMS};
  // entry j of list l: l = a chunk of a row; a finished beam's only entry stands in its first list
  auto total = [&](int l, int j, unsigned long long key) {
    const int f = l / a.chunks;
    Total x = none;
    if (sh_done[f]) {
      if (l % a.chunks == 0 && j == 0) x = {sh_score[f], key_of(0.f, a.eos), f};
    } else {
      if (key) x = {sh_score[f] + (((double)key_logit(key) - sh_top[f]) - sh_log[f]), key, f};
    }
    return isfinite(x.t) ? x : none;
  };
  auto entry = [&](int l, int j) { return total(l, j, a.words[(row0 * a.chunks + l) * k + j]); };
  Total best = none;
#pragma unroll
  for (int i = 0; i < AHEAD; i++) {
    const int r = tid + i * TP;
    if (r >= runs || r / lists >= k) continue;
    const Total x = total(r % lists, r / lists, head[i]);
    if (ahead_of(x, best)) best = x;
  }
  for (int r = tid + AHEAD * TP; r < runs; r += TP)
    if (r / lists < k) {
      const Total x = entry(r % lists, r / lists);
      if (ahead_of(x, best)) best = x;
    }
  const Total mine = best;
  part_t[tid] = best.t, part_key[tid] = best.key, part_f[tid] = best.f;
  __syncthreads();
  {
    const int from = tid / per + tid % per * parts;  // of this thread's part, TP / per of them
    best = {part_t[from], part_key[from], part_f[from]};
    for (int d = 1; d < per; d <<= 1) {
      const Total x = shfl_xor(best, d);
      if (ahead_of(x, best)) best = x;
    }
    __syncthreads();
    if (tid % per == 0) part_t[tid / per] = best.t, part_key[tid / per] = best.key, part_f[tid / per] = best.f;
    __syncthreads();
    int ahead = 0;
    for (int i = tid % per; i < parts; i += per) ahead += ahead_of({part_t[i], part_key[i], part_f[i]}, best);
    for (int d = 1; d < per; d <<= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, d);
    if (tid % per == 0 && ahead == k - 1 && best.t > -INFINITY) bound = best;
  }
  __syncthreads();
  const Total lim = bound;  // none where fewer than k parts have a continuation
  auto reaches = [&](const Total& x) { return x.t > -INFINITY && !ahead_of(lim, x); };
  if (reaches(mine)) {
    auto gather = [&](int l, int j, Total x) {  // from the run's entry j, x, on
      while (reaches(x)) {
        const int n = atomicAdd(&count, 1);
        if (n < CAP) found_t[n] = x.t, found_key[n] = x.key, found_f[n] = x.f;
        j += deal;
        if (j >= k) break;
        x = entry(l, j);
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
      const int r = tid + i * TP;
      if (r < runs && r / lists < k) gather(r % lists, r / lists, total(r % lists, r / lists, head[i]));
    }
    for (int r = tid + AHEAD * TP; r < runs; r += TP)
      if (r / lists < k) gather(r % lists, r / lists, entry(r % lists, r / lists));
  }
  __syncthreads();
  const int n = count;
  const long long o = (long long)blockIdx.x * k;
  auto put = [&](int j, const Total& x) {
    const int f = x.f, v = (int)~(uint32_t)x.key;
    a.out_scores[o + j] = (float)x.t;
    a.out_parents[o + j] = (int)row0 + f;
    a.out_tokens[o + j] = v;
    a.out_done[o + j] = v == a.eos || sh_done[f];
  };
  auto put_none = [&](int j) {
    a.out_scores[o + j] = -INFINITY;
    a.out_parents[o + j] = (int)row0 + j % F;
    a.out_tokens[o + j] = -1;
    a.out_done[o + j] = 1;
  };
  if (n <= CAP) {
    for (int i = tid; i < n; i += TP) {
      const Total x{found_t[i], found_key[i], found_f[i]};
      int ahead = 0;
      for (int j = 0; j < n; j++) {
        const double y = found_t[j];
        if (y > x.t) ahead++;
        else if (y == x.t) ahead += ahead_of({y, found_key[j], found_f[j]}, x);
      }
      if (ahead < k) put(ahead, x);
    }
    for (int j = n + tid; j < k; j += TP) put_none(j);
    return;
  }
  // far more than k reach the bound (words that stand together in a few of many lists): one by one, the best behind the last
  Total last{INFINITY, 0, -1};
  for (int j = 0; j < k; j++) {
    best = none;
    for (int r = tid; r < runs; r += TP)
      for (int i = r / lists; i < k; i += deal) {
        const Total x = entry(r % lists, i);
        if (!ahead_of(x, best)) break;
        if (ahead_of(last, x)) {
          best = x;
          break;
        }
      }
    for (int d = 1; d < 32; d <<= 1) {
      const Total x = shfl_xor(best, d);
      if (ahead_of(x, best)) best = x;
    }
    if (lane == 0) part_t[warp] = best.t, part_key[warp] = best.key, part_f[warp] = best.f;
    __syncthreads();
    for (int w = 0; w < TP / 32; w++) {
      const Total x{part_t[w], part_key[w], part_f[w]};
      if (ahead_of(x, best)) best = x;
    }
    __syncthreads();
    last = best;  // n > CAP >= k: there is one
    if (tid == 0) put(j, best);
  }
}

struct Plan {
  int chunks;  // of a row
  long long words_off, bytes;
};
static Plan make_plan(int S, int F, int V, int k) {
  Plan p;
  const long long rows = (long long)S * F;
  p.chunks = (int)(((long long)V + T * E - 1) / (T * E));
  p.words_off = (rows * p.chunks * 16 + 255) / 256 * 256;
  p.bytes = p.words_off + rows * p.chunks * k * 8;
  return p;
}

}  // namespace beam
}  // namespace vt

extern "C" {

long long vt_beam_select_ws_bytes(int S, int F, int V, int k) {
  using namespace vt;
  if (S <= 0 || F <= 0 || F > beam::MAX_BEAMS || V <= 0 || k <= 0 || k > beam::MAX_K) return 0;
  return beam::make_plan(S, F, V, k).bytes;
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
  const beam::Plan p = beam::make_plan(S, F, V, k);
  const long long rows = (long long)S * F, n = (long long)S * k, es = f32 ? 4 : 2;
  if (rows > 0xffffffLL || (long long)F * V > 0x7fff0000LL || rows * p.chunks > 0x7fffffffLL)
    return set_error(E_SHAPE, "%s: S=%d or F * V = %lld too large", what, S, (long long)F * V);
  const struct { const void* p; long long n; } in[] = {{logits, ((rows - 1) * ld + V) * es}, {scores, rows * 4}, {done, done ? rows : 0}, {ws, need}},
      outs[] = {{out_scores, n * 4}, {out_parents, n * 4}, {out_tokens, n * 4}, {out_done, n}};
  for (const auto& x : in)
    for (const auto& y : outs)
      if (x.n && kv8::overlap(x.p, x.n, y.p, y.n)) return set_error(E_SHAPE, "%s: an output overlaps an input", what);
  beam::Args a{logits, ld, scores, done, F, V, k, eos, p.chunks, out_scores, out_parents, out_tokens, out_done, (double2*)ws,
               (unsigned long long*)((char*)ws + p.words_off)};
  // rows that do not all begin on 16 bytes are read a word at a time: the words of a chunk must not depend on where its row begins
  const bool wide = aligned16(logits) && (rows == 1 || ld * es % 16 == 0);
  const unsigned ctas = (unsigned)(rows * p.chunks);
  if (f32) launch_k(wide ? beam::beam_words_kernel<float, 4> : beam::beam_words_kernel<float, 1>, ctas, beam::T, 0, st, a);
  else launch_k(wide ? beam::beam_words_kernel<uint16_t, 8> : beam::beam_words_kernel<uint16_t, 1>, ctas, beam::T, 0, st, a);
  launch_k(beam::beam_pick_kernel, S, beam::TP, 0, st, a);
  return check_launch(what);
}

}  // extern "C"
