// Attention over the 8-bit cache for sequences that share a prefix: S prefix caches, F = B / S sequences on each, every sequence
// with a cache of its own behind it.  A prefix is read once for the rows of all of its sequences; softmax over the two caches comes
// apart into parts with a maximum and a sum each, which are put together by weight:  out = sum w o / sum w,  w = l 2^(m - max m).
//
// Few rows on a prefix (F n G <= 32; 16 heads' dims of 128): one item per head with all keys in its list of tiles (kv8_split.cu).
// More: the rows of all sequences over the prefix on tcgen05 (kv8_tc.cu), each sequence's rows over its own slots by either, then
// attn_kv8_shared_join_kernel.
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {
namespace shared {

constexpr int MAXB = 2048;

struct JoinArgs {
  tc::Args p;     // the prefixes' call
  split::Args s;  // the sequences' own slots, by whichever of the two
  tc::Args t;
  bool own_tc, own_whole;
  int B, nt;
};

// Thread = 4 dims of a row of the output; 16 rows a CTA.  A part is a whole row (its kernel left it normalised) or one CTA's share.
template <int D>
__global__ void __launch_bounds__(128) attn_kv8_shared_join_kernel(const __grid_constant__ JoinArgs j) {
  __shared__ int tok[MAXB + 1], ppre[MAXB + 1], opre[MAXB + 1], scratch[4];
  constexpr int PER = 128 * 4 / D;
  const tc::Args& p = j.p;
  const int n = p.n, G = p.G, H = p.H, Hq = G * H, F = p.F;
  griddep_wait();
  griddep_launch();
  tc::token_list(p, tok, scratch);
  int prun = 0, orun = 0;
  if (p.items == 0) {
    prun = tc::tile_list<tc::SHARED>(p, ppre, scratch, tok);
    __syncthreads();
  }
  if (!j.own_whole) {
    if (j.own_tc) {
      orun = tc::tile_list(j.t, opre, scratch);
    } else {
      split::tile_list(j.s, split::keys_per_tile(D), 8 * j.nt, opre, scratch);
      orun = split::run_of(opre[j.B], j.s.ctas);
    }
  }
  const int d = threadIdx.x % (D / 4) * 4;
  const long long rows = (long long)j.B * n * Hq;
  for (int x = threadIdx.x / (D / 4); x < 16; x += PER) {
    const long long at = (long long)blockIdx.x * 16 + x;
    if (at >= rows) break;
    const int hq = (int)(at % Hq), i = (int)(at / Hq % n), b = (int)(at / Hq / n), s = b / F, h = hq / G;
    if (i >= tok[b + 1] - tok[b]) continue;
    // the row's parts: of the prefix, then of its own slots; [c0, c1] are the CTAs that share it, first the slot of c0's
    const int P = split::prefix_len(p.plens, s, p.C, false), rp = (tok[b] - tok[s * F] + i) * G + hq % G;
    const int pt = (P + tc::KEYS - 1) / tc::KEYS;
    int pc0 = 0, pc1 = pt ? 0 : -1, oc0 = 0, oc1 = 0;
    size_t pfirst = 0, ofirst = 0;
    if (pt && p.items == 0) {
      const int items = ((tok[(s + 1) * F] - tok[s * F]) * G + tc::ROWS - 1) / tc::ROWS;
      const int u0 = ppre[s] + (h * items + rp / tc::ROWS) * pt;
      pc0 = u0 / prun, pc1 = (u0 + pt - 1) / prun, pfirst = 2 * (size_t)pc0 + (u0 == pc0 * prun ? 0 : 1);
    }
    const Seq q = seq_of(p.lens, p.counts, b, n, p.Co, false);
    const int ro = i * G + hq % G;
    int group = 1 << 30;  // rows of an item of the own slots
    if (!j.own_whole) {
      int u0, tiles;
      if (j.own_tc) {
        group = tc::ROWS;
        u0 = opre[b] + (opre[b + 1] - opre[b]) / H * h;
        int qt = 0;
        for (; qt < ro / tc::ROWS; qt++) u0 += tc::item_tiles(j.t, q, qt);
        tiles = tc::item_tiles(j.t, q, qt);
      } else {
        group = 8 * j.nt;
        tiles = (q.len + q.cnt + split::keys_per_tile(D) - 1) / split::keys_per_tile(D);
        u0 = opre[b] + (h * split::row_groups(j.s, q, group) + ro / group) * tiles;
      }
      oc0 = u0 / orun, oc1 = (u0 + tiles - 1) / orun, ofirst = 2 * (size_t)oc0 + (u0 == oc0 * orun ? 0 : 1);
    }
    const float2* prow = p.row_ml + ((size_t)s * H + h) * p.rows + rp;
    const float2* orow = (j.own_tc ? j.t.row_ml : j.s.own_ml) + ((size_t)b * H + h) * (n * G) + ro;
    auto pslot = [&](int c) { return (c == pc0 ? pfirst : 2 * (size_t)c) * tc::ROWS + rp % tc::ROWS; };
    auto oslot = [&](int c) { return (c == oc0 ? ofirst : 2 * (size_t)c) * group + ro % group; };
    auto pml = [&](int c) {
      if (pc0 == pc1) return *prow;
      const float2 v = p.part_ml[pslot(c)];
      return make_float2(v.x, v.y * (1.f / tc::L_SCALE));
    };
    auto oml = [&](int c) {
      if (oc0 == oc1) return *orow;
      if (!j.own_tc) return j.s.part_ml[oslot(c)];
      const float2 v = j.t.part_ml[oslot(c)];
      return make_float2(v.x, v.y * (1.f / tc::L_SCALE));
    };
    float mx = -INFINITY;
    for (int c = pc0; c <= pc1; c++) mx = fmaxf(mx, pml(c).x);
    for (int c = oc0; c <= oc1; c++) mx = fmaxf(mx, oml(c).x);
    float sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    // a part adds f (its O as it stands) and l 2^(m - mx) to the sum; the halves keep 2^(m - mx) l from vanishing where l is large
    auto add = [&](const float2& ml, const float4& o, bool normal, float unit) {
      const float half = ml.x == -INFINITY ? 0.f : ex2_approx(0.5f * (ml.x - mx)), w = ml.y * half * half, f = normal ? w : half * half * unit;
      sum += w, v.x += o.x * f, v.y += o.y * f, v.z += o.z * f, v.w += o.w * f;
    };
    if (pc0 == pc1) add(*prow, *reinterpret_cast<const float4*>(p.row_o + (((size_t)s * H + h) * p.rows + rp) * D + d), true, 0.f);
    else
#pragma unroll 2
      for (int c = pc0; c <= pc1; c++) add(pml(c), *reinterpret_cast<const float4*>(p.part_o + pslot(c) * D + d), false, 1.f);
    if (oc0 == oc1)
      add(*orow, *reinterpret_cast<const float4*>((j.own_tc ? j.t.row_o : j.s.own_o) + (((size_t)b * H + h) * (n * G) + ro) * D + d), true, 0.f);
    else
#pragma unroll 2
      for (int c = oc0; c <= oc1; c++)
        add(oml(c), *reinterpret_cast<const float4*>((j.own_tc ? j.t.part_o : j.s.part_o) + oslot(c) * D + d), false, j.own_tc ? 1.f : split::P_SCALE);
    const float inv = 1.f / sum;
    *reinterpret_cast<uint2*>(p.out + b * p.so_b + i * p.so_t + hq * p.so_h + d) = make_uint2(pack_bf2(v.x * inv, v.y * inv), pack_bf2(v.z * inv, v.w * inv));
  }
}

// Fixed on the host from sizes alone.
struct Plan {
  bool few;           // one item per head with all rows and keys
  bool own_tc;
  split::Plan s;      // of few, or of the sequences' own slots
  tc::Plan p, t;
  long long p_row, p_ml, o_off, o_row, o_ml, bytes;  // workspace: the prefixes' call and rows, the own slots' call and rows
};
// With F n G rows up to which one kernel takes all; a CTA of eight warps takes a whole item where it has at most so many tiles (MEASURED)
constexpr int FEW_TILES = 32;
static int few_rows(int D) { return D == 64 ? split::FEW_ROWS : 16; }

static Plan make_plan(int S, int B, int n, int Hq, int H, int D, int Cp, int C, int sms) {
  Plan x{};
  const int F = B / S, G = Hq / H;
  const long long all = (long long)F * n * G;
  auto up = [](long long v) { return (v + 255) / 256 * 256; };
  x.few = all <= few_rows(D);
  if (x.few) {
    const int kt = split::keys_per_tile(D);
    x.s = split::make_plan(S, F * n, Hq, H, D, Cp, false, sms, Cp / kt + (long long)F * (C / kt), FEW_TILES);
    x.bytes = x.s.full_off;
    return x;
  }
  x.own_tc = n * G > split::FEW_ROWS;
  x.p = tc::make_plan(S, F * n, Hq, H, D, Cp, false, sms);
  x.p_row = up(x.p.lse_off), x.p_ml = x.p_row + up((long long)B * n * Hq * D * 4), x.o_off = x.p_ml + up((long long)B * n * Hq * 8);
  if (x.own_tc) x.t = tc::make_plan(B, n, Hq, H, D, C, false, sms), x.o_row = x.o_off + up(x.t.lse_off);
  else x.s = split::make_plan(B, n, Hq, H, D, C, false, sms), x.o_row = x.o_off + x.s.full_off;
  x.o_ml = x.o_row + up((long long)B * n * Hq * D * 4), x.bytes = x.o_ml + up((long long)B * n * Hq * 8);
  return x;
}

}  // namespace shared
}  // namespace kv8
}  // namespace vt

extern "C" {

long long vt_attn_kv8_shared_ws_bytes(int S, int B, int n, int Hq, int H, int D, int Cp, int C) {
  using namespace vt::kv8;
  if (S <= 0 || B <= 0 || B % S || n <= 0 || Hq <= 0 || H <= 0 || Hq % H || Cp <= 0 || C <= 0 || (D != 64 && D != 128)) return 0;
  // what n tokens need, and any fewer that may follow with the same workspace: at the largest n of each plan
  const int sms = vt::sm_count(), G = Hq / H, F = B / S;
  long long most = shared::make_plan(S, B, n, Hq, H, D, Cp, C, sms).bytes;
  for (const int rows : {shared::few_rows(D) / F, split::FEW_ROWS}) {
    const int m = rows / G;
    if (m <= 0 || m >= n) continue;
    const long long x = shared::make_plan(S, B, m, Hq, H, D, Cp, C, sms).bytes;
    if (x > most) most = x;
  }
  return most;
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
  const long long most = 0x20000000LL;  // tiles of a list, four rows
  if ((long long)B * n * Hq > most / 4 || (long long)S * H * (Cp / kv8::BLK) * ((long long)F * n * G / 32 + 1) > most ||
      (long long)B * H * (C / kv8::BLK) * ((long long)n * G / 8 + 1) > most)
    return set_error(E_SHAPE, "%s: B * Hq * n or B * H * C too large", what);
  const kv8::shared::Plan x = kv8::shared::make_plan(S, B, n, Hq, H, D, Cp, C, sms);
  char* w8 = static_cast<char*>(ws);
  const float c = scale * kv8::LOG2E;
  kv8::split::Args sa{q, sq_b, sq_t, sq_h, kc, vc, ks, vs, lens, counts, x.few ? S : B, n, G, H, C, 1, x.few ? F * n * G : n * G, x.few ? 1 : x.s.rg, x.s.ctas, c,
                      out, so_b, so_t, so_h, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, pk, pv, pks, pvs, plens, Cp, F, nullptr, nullptr};
  if (x.few) {
    sa.part_o = (float*)(w8 + x.s.o_off), sa.part_ml = (float2*)(w8 + x.s.ml_off);
    return kv8::split::launch_any<kv8::split::SHARED>(st, sa, D, x.s.nt, x.s.whole, what);
  }
  kv8::tc::Args pa{q, sq_b, sq_t, sq_h, pk, pv, pks, pvs, lens, counts, S, n, G, H, Cp, 0, F * n * G, x.p.ctas,
                   x.p.whole ? (int)(((long long)F * n * G + kv8::tc::ROWS - 1) / kv8::tc::ROWS) : 0, c, out, so_b, so_t, so_h,
                   (float*)w8, (float2*)(w8 + x.p.ml_off), nullptr, nullptr, nullptr, plens, F, C, (float*)(w8 + x.p_row), (float2*)(w8 + x.p_ml)};
  kv8::tc::Args ta{q, sq_b, sq_t, sq_h, kc, vc, ks, vs, lens, counts, B, n, G, H, C, 1, n * G, x.t.ctas,
                   x.own_tc && x.t.whole ? (n * G + kv8::tc::ROWS - 1) / kv8::tc::ROWS : 0, c, out, so_b, so_t, so_h,
                   (float*)(w8 + x.o_off), (float2*)(w8 + x.o_off + x.t.ml_off), nullptr, nullptr, nullptr, nullptr, 1, C,
                   (float*)(w8 + x.o_row), (float2*)(w8 + x.o_ml)};
  sa.part_o = (float*)(w8 + x.o_off + x.s.o_off), sa.part_ml = (float2*)(w8 + x.o_off + x.s.ml_off);
  sa.own_o = (float*)(w8 + x.o_row), sa.own_ml = (float2*)(w8 + x.o_ml);
  rc = D == 64 ? kv8::tc::launch<64, kv8::tc::SHARED>(st, pa, what) : kv8::tc::launch<128, kv8::tc::SHARED>(st, pa, what);
  if (rc) return rc;
  if (!x.own_tc) rc = kv8::split::launch_any<kv8::split::OWN>(st, sa, D, x.s.nt, x.s.whole, what);
  else rc = D == 64 ? kv8::tc::launch<64, kv8::tc::OWN>(st, ta, what) : kv8::tc::launch<128, kv8::tc::OWN>(st, ta, what);
  if (rc) return rc;
  kv8::shared::JoinArgs j{pa, sa, ta, x.own_tc, x.own_tc ? x.t.whole : x.s.whole, B, x.s.nt};
  const unsigned ctas = (unsigned)(((long long)B * n * Hq + 15) / 16);
  if (D == 64) launch_k(kv8::shared::attn_kv8_shared_join_kernel<64>, ctas, 128, 0, st, j);
  else launch_k(kv8::shared::attn_kv8_shared_join_kernel<128>, ctas, 128, 0, st, j);
  return check_launch(what);
}

}  // extern "C"
