// Attention over the 8-bit cache: the entry point, which chooses between few rows (kv8_split.cu) and many (kv8_tc.cu).
#include "vt_common.cuh"
#include "vt_host.h"

namespace vt {
namespace kv8 {

static bool few_rows(int n, int Hq, int H) { return (long long)n * (Hq / H) <= split::FEW_ROWS; }

}  // namespace kv8
}  // namespace vt

extern "C" {

long long vt_attn_kv8_ws_bytes(int B, int n, int Hq, int H, int D, int C, int weights) {
  if (B <= 0 || n <= 0 || Hq <= 0 || H <= 0 || Hq % H || C <= 0 || (D != 64 && D != 128)) return 0;
  // what n tokens need, and any fewer that may follow with the same workspace
  const int few = vt::kv8::split::FEW_ROWS / (Hq / H), nf = n < few ? n : few;
  const long long split = nf ? vt::kv8::split::make_plan(B, nf, Hq, H, D, C, weights != 0, vt::sm_count()).bytes : 0;
  const long long many = n > few ? vt::kv8::tc::make_plan(B, n, Hq, H, D, C, weights != 0, vt::sm_count()).bytes : 0;
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
  if (!(scale >= 0.f && scale < 0x1p100f)) return set_error(E_SHAPE, "vt_attn_kv8: scale %g is not 0 .. 2^100", scale);
  if (weights_in && !weights) return set_error(E_SHAPE, "vt_attn_kv8: weights_in without weights");
  const long long need = vt_attn_kv8_ws_bytes(B, n, Hq, H, D, C, weights != nullptr);
  if (need && (!ws || !aligned16(ws) || ws_bytes < need))
    return set_error(E_SHAPE, "vt_attn_kv8: workspace of %lld bytes, %lld needed (16-byte aligned)", ws ? ws_bytes : 0LL, need);
  const bool meet = kv8::rows_meet({q, sq_b, sq_t, (Hq - 1) * sq_h + D}, {out, so_b, so_t, (Hq - 1) * so_h + D}, B, n);
  if (kv8::few_rows(n, Hq, H)) {
    const kv8::split::Plan p = kv8::split::make_plan(B, n, Hq, H, D, C, weights != nullptr, sm_count());
    if (B > kv8::split::MAXB || (long long)B * H * p.rg * (C / kv8::split::keys_per_tile(D)) > 0x40000000LL)
      return set_error(E_SHAPE, "vt_attn_kv8: B=%d (at most %d) or B * H * C too large", B, kv8::split::MAXB);
    if (meet) return set_error(E_SHAPE, "vt_attn_kv8: out overlaps q");
    char* w8 = static_cast<char*>(ws);
    kv8::split::Args a{q, sq_b, sq_t, sq_h, kc, vc, ks, vs, lens, counts, B, n, Hq / H, H, C, causal, p.rows, p.rg, p.ctas,
                       scale * kv8::LOG2E, out, so_b, so_t, so_h, (float*)(w8 + p.o_off), (float2*)(w8 + p.ml_off),
                       (float2*)(w8 + p.full_off), weights ? (float*)(w8 + p.s_off) : nullptr, weights, weights_in};
    if (D == 64) return p.nt == 1 ? kv8::split::launch<64, 1>(st, a, p.whole) : p.nt == 2 ? kv8::split::launch<64, 2>(st, a, p.whole) : kv8::split::launch<64, 4>(st, a, p.whole);
    return p.nt == 1 ? kv8::split::launch<128, 1>(st, a, p.whole) : kv8::split::launch<128, 2>(st, a, p.whole);
  }
  const kv8::tc::Plan p = kv8::tc::make_plan(B, n, Hq, H, D, C, weights != nullptr, sm_count());
  const long long items = (p.rows + kv8::tc::ROWS - 1) / kv8::tc::ROWS;
  if (B > kv8::tc::MAXB || (long long)n * (Hq / H) > 0x3fffffffLL || B * items * H * (C / kv8::BLK) > 0x40000000LL)
    return set_error(E_SHAPE, "vt_attn_kv8: B=%d (at most %d) or B * H * n * C too large", B, kv8::tc::MAXB);
  if (meet) return set_error(E_SHAPE, "vt_attn_kv8: out overlaps q");
  char* w8 = static_cast<char*>(ws);
  kv8::tc::Args a{q, sq_b, sq_t, sq_h, kc, vc, ks, vs, lens, counts, B, n, Hq / H, H, C, causal, p.rows, p.ctas,
                  p.whole ? (int)items : 0, scale * kv8::LOG2E,
                  out, so_b, so_t, so_h, (float*)w8, (float2*)(w8 + p.ml_off), weights ? (float*)(w8 + p.lse_off) : nullptr,
                  weights, weights_in};
  return D == 64 ? kv8::tc::launch<64>(st, a) : kv8::tc::launch<128>(st, a);
}

}  // extern "C"
