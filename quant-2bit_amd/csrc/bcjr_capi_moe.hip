// C ABI of the mixture-of-experts and distillation operators
// (include/bcjr_hip.h): validation and launches on the caller's stream.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/bcjr_hip.h"
#include "bcjr_moe_kernels.h"

namespace {

int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return bcjr::report_failure(status, buf);
}

int launched(hipError_t e, const char* what) {
  return e == hipSuccess ? BCJR_OK : fail(BCJR_EHIP, "%s: %s", what, hipGetErrorString(e));
}

typedef long long ll;

int check_dtype(int dtype) {
  return dtype == BCJR_F32 || dtype == BCJR_BF16 || dtype == BCJR_F16
             ? BCJR_OK
             : fail(BCJR_EINVAL, "unknown element type %d", dtype);
}

int check_routing(int dtype, int64_t ld, int64_t T, int64_t E, int k) {
  if (int rc = check_dtype(dtype)) return rc;
  if (E < 1 || E > bcjr::kRouteMaxExperts)
    return fail(E < 1 ? BCJR_EINVAL : BCJR_EUNSUPPORTED, "E=%lld experts outside [1, %d]", (ll)E,
                bcjr::kRouteMaxExperts);
  if (k < 1 || k > E || k > bcjr::kRouteMaxPicks)
    return fail(BCJR_EINVAL, "k=%d outside [1, min(E=%lld, %d)]", k, (ll)E, bcjr::kRouteMaxPicks);
  if (T < 0 || T * k > INT32_MAX) return fail(BCJR_EINVAL, "T=%lld tokens with k=%d: T*k must be in [0, 2^31)", (ll)T, k);
  if (T > 1 && ld < E) return fail(BCJR_EINVAL, "row stride %lld is below E=%lld", (ll)ld, (ll)E);
  return BCJR_OK;
}

size_t route_ws(int64_t T, int64_t E) {
  return T <= bcjr::kRouteOneBlock ? 0 : (size_t)(bcjr::route_blocks(T) + 1) * (size_t)E * sizeof(int32_t);
}

constexpr int64_t kMaxDim = 1 << 20;

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

int check_grouped(int dtype, int64_t E, int64_t M, int64_t N, int64_t K) {
  if (int rc = check_dtype(dtype)) return rc;
  if (dtype == BCJR_F32) return fail(BCJR_EUNSUPPORTED, "grouped products are built for bfloat16 and float16 operands");
  if (E < 1 || E > bcjr::kRouteMaxExperts)
    return fail(E < 1 ? BCJR_EINVAL : BCJR_EUNSUPPORTED, "E=%lld experts outside [1, %d]", (ll)E,
                bcjr::kRouteMaxExperts);
  if (M < 0 || M > INT32_MAX) return fail(BCJR_EINVAL, "M=%lld rows outside [0, 2^31)", (ll)M);
  if (N < 1 || N > kMaxDim || K < 1 || K > kMaxDim)
    return fail(BCJR_EINVAL, "N=%lld, K=%lld must be in [1, %lld]", (ll)N, (ll)K, (ll)kMaxDim);
  // A launch has fewer than 2^32 threads a dimension: 512 a tile of 256 x 256, a few
  // more for the eight dies' equal shares, 256 a row tile of 64 in the slow kernel.
  const int64_t most = (1 << 23) - 16, n = N / 256 + 1, k = K / 256 + 1;
  if ((M / 256 + E + 1) * (n > k ? n : k) >= most || E * (n + 7) * (k + 7) >= most || M >= (1 << 30) - (1 << 17))
    return fail(BCJR_EUNSUPPORTED, "M=%lld, N=%lld, K=%lld, E=%lld: more tiles than a launch holds", (ll)M, (ll)N, (ll)K,
                (ll)E);
  return BCJR_OK;
}

int check_combine(int dtype, int64_t ldy, int64_t T, int k, int64_t M, int64_t N) {
  if (int rc = check_dtype(dtype)) return rc;
  if (k < 1) return fail(BCJR_EINVAL, "k=%d must be >= 1", k);
  if (T < 0 || M < 0 || M > INT32_MAX) return fail(BCJR_EINVAL, "T=%lld tokens, M=%lld rows outside [0, 2^31)", (ll)T, (ll)M);
  if (T >= 1 << 24) return fail(BCJR_EUNSUPPORTED, "T=%lld tokens: combine is built for fewer than 2^24", (ll)T);
  if (N < 1 || N > kMaxDim) return fail(BCJR_EINVAL, "N=%lld must be in [1, %lld]", (ll)N, (ll)kMaxDim);
  if (M > 1 && ldy < N) return fail(BCJR_EINVAL, "row stride %lld is below N=%lld", (ll)ldy, (ll)N);
  return BCJR_OK;
}

int check_distill(int dtype, int64_t ld, float temperature, int64_t T, int64_t V, int64_t K) {
  if (int rc = check_dtype(dtype)) return rc;
  if (!(temperature > 0.f) || !std::isfinite(temperature) || !std::isfinite(1.f / temperature))
    return fail(BCJR_EINVAL, "temperature %g must be finite and > 0", (double)temperature);
  if (T < 0) return fail(BCJR_EINVAL, "T=%lld rows must be >= 0", (ll)T);
  if (T >= 1 << 22) return fail(BCJR_EUNSUPPORTED, "T=%lld rows: the loss is built for fewer than 2^22", (ll)T);
  if (V < 1 || V > bcjr::kDistillMaxVocab)
    return fail(V < 1 ? BCJR_EINVAL : BCJR_EUNSUPPORTED, "V=%lld outside [1, %d]", (ll)V, bcjr::kDistillMaxVocab);
  if (K < 0 || K > V) return fail(BCJR_EINVAL, "K=%lld teacher entries outside [0, V=%lld]", (ll)K, (ll)V);
  if (T > 1 && ld < V) return fail(BCJR_EINVAL, "row stride %lld is below V=%lld", (ll)ld, (ll)V);
  return BCJR_OK;
}

bcjr::DistillParams distill_params(const void* logits, int64_t ld, const float* values, const int32_t* indices,
                                   const float* teacher_lse, float temperature, int64_t T, int64_t V, int64_t K) {
  bcjr::DistillParams P = {};
  P.logits = logits;
  P.values = values;
  P.indices = indices;
  P.teacher_lse = teacher_lse;
  P.T = T;
  P.ld = T > 1 ? ld : V;
  P.V = (int)V;
  P.K = (int)K;
  P.inv_tau = 1. / (double)temperature;
  const double scale = 1.4426950408889634 * P.inv_tau;
  P.scale_hi = (float)scale;
  if ((double)P.scale_hi >= scale) P.scale_hi = std::nextafterf(P.scale_hi, 0.f);
  P.scale_lo = (float)(scale - (double)P.scale_hi);
  return P;
}

}  // namespace

extern "C" {

int bcjr_moe_route_workspace(int64_t T, int64_t E, size_t* bytes) {
  if (!bytes) return fail(BCJR_EINVAL, "bytes must be non-NULL");
  if (int rc = check_routing(BCJR_F32, E, T, E, 1)) return rc;
  *bytes = route_ws(T, E);
  return BCJR_OK;
}

int bcjr_moe_route(const void* logits, int dtype, int64_t ld, const uint8_t* valid, int64_t T, int64_t E, int k,
                   int renormalize, float* weights, int32_t* experts, int32_t* offsets, int32_t* rows, int32_t* slots,
                   void* ws, size_t ws_bytes, hipStream_t stream) {
  if (int rc = check_routing(dtype, ld, T, E, k)) return rc;
  if (!offsets) return fail(BCJR_EINVAL, "offsets must be non-NULL");
  if (T > 0 && (!logits || !weights || !experts || !rows || !slots))
    return fail(BCJR_EINVAL, "logits, weights, experts, rows and slots must be non-NULL");
  const size_t need = route_ws(T, E);
  if (need && !ws) return fail(BCJR_EINVAL, "ws must be non-NULL");
  if (ws_bytes < need) return fail(BCJR_EWORKSPACE, "ws_bytes=%zu: routing needs %zu bytes", ws_bytes, need);
  bcjr::RouteParams P = {logits, valid,        weights, experts, offsets, rows,
                         slots,  (int32_t*)ws, T,       ld,      (int)E,  k, renormalize ? 1 : 0, 0};
  return launched(bcjr::launch_route(P, dtype, stream), "bcjr_moe_route launch");
}

int bcjr_moe_route_backward(const void* logits, int dtype, int64_t ld, const uint8_t* valid, int64_t T, int64_t E,
                            int k, int renormalize, const float* weights, const int32_t* experts,
                            const float* g_weights, void* g_logits, hipStream_t stream) {
  if (int rc = check_routing(dtype, ld, T, E, k)) return rc;
  if (T == 0) return BCJR_OK;
  if (!logits || !weights || !experts || !g_weights || !g_logits)
    return fail(BCJR_EINVAL, "logits, weights, experts, g_weights and g_logits must be non-NULL");
  if (T >= 1 << 26)
    return fail(BCJR_EUNSUPPORTED, "T=%lld tokens: the routing's gradient is built for fewer than 2^26", (ll)T);
  const bcjr::RouteBwdParams P = {logits, valid, weights, experts, g_weights, g_logits,
                                  T,      ld,    (int)E,  k,       renormalize ? 1 : 0};
  return launched(bcjr::launch_route_backward(P, dtype, stream), "bcjr_moe_route_backward launch");
}

int bcjr_grouped_matmul(const void* a, int dtype, int64_t lda, int64_t a_rows, const int32_t* rows, const void* b,
                        int64_t ldb, int b_is_nk, const int32_t* offsets, int64_t E, int64_t M, int64_t N, int64_t K,
                        int zero_padded, void* out, hipStream_t stream) {
  if (int rc = check_grouped(dtype, E, M, N, K)) return rc;
  if (a_rows < 0 || (!rows && a_rows < M))
    return fail(BCJR_EINVAL, "a has %lld rows for M=%lld", (ll)a_rows, (ll)M);
  const int64_t across = b_is_nk ? K : N;
  if (a_rows > 1 && lda < K) return fail(BCJR_EINVAL, "row stride %lld is below K=%lld", (ll)lda, (ll)K);
  if (ldb < across) return fail(BCJR_EINVAL, "row stride %lld of b is below %lld", (ll)ldb, (ll)across);
  if (zero_padded && (ldb < up8(across) || (a_rows > 1 && lda < up8(K)) || ldb % 8 || lda % 8))
    return fail(BCJR_EINVAL, "zero-padded rows: strides %lld, %lld do not hold K=%lld, N=%lld in eights", (ll)lda,
                (ll)ldb, (ll)K, (ll)N);
  if (M == 0) return BCJR_OK;
  if ((!a && a_rows) || !b || !offsets || !out) return fail(BCJR_EINVAL, "a, b, offsets and out must be non-NULL");
  bcjr::GroupedParams P = {};
  P.a = a, P.b = b, P.rows = rows, P.offsets = offsets, P.out = out;
  P.lda = lda, P.ldb = ldb, P.a_rows = a_rows, P.M = M, P.N = N, P.K = K, P.E = (int)E;
  P.zero_padded = zero_padded != 0;
  return launched(bcjr::launch_grouped(P, dtype, b_is_nk != 0, stream), "bcjr_grouped_matmul launch");
}

int bcjr_grouped_wgrad(const void* a, int dtype, int64_t lda, const void* b, int64_t ldb, int64_t b_rows,
                       const int32_t* rows, const int32_t* offsets, int64_t E, int64_t M, int64_t N, int64_t K,
                       int zero_padded, int out_f32, void* out, hipStream_t stream) {
  if (int rc = check_grouped(dtype, E, M, N, K)) return rc;
  if (b_rows < 0 || (!rows && b_rows < M)) return fail(BCJR_EINVAL, "b has %lld rows for M=%lld", (ll)b_rows, (ll)M);
  if (M > 1 && lda < N) return fail(BCJR_EINVAL, "row stride %lld is below N=%lld", (ll)lda, (ll)N);
  if (b_rows > 1 && ldb < K) return fail(BCJR_EINVAL, "row stride %lld is below K=%lld", (ll)ldb, (ll)K);
  if (zero_padded && (lda < up8(N) || ldb < up8(K) || lda % 8 || ldb % 8))
    return fail(BCJR_EINVAL, "zero-padded rows: strides %lld, %lld do not hold N=%lld, K=%lld in eights", (ll)lda,
                (ll)ldb, (ll)N, (ll)K);
  if (!offsets || !out || (M && (!a || (!b && b_rows))))
    return fail(BCJR_EINVAL, "a, b, offsets and out must be non-NULL");
  bcjr::GroupedParams P = {};
  P.a = a, P.b = b, P.rows = rows, P.offsets = offsets, P.out = out;
  P.lda = lda, P.ldb = ldb, P.a_rows = M, P.b_rows = b_rows, P.M = M, P.N = N, P.K = K, P.E = (int)E;
  P.zero_padded = zero_padded != 0;
  return launched(bcjr::launch_grouped_wgrad(P, dtype, out_f32 != 0, stream), "bcjr_grouped_wgrad launch");
}

int bcjr_grouped_matmul_f32w(const void* a, int dtype, int64_t lda, int64_t a_rows, const int32_t* rows,
                             const float* b, int64_t ldb, const int32_t* offsets, int64_t E, int64_t M, int64_t N,
                             int64_t K, void* out, void* b_copy, hipStream_t stream) {
  if (int rc = check_grouped(dtype, E, M, N, K)) return rc;
  if (a_rows < 0 || (!rows && a_rows < M))
    return fail(BCJR_EINVAL, "a has %lld rows for M=%lld", (ll)a_rows, (ll)M);
  if (a_rows > 1 && lda < K) return fail(BCJR_EINVAL, "row stride %lld is below K=%lld", (ll)lda, (ll)K);
  if (ldb < K) return fail(BCJR_EINVAL, "row stride %lld of b is below %lld", (ll)ldb, (ll)K);
  if (!bcjr::grouped_f32w_fits(a, lda, rows ? a_rows : 0, b, ldb, K) || (reinterpret_cast<uintptr_t>(b_copy) & 7))
    return fail(BCJR_EUNSUPPORTED, "float32 weights need rows in 16-byte chunks: K=%lld, strides %lld, %lld", (ll)K,
                (ll)lda, (ll)ldb);
  if (M == 0) return BCJR_OK;
  if ((!a && a_rows) || !b || !offsets || !out) return fail(BCJR_EINVAL, "a, b, offsets and out must be non-NULL");
  bcjr::GroupedParams P = {};
  P.a = a, P.b = b, P.rows = rows, P.offsets = offsets, P.out = out;
  P.lda = lda, P.ldb = ldb, P.a_rows = a_rows, P.M = M, P.N = N, P.K = K, P.E = (int)E;
  P.b_f32 = true, P.b_copy = b_copy;
  return launched(bcjr::launch_grouped(P, dtype, true, stream), "bcjr_grouped_matmul_f32w launch");
}

int bcjr_pad_rows(const void* x, int dtype_in, int64_t ld, int64_t rows, int64_t n, int dtype, void* out, int64_t ldo,
                  hipStream_t stream) {
  if (int rc = check_dtype(dtype_in)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (dtype == BCJR_F32 || (dtype_in != BCJR_F32 && dtype_in != dtype))
    return fail(BCJR_EUNSUPPORTED, "padded copies are built from float32 or the 16-bit type itself to that type");
  if (rows < 0 || n < 0) return fail(BCJR_EINVAL, "rows=%lld, n=%lld must be >= 0", (ll)rows, (ll)n);
  if (rows > 1 && ld < n) return fail(BCJR_EINVAL, "row stride %lld is below n=%lld", (ll)ld, (ll)n);
  if (ldo < n || ldo % 8) return fail(BCJR_EINVAL, "ldo=%lld must be a multiple of 8, at least n=%lld", (ll)ldo, (ll)n);
  if (rows == 0 || ldo == 0) return BCJR_OK;
  if ((!x && n) || !out) return fail(BCJR_EINVAL, "x and out must be non-NULL");
  if (reinterpret_cast<uintptr_t>(out) & 15) return fail(BCJR_EINVAL, "out must be 16-byte aligned");
  return launched(bcjr::launch_pad_rows(x, dtype_in, ld, rows, n, dtype, out, ldo, stream), "bcjr_pad_rows launch");
}

int bcjr_moe_combine(const void* y, int dtype, int64_t ldy, const float* weights, const int32_t* slots, int64_t T,
                     int k, int64_t M, int64_t N, void* out, hipStream_t stream) {
  if (int rc = check_combine(dtype, ldy, T, k, M, N)) return rc;
  if (T == 0) return BCJR_OK;
  if ((!y && M) || !slots || !out) return fail(BCJR_EINVAL, "y, slots and out must be non-NULL");
  const bcjr::CombineParams P = {y, weights, slots, out, T, M, N, ldy, k};
  return launched(bcjr::launch_combine(P, dtype, stream), "bcjr_moe_combine launch");
}

int bcjr_moe_combine_backward(const void* y, int dtype, int64_t ldy, const float* weights, const int32_t* slots,
                              const int32_t* rows, const void* g_out, int64_t ldg, int64_t T, int k, int64_t M,
                              int64_t N, void* g_y, float* g_weights, hipStream_t stream) {
  if (int rc = check_combine(dtype, ldy, T, k, M, N)) return rc;
  if (M != T * k) return fail(BCJR_EINVAL, "M=%lld rows for T*k=%lld pairs", (ll)M, (ll)(T * k));
  if (T > 1 && ldg < N) return fail(BCJR_EINVAL, "row stride %lld is below N=%lld", (ll)ldg, (ll)N);
  if (T == 0) return BCJR_OK;
  if (!y || !weights || !slots || !rows || !g_out || !g_y || !g_weights)
    return fail(BCJR_EINVAL, "y, weights, slots, rows, g_out, g_y and g_weights must be non-NULL");
  const bcjr::CombineBwdParams P = {y, weights, slots, rows, g_out, g_y, g_weights, T, M, N, ldy, ldg, k};
  return launched(bcjr::launch_combine_backward(P, dtype, stream), "bcjr_moe_combine_backward launch");
}

int bcjr_topk_distill(const void* logits, int dtype, int64_t ld, const float* values, const int32_t* indices,
                      const float* teacher_lse, float temperature, int64_t T, int64_t V, int64_t K, float* loss,
                      float* stats, hipStream_t stream) {
  if (int rc = check_distill(dtype, ld, temperature, T, V, K)) return rc;
  if (T == 0) return BCJR_OK;
  if (!logits || !loss || (K && (!values || !indices)))
    return fail(BCJR_EINVAL, "logits, values, indices and loss must be non-NULL");
  if (reinterpret_cast<uintptr_t>(stats) & 15) return fail(BCJR_EINVAL, "stats must be 16-byte aligned");
  bcjr::DistillParams P = distill_params(logits, ld, values, indices, teacher_lse, temperature, T, V, K);
  P.loss = loss;
  P.stats = (float4*)stats;
  return launched(bcjr::launch_distill(P, dtype, bcjr::DISTILL_LOSS, stream), "bcjr_topk_distill launch");
}

int bcjr_topk_distill_backward(const void* logits, int dtype, int64_t ld, const float* values,
                               const int32_t* indices, float temperature, int64_t T, int64_t V, int64_t K,
                               const float* stats, const float* g_loss, void* g_logits, hipStream_t stream) {
  if (int rc = check_distill(dtype, ld, temperature, T, V, K)) return rc;
  if (T == 0) return BCJR_OK;
  if (!logits || !stats || !g_loss || !g_logits || (K && (!values || !indices)))
    return fail(BCJR_EINVAL, "logits, values, indices, stats, g_loss and g_logits must be non-NULL");
  if (reinterpret_cast<uintptr_t>(stats) & 15) return fail(BCJR_EINVAL, "stats must be 16-byte aligned");
  bcjr::DistillParams P = distill_params(logits, ld, values, indices, nullptr, temperature, T, V, K);
  P.stats = (float4*)stats;
  P.g_rows = g_loss;
  P.grad = g_logits;
  return launched(bcjr::launch_distill(P, dtype, bcjr::DISTILL_BACKWARD, stream), "bcjr_topk_distill_backward launch");
}

int bcjr_topk_distill_both(const void* logits, int dtype, int64_t ld, const float* values, const int32_t* indices,
                           const float* teacher_lse, float temperature, int64_t T, int64_t V, int64_t K,
                           const float* g_loss, float* loss, void* g_logits, hipStream_t stream) {
  if (int rc = check_distill(dtype, ld, temperature, T, V, K)) return rc;
  if (T == 0) return BCJR_OK;
  if (!logits || !g_loss || !loss || !g_logits || (K && (!values || !indices)))
    return fail(BCJR_EINVAL, "logits, values, indices, g_loss, loss and g_logits must be non-NULL");
  bcjr::DistillParams P = distill_params(logits, ld, values, indices, teacher_lse, temperature, T, V, K);
  P.loss = loss;
  P.g_rows = g_loss;
  P.grad = g_logits;
  return launched(bcjr::launch_distill(P, dtype, bcjr::DISTILL_BOTH, stream), "bcjr_topk_distill_both launch");
}

}  // extern "C"
