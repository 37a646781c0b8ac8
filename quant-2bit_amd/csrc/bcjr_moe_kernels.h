// Host-side view of the mixture-of-experts and distillation kernels: parameter
// blocks and launches.  The C ABI (bcjr_capi_moe.hip) validates before it
// launches.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace bcjr {

// Tokens that one workgroup routes whole; more take two launches.
constexpr int64_t kRouteOneBlock = 256;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxPicks = 64;

// 64-token words of a routing block: one (64 tokens) up to 16,384 tokens, so
// that the chip is full, then as many as keep 256 blocks, at most 16.
inline int route_words(int64_t T) {
  const int64_t w = (T + 64 * 256 - 1) / (64 * 256);
  return (int)(w < 1 ? 1 : w > 16 ? 16 : w);
}
inline int64_t route_blocks(int64_t T) {
  const int64_t per = 64 * (int64_t)route_words(T);
  return (T + per - 1) / per;
}

struct RouteParams {
  const void* logits;    // (T, E), row stride ld
  const uint8_t* valid;  // (T) or null
  float* weights;        // (T, k)
  int32_t* experts;      // (T, k)
  int32_t* offsets;      // (E + 1)
  int32_t* rows;         // (T * k)
  int32_t* slots;        // (T, k)
  int32_t* counts;       // (blocks + 1, E): workspace of more than one block
  int64_t T, ld;
  int E, k, renormalize, words;
};

struct RouteBwdParams {
  const void* logits;
  const uint8_t* valid;
  const float* weights;
  const int32_t* experts;
  const float* g_weights;  // (T, k)
  void* g_logits;          // (T, E)
  int64_t T, ld;
  int E, k, renormalize;
};

struct CombineParams {
  const void* y;         // (M, N), row stride ldy
  const float* weights;  // (T, k), or null for ones
  const int32_t* slots;  // (T, k)
  void* out;             // (T, N)
  int64_t T, M, N, ldy;
  int k;
};

struct CombineBwdParams {
  const void* y;
  const float* weights;
  const int32_t* slots;
  const int32_t* rows;  // (M)
  const void* g_out;    // (T, N), row stride ldg
  void* g_y;            // (M, N)
  float* g_weights;     // (T, k)
  int64_t T, M, N, ldy, ldg;
  int k;
};

struct GroupedParams {
  const void* a;         // rows of the left operand (ragged), row stride lda
  const void* b;         // see launch_grouped
  const int32_t* rows;   // (M) row of a for each sorted place, or null
  const int32_t* offsets;  // (E + 1); the first is taken as 0
  void* out;
  int64_t lda, ldb, a_rows, b_rows;
  int64_t M, N, K;
  int E;
  // zeros follow the rows of a and b up to a multiple of 8 elements
  bool zero_padded;
  // b is float32 (E, N, K), rounded to a's type as it is read; b_copy (E, N, K), or
  // null, gets the rounded weights of the experts that have rows
  bool b_f32;
  void* b_copy;
  // set by the launch: dies across the rows of the weights' gradient, and whether it
  // is stored past the caches
  int split;
  bool past;
};

struct DistillParams {
  const void* logits;       // (T, V), row stride ld
  const float* values;      // (T, K)
  const int32_t* indices;   // (T, K)
  const float* teacher_lse; // (T) or null
  const float* g_rows;      // (T): gradient of each row's loss
  float* loss;              // (T)
  float4* stats;            // (T, 2): see bcjr_distill.hip
  void* grad;               // (T, V)
  int64_t T, ld;
  int V, K;
  double inv_tau;
  float scale_hi, scale_lo;  // log2(e) / tau in two parts, the second above 0
};

// Gradients of more bytes than the last-level cache holds are stored past the caches,
// which keep what is read instead; smaller ones are found there by their reader.
// (Microseconds, cached / past.  Distillation's loss and gradient and a copy of the
// gradient: 1,024 x 32,000 bfloat16, 66 MB, 55 / 59; 4,096 x 32,000, 262 MB, 238 / 241;
// 4,096 x 50,257, 412 MB, 360 / 357; without the copy 8,192 x 131,072, 2.1 GB, 976 / 911 (gradient alone 845 / 785).
// Weights' gradient of 64 experts, 2048 x 2048 float32, 1.07 GB, 8,192 rows: 272 / 236.)
constexpr int64_t kPastCaches = 300 << 20;

// Stores `text` for bcjr_last_error() and returns the status (bcjr_capi.hip).
int report_failure(int status, const char* text);

hipError_t launch_route(RouteParams P, int dtype, hipStream_t stream);
hipError_t launch_route_backward(const RouteBwdParams& P, int dtype, hipStream_t stream);
hipError_t launch_combine(const CombineParams& P, int dtype, hipStream_t stream);
hipError_t launch_combine_backward(const CombineBwdParams& P, int dtype, hipStream_t stream);
// out (M, N) = a (M, K) times b (E, N, K) transposed (b_is_nk) or b (E, K, N).
hipError_t launch_grouped(const GroupedParams& P, int dtype, bool b_is_nk, hipStream_t stream);
// Whether the kernel on float32 weights takes these operands (gathered_rows: the
// rows of a that places name, 0 if they are in order).
bool grouped_f32w_fits(const void* a, int64_t lda, int64_t gathered_rows, const void* b, int64_t ldb, int64_t K);
// out (E, N, K) = a^T b over each group's rows, a (M, N), b (M, K) (rows of b
// through P.rows); out in float32 or the operands' type.
hipError_t launch_grouped_wgrad(const GroupedParams& P, int dtype, bool out_f32, hipStream_t stream);

// Rows of n elements (float32 or of the 16-bit `dtype`) to rows of ldo (a
// multiple of 8) of `dtype`, zeros behind them; out 16-byte aligned.
hipError_t launch_pad_rows(const void* x, int dtype_in, int64_t ld, int64_t rows, int64_t n, int dtype, void* out,
                           int64_t ldo, hipStream_t stream);

enum { DISTILL_LOSS = 0, DISTILL_BACKWARD = 1, DISTILL_BOTH = 2 };
constexpr int kDistillMaxVocab = 1 << 20;
hipError_t launch_distill(const DistillParams& P, int dtype, int kind, hipStream_t stream);

}  // namespace bcjr
