// Products with the weights of many experts over ragged groups of rows.
//
//   forward   y[p] = w[e] x[row(p)]          w (E, N, K), group e = places
//   rows'     dx[p] = w[e]^T dy[p]           [offsets[e], offsets[e+1])
//   weights'  dw[e] = sum_p dy[p] x[row(p)]^T
//
// The group sizes are known to the device only.  The host launches as many
// row tiles as any division of M rows into E groups needs (M / BM + E + 1, and
// no more than M); every workgroup finds its expert and rows from the offsets,
// which it clamps to [0, M], and those behind the last tile leave.  The rows
// behind the last group are a group of their own, written as zeros.
#include "bcjr_moe_device.h"
#include "bcjr_moe_kernels.h"

namespace bcjr {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

// c (16 x 16, float32) += a (16 x 32) b (32 x 16).  Lane l holds a[l & 15] and
// b[.][l & 15] at k = 8 (l >> 4) .. + 7, and c[4 (l >> 4) + r][l & 15] in c[r].
template <class E>
__device__ __forceinline__ f32x4 mfma16(u16x8 a, u16x8 b, f32x4 c) {
  if constexpr (__is_same(E, BF16))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

struct Tile {
  int e;           // expert; E for the rows behind the last group, -1 for none
  int64_t r0, r1;  // its rows
};

// The tile-th row tile of height BM over the groups, E + 1 of them.  Called by
// whole waves; every wave finds the same.
template <int BM>
__device__ __forceinline__ Tile find_tile(const int32_t* offsets, int E, int64_t M, int64_t tile) {
  const int lane = threadIdx.x & 63;
  int64_t done = 0;
  for (int i = 0; i <= E; i += 64) {
    const int e = i + lane;
    int64_t a = 0, b = 0;
    if (e <= E) {
      a = e == 0 ? 0 : min((int64_t)max(offsets[e], 0), M);
      b = e == E ? M : min((int64_t)max(offsets[e + 1], 0), M);
      b = max(a, b);
    }
    const int n = (int)((b - a + BM - 1) / BM);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(upto, o);
      if (lane >= o) upto += y;
    }
    const int64_t first = done + upto - n;
    const unsigned long long here = __ballot(tile >= first && tile < first + n);
    if (here) {
      const int src = __ffsll(here) - 1;
      const int ea = __shfl((int)a, src), eb = __shfl((int)b, src);
      const int64_t f = done + __shfl(upto - n, src);
      const int64_t r0 = ea + (tile - f) * BM;
      return {i + src, r0, min(r0 + BM, (int64_t)eb)};
    }
    done += __shfl(upto, 63);
  }
  return {-1, 0, 0};
}

// Most row tiles of height BM that M rows in E groups and a rest can have.
int64_t max_tiles(int64_t M, int64_t E, int BM) {
  const int64_t t = M / BM + E + 1;
  return t < M ? t : M;
}

// ------------------------------------------------------- any size, any stride
//
// 64 x 64 tiles of the output, 32 of the reduction at a time, element loads
// with bounds into LDS: for row lengths and strides that 16-byte loads cannot
// take.  Four waves, 32 x 32 outputs each.
constexpr int kT = 64, kTk = 32, kPad = kTk + 8;

template <class E>
__device__ __forceinline__ void any_step(const uint16_t (*As)[kPad], const uint16_t (*Bs)[kPad], f32x4 (*acc)[2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  u16x8 a[2], b[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    a[i] = *(const u16x8*)&As[wm + 16 * i + (lane & 15)][8 * (lane >> 4)];
    b[i] = *(const u16x8*)&Bs[wn + 16 * i + (lane & 15)][8 * (lane >> 4)];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = mfma16<E>(a[i], b[j], acc[i][j]);
}

template <class E, bool NK>
__global__ __launch_bounds__(256) void grouped_any_kernel(GroupedParams P) {
  __shared__ __align__(16) uint16_t As[kT][kPad], Bs[kT][kPad];
  __shared__ int64_t row_of[kT];
  const Tile t = find_tile<kT>(P.offsets, P.E, P.M, blockIdx.x);
  if (t.e < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t n0 = (int64_t)blockIdx.y * kT;
  const int nr = (int)(t.r1 - t.r0), nc = (int)min((int64_t)kT, P.N - n0);
  uint16_t* out = (uint16_t*)P.out;
  if (t.e == P.E) {
    for (int i = tid; i < nr * nc; i += 256) out[(t.r0 + i / nc) * P.N + n0 + i % nc] = 0;
    return;
  }
  if (tid < kT) {
    int64_t r = -1;
    if (tid < nr) {
      r = P.rows ? P.rows[t.r0 + tid] : t.r0 + tid;
      if (r >= P.a_rows) r = -1;
    }
    row_of[tid] = r;
  }
  __syncthreads();
  const uint16_t* a = (const uint16_t*)P.a;
  const uint16_t* b = (const uint16_t*)P.b + (int64_t)t.e * P.N * P.K;
  f32x4 acc[2][2] = {};
  for (int64_t k0 = 0; k0 < P.K; k0 += kTk) {
    const int kc = (int)min((int64_t)kTk, P.K - k0);
    for (int i = tid; i < kT * kTk; i += 256) {
      const int m = i / kTk, k = i % kTk;
      const int64_t r = row_of[m];
      As[m][k] = r >= 0 && k < kc ? a[r * P.lda + k0 + k] : (uint16_t)0;
      if (NK) {
        Bs[m][k] = m < nc && k < kc ? b[(n0 + m) * P.K + k0 + k] : (uint16_t)0;
      } else {
        const int n = i % kT, kk = i / kT;
        Bs[n][kk] = n < nc && kk < kc ? b[(k0 + kk) * P.N + n0 + n] : (uint16_t)0;
      }
    }
    __syncthreads();
    any_step<E>(As, Bs, acc);
    __syncthreads();
  }
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = wm + 16 * i + 4 * (lane >> 4) + r, n = wn + 16 * j + (lane & 15);
        if (m < nr && n < nc) out[(t.r0 + m) * P.N + n0 + n] = E::put(acc[i][j][r]);
      }
}

// out (E, N, K): a = dy (M, N), b = x rows (., K).
template <class E, class O>
__global__ __launch_bounds__(256) void wgrad_any_kernel(GroupedParams P) {
  __shared__ __align__(16) uint16_t As[kT][kPad], Bs[kT][kPad];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int e = blockIdx.z;
  const int64_t n0 = (int64_t)blockIdx.x * kT, k0 = (int64_t)blockIdx.y * kT;
  const int64_t ra = e == 0 ? 0 : min((int64_t)max(P.offsets[e], 0), P.M);
  const int64_t rb = max(ra, min((int64_t)max(P.offsets[e + 1], 0), P.M));
  const int nc = (int)min((int64_t)kT, P.N - n0), kc = (int)min((int64_t)kT, P.K - k0);
  const uint16_t* a = (const uint16_t*)P.a;
  const uint16_t* b = (const uint16_t*)P.b;
  f32x4 acc[2][2] = {};
  for (int64_t r0 = ra; r0 < rb; r0 += kTk) {
    const int nr = (int)min((int64_t)kTk, rb - r0);
    for (int i = tid; i < kT * kTk; i += 256) {
      const int c = i % kT, m = i / kT;
      int64_t r = -1;
      if (m < nr) {
        r = P.rows ? P.rows[r0 + m] : r0 + m;
        if (r >= P.b_rows) r = -1;
      }
      As[c][m] = m < nr && c < nc ? a[(r0 + m) * P.lda + n0 + c] : (uint16_t)0;
      Bs[c][m] = r >= 0 && c < kc ? b[r * P.ldb + k0 + c] : (uint16_t)0;
    }
    __syncthreads();
    any_step<E>(As, Bs, acc);
    __syncthreads();
  }
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  typename O::raw* out = (typename O::raw*)P.out + (int64_t)e * P.N * P.K;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = wm + 16 * i + 4 * (lane >> 4) + r, k = wn + 16 * j + (lane & 15);
        if (n < nc && k < kc) out[(n0 + n) * P.K + k0 + k] = O::put(acc[i][j][r]);
      }
}

}  // namespace

hipError_t launch_grouped(const GroupedParams& P, int dtype, bool b_is_nk, hipStream_t stream) {
  const void* fn = dtype == 1 ? (b_is_nk ? (const void*)grouped_any_kernel<BF16, true>
                                         : (const void*)grouped_any_kernel<BF16, false>)
                              : (b_is_nk ? (const void*)grouped_any_kernel<F16, true>
                                         : (const void*)grouped_any_kernel<F16, false>);
  void* args[] = {(void*)&P};
  return hipLaunchKernel(fn, dim3((unsigned)max_tiles(P.M, P.E, kT), (unsigned)((P.N + kT - 1) / kT)), dim3(256), args,
                         0, stream);
}

hipError_t launch_grouped_wgrad(const GroupedParams& P, int dtype, bool out_f32, hipStream_t stream) {
  const void* fn = dtype == 1 ? (out_f32 ? (const void*)wgrad_any_kernel<BF16, F32>
                                         : (const void*)wgrad_any_kernel<BF16, BF16>)
                              : (out_f32 ? (const void*)wgrad_any_kernel<F16, F32>
                                         : (const void*)wgrad_any_kernel<F16, F16>);
  void* args[] = {(void*)&P};
  return hipLaunchKernel(fn, dim3((unsigned)((P.N + kT - 1) / kT), (unsigned)((P.K + kT - 1) / kT), (unsigned)P.E),
                         dim3(256), args, 0, stream);
}

}  // namespace bcjr
