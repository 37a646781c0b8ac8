// Routing of tokens to experts, and the weighted sum of the experts' rows.
//
// Routing (moe_route).  Per token: p = softmax(l) over E experts, the k largest
// logits (equal ones by the lowest index, a logit of -inf never), and their
// weights: p, or p over the sum of the chosen.  The T*k (token, expert) pairs
// are sorted by expert and, within one, by token: `rows` gives each sorted
// place's token, `slots` each pair's place.
//
// A token is held by 16 lanes (64 where E > 256 or k > 16), the logits in
// registers; one of the k picks is a maximum of 64-bit keys (order of the
// logit, then lowest index) over the registers and the lanes.  The sort needs
// no global atomics: the pairs of a block of tokens set one bit per token in
// the expert's mask in LDS, so a pair's place in its block is the number of
// lower bits, a block's count the number of bits, and a block's start the sum
// of the counts before it.  Equal calls give equal results.
//
// Up to kRouteOneBlock tokens one launch does all; more take two, one for the
// picks and the counts of every block, one for the places, whose blocks sum the
// counts before their own; above 256 blocks that would read too much, and a
// launch between the two sums them once.
//
// Nothing here is bound by bytes: 16,384 tokens of 64 experts, 8 chosen, float32
// move 11 MB there and back, 2 us of a copy, and take 9.1 us (picks), 7.9 (places)
// and 5.4 (gradient).  A pick is a chain of four exchanges between lanes, k of them
// in series; the places wait for the counts of all blocks.  One launch for 4
// tokens takes 5.5 us, hardly more than an empty one.
#include <algorithm>

#include "bcjr_moe_device.h"
#include "bcjr_moe_kernels.h"

namespace bcjr {

namespace {

constexpr int kThreads = 1024;

// Order of a float as an unsigned: NaN above all, -0 with +0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
constexpr uint32_t kOrderNone = 0x007fffffu;  // of -inf: never chosen

template <int LPT>
__device__ __forceinline__ float lanes_max(float x) {
#pragma unroll
  for (int o = LPT / 2; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, LPT));
  return x;
}
template <int LPT>
__device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
  for (int o = LPT / 2; o; o >>= 1) x += __shfl_xor(x, o, LPT);
  return x;
}

// Places of the pairs of a block from the masks in LDS: base[e] is the sorted
// place of the block's first pair of expert e.
__device__ __forceinline__ int rank_in_block(const unsigned long long* mask, int words, int e, int t) {
  const unsigned long long* m = mask + e * words;
  int n = __popcll(m[t >> 6] & ((1ull << (t & 63)) - 1));
  for (int w = 0; w < (t >> 6); ++w) n += __popcll(m[w]);
  return n;
}

// Exclusive sum of n counts in LDS by the first wave; the total goes to [n].
__device__ __forceinline__ void exclusive_sum(int* c, int n) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int carry = 0;
    for (int i = 0; i < n; i += 64) {
      const int own = i + lane < n ? c[i + lane] : 0;
      int x = own;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
      }
      if (i + lane < n) c[i + lane] = carry + x - own;
      carry += __shfl(x, 63);
    }
    if (lane == 0) c[n] = carry;
  }
  __syncthreads();
}

// ONE: the whole sort in this launch (one workgroup); else the block's counts
// go to counts[block][E].
template <class E, int LPT, int VPL, bool ONE>
__global__ __launch_bounds__(kThreads) void route_kernel(RouteParams P) {
  extern __shared__ __align__(16) char lds[];
  unsigned long long* mask = (unsigned long long*)lds;  // E * words
  int* count = (int*)(mask + (size_t)P.E * P.words);    // E + 1 (ONE)
  const int tid = threadIdx.x, sub = tid % LPT, TB = P.words * 64;
  const int64_t t0 = (int64_t)blockIdx.x * TB;
  const int nt = (int)(P.T - t0 < TB ? P.T - t0 : TB);
  for (int i = tid; i < P.E * P.words; i += kThreads) mask[i] = 0;
  __syncthreads();

  for (int tb = tid / LPT; tb < nt; tb += kThreads / LPT) {
    const int64_t t = t0 + tb;
    const typename E::raw* l = (const typename E::raw*)P.logits + t * P.ld;
    const bool valid = !P.valid || P.valid[t];
    float x[VPL];
    uint32_t key[VPL];
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int e = v * LPT + sub;
      x[v] = e < P.E && valid ? E::get(l[e]) : -INFINITY;
      key[v] = order_of(x[v]);
      top = fmaxf(top, x[v]);
    }
    top = lanes_max<LPT>(top);
    if (top == -INFINITY) top = 0.f;  // nothing to choose, or only NaN
    float total = 0.f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) total += __expf(x[v] - top);
    total = lanes_sum<LPT>(total);

    // lane j keeps the j-th pick
    int my_e = -1;
    float my_x = -INFINITY;
    for (int j = 0; j < P.k; ++j) {
      uint32_t bk = 0;
      int bv = 0;
#pragma unroll
      for (int v = 0; v < VPL; ++v)
        if (key[v] > bk) bk = key[v], bv = v;
      uint64_t best = ((uint64_t)bk << 32) | (uint32_t)~(bv * LPT + sub);
#pragma unroll
      for (int o = LPT / 2; o; o >>= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)best, o, LPT);
        best = other > best ? other : best;
      }
      if ((uint32_t)(best >> 32) <= kOrderNone) break;  // the same for all lanes of the token
      const int e = (int)~(uint32_t)best;
      float xe = 0.f;
#pragma unroll
      for (int v = 0; v < VPL; ++v)
        if (v * LPT + sub == e) xe = x[v], key[v] = 0;
      xe = __shfl(xe, e % LPT, LPT);
      if (sub == j) my_e = e, my_x = xe;
    }
    float w = my_e >= 0 ? __expf(my_x - top) : 0.f;
    if (P.renormalize) total = lanes_sum<LPT>(w);
    if (my_e >= 0) w /= total;
    if (sub < P.k) {
      P.weights[t * P.k + sub] = w;
      P.experts[t * P.k + sub] = my_e;
      if (my_e >= 0) atomicOr(&mask[my_e * P.words + (tb >> 6)], 1ull << (tb & 63));
    }
  }
  __syncthreads();

  for (int e = tid; e < P.E; e += kThreads) {
    int n = 0;
    for (int w = 0; w < P.words; ++w) n += __popcll(mask[e * P.words + w]);
    if (ONE)
      count[e] = n;
    else
      P.counts[(size_t)blockIdx.x * P.E + e] = n;
  }
  if (ONE) {
    __syncthreads();
    exclusive_sum(count, P.E);
    for (int e = tid; e <= P.E; e += kThreads) P.offsets[e] = count[e];
    const int pairs = nt * P.k, live = count[P.E];
    for (int i = tid; i < pairs; i += kThreads) {
      const int t = i / P.k, e = P.experts[i];
      int at = -1;
      if (e >= 0) {
        at = count[e] + rank_in_block(mask, P.words, e, t);
        P.rows[at] = t;
      }
      P.slots[i] = at;
      if (i >= live) P.rows[i] = -1;
    }
  }
}

// counts[block][e] becomes the sum of the blocks before it; the totals follow
// behind the last block.  A workgroup takes 64 experts, its waves parts of the
// blocks.
__global__ __launch_bounds__(kThreads) void route_scan_kernel(int32_t* counts, int nb, int E) {
  constexpr int kParts = kThreads / 64;
  __shared__ int sums[kParts][64];
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6, e = blockIdx.x * 64 + lane;
  const int per = (nb + kParts - 1) / kParts, b0 = min(part * per, nb), b1 = min(b0 + per, nb);
  int sum = 0;
  if (e < E)
    for (int b = b0; b < b1; ++b) sum += counts[(size_t)b * E + e];
  sums[part][lane] = sum;
  __syncthreads();
  int at = 0;
  for (int p = 0; p < part; ++p) at += sums[p][lane];
  if (e >= E) return;
  for (int b = b0; b < b1; ++b) {
    const int c = counts[(size_t)b * E + e];
    counts[(size_t)b * E + e] = at;
    at += c;
  }
  if (part == kParts - 1) counts[(size_t)nb * E + e] = at;
}

// The places of one block's pairs.  Unless SCANNED, every block sums the counts
// it needs.
template <bool SCANNED>
__global__ __launch_bounds__(kThreads) void route_place_kernel(RouteParams P) {
  extern __shared__ __align__(16) char lds[];
  unsigned long long* mask = (unsigned long long*)lds;
  int* start = (int*)(mask + (size_t)P.E * P.words);  // E + 1: first the totals of all blocks
  int* before = start + P.E + 1;                      // E: pairs of the blocks before this one
  const int tid = threadIdx.x, TB = P.words * 64;
  const int64_t t0 = (int64_t)blockIdx.x * TB;
  const int nt = (int)(P.T - t0 < TB ? P.T - t0 : TB);
  for (int i = tid; i < P.E * P.words; i += kThreads) mask[i] = 0;
  for (int e = tid; e < P.E; e += kThreads) start[e] = before[e] = 0;
  __syncthreads();
  const int nb = gridDim.x;
  if (SCANNED) {
    for (int e = tid; e < P.E; e += kThreads) {
      before[e] = P.counts[(size_t)blockIdx.x * P.E + e];
      start[e] = P.counts[(size_t)nb * P.E + e];
    }
  } else {
    // a wave sums 64 experts' counts over every nparts-th block
    const int groups = (P.E + 63) / 64, nparts = max(1, kThreads / 64 / groups);
    for (int wg = tid >> 6; wg < groups * nparts; wg += kThreads / 64) {
      const int e = wg % groups * 64 + (tid & 63), part = wg / groups;
      if (e < P.E) {
        int all = 0, mine = 0;
        for (int b = part; b < nb; b += nparts) {
          const int c = P.counts[(size_t)b * P.E + e];
          all += c;
          if (b < (int)blockIdx.x) mine += c;
        }
        atomicAdd(&start[e], all);  // whole numbers: the order does not matter
        atomicAdd(&before[e], mine);
      }
    }
  }
  const int64_t p0 = t0 * P.k;
  const int pairs = nt * P.k;
  for (int i = tid; i < pairs; i += kThreads) {
    const int e = P.experts[p0 + i], t = i / P.k;
    if (e >= 0) atomicOr(&mask[e * P.words + (t >> 6)], 1ull << (t & 63));
  }
  __syncthreads();
  exclusive_sum(start, P.E);
  if (blockIdx.x == 0)
    for (int e = tid; e <= P.E; e += kThreads) P.offsets[e] = start[e];
  const int live = start[P.E];
  for (int i = tid; i < pairs; i += kThreads) {
    const int t = i / P.k, e = P.experts[p0 + i];
    int at = -1;
    if (e >= 0) {
      at = start[e] + before[e] + rank_in_block(mask, P.words, e, t);
      P.rows[at] = (int)(t0 + t);
    }
    P.slots[p0 + i] = at;
    if (p0 + i >= live) P.rows[p0 + i] = -1;
  }
}

// dl_e = [e chosen] w_e g_e - c_e sum_j w_j g_j with c_e = p_e, or w_e of the
// chosen where the weights are renormalised.  p is computed again from the logits
// rather than kept by the forward: the same bytes, and no T x E buffer between.
template <class E, int LPT, int VPL>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteBwdParams P) {
  const int tid = threadIdx.x, sub = tid % LPT;
  const int64_t t = (int64_t)blockIdx.x * (256 / LPT) + tid / LPT;
  if (t >= P.T) return;
  const typename E::raw* l = (const typename E::raw*)P.logits + t * P.ld;
  const bool valid = !P.valid || P.valid[t];
  float x[VPL], d[VPL];
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const int e = v * LPT + sub;
    x[v] = e < P.E && valid ? E::get(l[e]) : -INFINITY;
    top = fmaxf(top, x[v]);
    d[v] = 0.f;
  }
  // one lane's pick each, passed round below
  const int my_e = sub < P.k ? P.experts[t * P.k + sub] : -1;
  const float my_w = my_e >= 0 ? P.weights[t * P.k + sub] : 0.f;
  const float my_wg = my_e >= 0 ? my_w * P.g_weights[t * P.k + sub] : 0.f;
  const float dot = lanes_sum<LPT>(my_wg);
  for (int j = 0; j < P.k; ++j) {
    const int e = __shfl(my_e, j, LPT);
    const float wg = __shfl(my_wg, j, LPT), w = __shfl(my_w, j, LPT);
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if (v * LPT + sub == e) d[v] = P.renormalize ? wg - w * dot : wg;
  }
  if (!P.renormalize) {
    top = lanes_max<LPT>(top);
    const bool none = top == -INFINITY;
    if (none) top = 0.f;
    float total = 0.f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      x[v] = __expf(x[v] - top);
      total += x[v];
    }
    total = lanes_sum<LPT>(total);
    const float c = total == 0.f ? 0.f : dot / total;
#pragma unroll
    for (int v = 0; v < VPL; ++v) d[v] -= c * x[v];
  }
  typename E::raw* g = (typename E::raw*)P.g_logits + t * P.E;
#pragma unroll
  for (int v = 0; v < VPL; ++v)
    if (v * LPT + sub < P.E) g[v * LPT + sub] = E::put(d[v]);
}

template <class E>
const void* route_ptr(int variant, bool one) {
  switch (variant) {
    case 0: return one ? (const void*)route_kernel<E, 16, 4, true> : (const void*)route_kernel<E, 16, 4, false>;
    case 1: return one ? (const void*)route_kernel<E, 16, 8, true> : (const void*)route_kernel<E, 16, 8, false>;
    case 2: return one ? (const void*)route_kernel<E, 16, 16, true> : (const void*)route_kernel<E, 16, 16, false>;
    default: return one ? (const void*)route_kernel<E, 64, 16, true> : (const void*)route_kernel<E, 64, 16, false>;
  }
}

template <class E>
const void* route_backward_ptr(int variant) {
  switch (variant) {
    case 0: return (const void*)route_backward_kernel<E, 16, 4>;
    case 1: return (const void*)route_backward_kernel<E, 16, 8>;
    case 2: return (const void*)route_backward_kernel<E, 16, 16>;
    default: return (const void*)route_backward_kernel<E, 64, 16>;
  }
}

int route_variant(int E, int k) { return k > 16 || E > 256 ? 3 : E > 128 ? 2 : E > 64 ? 1 : 0; }

// ------------------------------------------------------------------- combine

// out[t] = sum_j w[t][j] y[slots[t][j]], in the order of j, float32.  One
// thread holds 16 bytes of columns and reads them of four rows at a time; a place
// outside [0, M) counts nothing.  Bound by the read of y: 4,096 tokens of 8 rows of
// 2,048 bfloat16 take 27.8 us, 5.4 TB/s (a copy's rate is 5.1).
template <class E, bool VEC>
__global__ __launch_bounds__(256) void combine_kernel(CombineParams P) {
  constexpr int N = VEC ? Vec16<E>::N : 1;
  using raw = typename E::raw;
  const int64_t t = blockIdx.x;
  const int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * N;
  if (c >= P.N) return;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  const int32_t* slots = P.slots + t * P.k;
  const float* weights = P.weights ? P.weights + t * P.k : nullptr;
#pragma unroll 4
  for (int j = 0; j < P.k; ++j) {
    const int s = slots[j];
    if (s < 0 || s >= P.M) continue;
    const float w = weights ? weights[j] : 1.f;
    const raw* y = (const raw*)P.y + s * P.ldy + c;
    if constexpr (VEC) {
      const Vec16<E> v = *(const Vec16<E>*)y;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = fmaf(w, E::get(v.v[i]), acc[i]);
    } else {
      acc[0] = fmaf(w, E::get(*y), acc[0]);
    }
  }
  raw* o = (raw*)P.out + t * P.N + c;
  if constexpr (VEC) {
    Vec16<E> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v.v[i] = E::put(acc[i]);
    *(Vec16<E>*)o = v;
  } else {
    *o = E::put(acc[0]);
  }
}

// dy[slots[t][j]] = w[t][j] dout[t]; dw[t][j] = <dout[t], y[slots[t][j]]>; the
// rows that no pair names get zeros.  A workgroup takes one token, reads each
// of its rows of y once, and writes each row of dy once; dout[t] stays in the
// first-level cache.  The dot products meet in LDS in the waves' order, so that
// equal calls have equal bits.  Bound by bytes: 4,096 tokens of 8 rows of 2,048
// bfloat16 take 52.4 us, 5.4 TB/s.
constexpr int kCombineDots = 64;  // pairs whose dot products LDS holds at a time
template <class E, bool VEC>
__global__ __launch_bounds__(256) void combine_backward_kernel(CombineBwdParams P) {
  constexpr int N = VEC ? Vec16<E>::N : 1;
  using raw = typename E::raw;
  __shared__ float part[kCombineDots][4];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x;
  const raw* go = (const raw*)P.g_out + t * P.ldg;
  for (int j0 = 0; j0 < P.k; j0 += kCombineDots) {
    const int nj = min(kCombineDots, P.k - j0);
    for (int j = 0; j < nj; ++j) {
      const int64_t pair = t * P.k + j0 + j;
      const int s = P.slots[pair];
      const float w = P.weights[pair];
      float dot = 0.f;
      if (s >= 0 && s < P.M) {
        for (int64_t c = (int64_t)tid * N; c < P.N; c += 256 * N) {
          const raw* y = (const raw*)P.y + s * P.ldy + c;
          raw* gy = (raw*)P.g_y + s * P.N + c;
          if constexpr (VEC) {
            const Vec16<E> a = *(const Vec16<E>*)(go + c), b = *(const Vec16<E>*)y;
            Vec16<E> r;
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const float g = E::get(a.v[i]);
              dot = fmaf(g, E::get(b.v[i]), dot);
              r.v[i] = E::put(w * g);
            }
            *(Vec16<E>*)gy = r;
          } else {
            const float g = E::get(go[c]);
            dot = fmaf(g, E::get(*y), dot);
            *gy = E::put(w * g);
          }
        }
      }
      dot = wave_sum(dot);
      if ((tid & 63) == 0) part[j][tid >> 6] = dot;
    }
    __syncthreads();
    for (int j = tid; j < nj; j += 256)
      P.g_weights[t * P.k + j0 + j] = (part[j][0] + part[j][1]) + (part[j][2] + part[j][3]);
    __syncthreads();
  }
  // this token's share of the places that no pair has
  for (int j = 0; j < P.k; ++j) {
    const int64_t p = t * P.k + j;
    if (p < P.M && P.rows[p] < 0)
      for (int64_t c = tid; c < P.N; c += 256) ((raw*)P.g_y)[p * P.N + c] = 0;
  }
}

template <template <class> class F>
const void* by_type(int dtype, bool vec) {
  return dtype == 0 ? F<F32>::ptr(vec) : dtype == 1 ? F<BF16>::ptr(vec) : F<F16>::ptr(vec);
}
template <class E>
struct CombineOf {
  static const void* ptr(bool vec) {
    return vec ? (const void*)combine_kernel<E, true> : (const void*)combine_kernel<E, false>;
  }
};
template <class E>
struct CombineBackwardOf {
  static const void* ptr(bool vec) {
    return vec ? (const void*)combine_backward_kernel<E, true> : (const void*)combine_backward_kernel<E, false>;
  }
};

size_t elem_size(int dtype) { return dtype == 0 ? 4 : 2; }
bool aligned(const void* p, int64_t ld, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * elem_size(dtype)) % 16 == 0;
}

}  // namespace

hipError_t launch_route(RouteParams P, int dtype, hipStream_t stream) {
  const int v = route_variant(P.E, P.k);
  const bool one = P.T <= kRouteOneBlock;
  const int words = one ? (int)std::max<int64_t>(1, (P.T + 63) / 64) : route_words(P.T);
  P.words = words;
  const unsigned nb = (unsigned)std::max<int64_t>(1, (P.T + words * 64 - 1) / (words * 64));
  const size_t lds = (size_t)P.E * words * 8 + (2 * (size_t)P.E + 1) * 4;
  const void* fn = dtype == 0 ? route_ptr<F32>(v, one) : dtype == 1 ? route_ptr<BF16>(v, one) : route_ptr<F16>(v, one);
  hipError_t e = hipSuccess;
  if (lds > 65536) e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (e != hipSuccess) return e;
  void* args[] = {&P};
  e = hipLaunchKernel(fn, dim3(nb), dim3(kThreads), args, lds, stream);
  if (e != hipSuccess || one) return e;
  const bool scan = nb > 256;
  if (scan) {
    int n = (int)nb;
    void* sargs[] = {&P.counts, &n, &P.E};
    e = hipLaunchKernel((const void*)route_scan_kernel, dim3((unsigned)((P.E + 63) / 64)), dim3(kThreads), sargs, 0,
                        stream);
    if (e != hipSuccess) return e;
  }
  fn = scan ? (const void*)route_place_kernel<true> : (const void*)route_place_kernel<false>;
  if (lds > 65536) e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (e != hipSuccess) return e;
  return hipLaunchKernel(fn, dim3(nb), dim3(kThreads), args, lds, stream);
}

hipError_t launch_route_backward(const RouteBwdParams& P, int dtype, hipStream_t stream) {
  const int v = route_variant(P.E, P.k), per = v == 3 ? 4 : 16;
  const void* fn = dtype == 0   ? route_backward_ptr<F32>(v)
                   : dtype == 1 ? route_backward_ptr<BF16>(v)
                                : route_backward_ptr<F16>(v);
  void* args[] = {(void*)&P};
  return hipLaunchKernel(fn, dim3((unsigned)((P.T + per - 1) / per)), dim3(256), args, 0, stream);
}

hipError_t launch_combine(const CombineParams& P, int dtype, hipStream_t stream) {
  const bool vec = aligned(P.y, P.ldy, dtype) && aligned(P.out, P.N, dtype);
  const int64_t per = 256 * (vec ? (int64_t)(16 / elem_size(dtype)) : 1);
  void* args[] = {(void*)&P};
  return hipLaunchKernel(by_type<CombineOf>(dtype, vec), dim3((unsigned)P.T, (unsigned)((P.N + per - 1) / per)),
                         dim3(256), args, 0, stream);
}

hipError_t launch_combine_backward(const CombineBwdParams& P, int dtype, hipStream_t stream) {
  const bool vec = aligned(P.y, P.ldy, dtype) && aligned(P.g_out, P.ldg, dtype) && aligned(P.g_y, P.N, dtype);
  void* args[] = {(void*)&P};
  return hipLaunchKernel(by_type<CombineBackwardOf>(dtype, vec), dim3((unsigned)P.T), dim3(256), args, 0, stream);
}

}  // namespace bcjr
