// Divergence of a student's logits from a teacher's top logits.
//
// Row by row, with z = logits / tau, p = softmax(z) over V and the teacher's K
// entries (i_k, t_k):
//   q_k = exp(t_k / tau - n), n the teacher's log-sum-exp over its whole
//   vocabulary if it is given, else over the K entries,
//   loss = sum_k q_k (log q_k - log p_{i_k}) + r (log r - log p_r),
// where r = 1 - sum q is the teacher's mass outside its entries and p_r the
// student's there (r = 0 without the teacher's normaliser).  With c = sum q + r:
//   d loss / d z_i = c p_i - q_i on the entries, p_i (c - r / p_r) elsewhere.
// p_r is summed over the elements outside the entries (a bitmap in LDS marks
// them), not subtracted from 1, so a small one keeps its digits.
//
// One workgroup takes a row.  The loss reads it once, with a running maximum
// and sum per thread; the gradient reads it again and writes it once, and
// overwrites the K entries behind a barrier.  Exponents are base 2, sums
// float32.  stats[row] = (log2-sum of z, c, c - r / p_r, n in log2 units).
#include "bcjr_moe_device.h"
#include "bcjr_moe_kernels.h"

namespace bcjr {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kUnroll = 4;  // vectors in flight per thread
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// A teacher's mass outside its entries below this is what float32 sums leave of
// 1 by rounding: none.
constexpr float kRest = 1e-6f;

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float lg2(float x) { return __builtin_amdgcn_logf(x); }

// Running maximum, sum and sum outside the entries of one thread, z in log2 units.
struct Run {
  float m = -INFINITY, l = 0.f, r = 0.f;
  __device__ __forceinline__ void raise(float to) {
    if (to > m) {
      const float f = ex2(m - to);  // 0 the first time
      l *= f;
      r *= f;
      m = to;
    }
  }
  __device__ __forceinline__ float ref() const { return m == -INFINITY ? 0.f : m; }
};

template <class E, int KIND, bool VEC>
__global__ __launch_bounds__(kThreads) void distill_kernel(DistillParams P) {
  constexpr int N = VEC ? Vec16<E>::N : 1;
  using raw = typename E::raw;
  extern __shared__ __align__(16) uint32_t marked[];  // one bit per element, from `lead` on
  __shared__ float part[6][kWaves];
  __shared__ int repeated;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const raw* x = (const raw*)P.logits + row * P.ld;
  raw* g = KIND == DISTILL_LOSS ? nullptr : (raw*)P.grad + row * P.V;
  const float* tv = P.values + row * P.K;
  const int32_t* ti = P.indices + row * P.K;
  const float s2 = P.inv_tau * kLog2e;  // logits to log2 units
  const bool rest = P.teacher_lse != nullptr;
  // elements of the row's first 16-byte block that lie before the row
  const int lead = VEC ? (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(raw)) : 0;
  const int nvec = (P.V + lead + N - 1) / N;
  const int words = (P.V + lead + 31) / 32;
  const int v0 = lead ? 1 : 0, v1 = (P.V + lead) / N;  // whole vectors
  const raw* xv = x - lead;

  const float gr = KIND == DISTILL_LOSS ? 0.f : P.g_rows[row];
  for (int i = tid; i < words; i += kThreads) marked[i] = 0;
  if (tid == 0) repeated = 0;
  __syncthreads();
  for (int k = tid; k < P.K; k += kThreads) {
    const int i = ti[k];
    if (i >= 0 && i < P.V) {
      const uint32_t bit = 1u << ((i + lead) & 31);
      if (atomicOr(&marked[(i + lead) >> 5], bit) & bit) repeated = 1;
    }
  }

  float lse2, c, outside, n2;
  if constexpr (KIND == DISTILL_BACKWARD) {
    const float4 s = P.stats[row];
    lse2 = s.x, c = s.y, outside = s.z, n2 = s.w;
    __syncthreads();
  } else {
    // the teacher's normaliser, log2 units
    if (rest) {
      n2 = P.teacher_lse[row] * kLog2e;
      __syncthreads();
    } else {
      float m = -INFINITY, l = 0.f;
      for (int k = tid; k < P.K; k += kThreads)
        if (ti[k] >= 0 && ti[k] < P.V) m = fmaxf(m, tv[k] * s2);
      m = group_max<kWaves>(m, part[0]);
      const float ref = m == -INFINITY ? 0.f : m;
      for (int k = tid; k < P.K; k += kThreads)
        if (ti[k] >= 0 && ti[k] < P.V) l += ex2(tv[k] * s2 - ref);
      l = group_sum<kWaves>(l, part[1]);
      n2 = ref + lg2(l);  // -inf for a row without entries
    }

    Run a;
    auto add = [&](const float* z, uint32_t bits) {
      const float ref = a.ref();
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) s += ex2(z[i] - ref);
      a.l += s;
      if (rest) {
        if (bits) {
          s = 0.f;
#pragma unroll
          for (int i = 0; i < N; ++i) s += (bits >> i) & 1 ? 0.f : ex2(z[i] - ref);
        }
        a.r += s;
      }
    };
    auto bits_of = [&](int v) {
      return rest ? (marked[(v * N) >> 5] >> ((v * N) & 31)) & ((1u << N) - 1) : 0u;
    };
    for (int v = v0 + tid; v < v1; v += kThreads * kUnroll) {
      float z[kUnroll][N];
      int nv = 0;
      float m = -INFINITY;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (v + u * kThreads >= v1) break;
        nv = u + 1;
        if constexpr (VEC) {
          const Vec16<E> t = *(const Vec16<E>*)(xv + (int64_t)(v + u * kThreads) * N);
#pragma unroll
          for (int i = 0; i < N; ++i) z[u][i] = E::get(t.v[i]);
        } else {
          z[u][0] = E::get(xv[v + u * kThreads]);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (u >= nv) break;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          z[u][i] *= s2;
          m = fmaxf(m, z[u][i]);
        }
      }
      a.raise(m);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (u >= nv) break;
        add(z[u], bits_of(v + u * kThreads));
      }
    }
    // the row's ends, inside vectors that it shares with its neighbours
    if (VEC && tid < 2) {
      const int v = tid == 0 ? 0 : v1;
      if ((tid == 0 ? v0 == 1 : v1 < nvec && v1 >= v0) ) {
        float z[N], m = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int e = v * N + i - lead;
          z[i] = e >= 0 && e < P.V ? E::get(x[e]) * s2 : -INFINITY;
          m = fmaxf(m, z[i]);
        }
        a.raise(m);
        add(z, bits_of(v));
      }
    }
    const float m = group_max<kWaves>(a.m, part[2]);
    const float ref = m == -INFINITY ? 0.f : m;
    const float f = ex2(a.ref() - ref);
    const float total = group_sum<kWaves>(a.m == -INFINITY ? a.l : a.l * f, part[3]);
    lse2 = ref + lg2(total);

    // the entries
    float term = 0.f, mass = 0.f;
    for (int k = tid; k < P.K; k += kThreads) {
      const int i = ti[k];
      if (i < 0 || i >= P.V) continue;
      const float lq = tv[k] * s2 - n2, q = ex2(lq);
      mass += q;
      if (q != 0.f) term += q * (lq - (E::get(x[i]) * s2 - lse2)) * kLn2;
    }
    term = group_sum<kWaves>(term, part[4]);
    mass = group_sum<kWaves>(mass, part[5]);
    outside = c = rest ? mass : (n2 == -INFINITY ? 0.f : 1.f);
    if (rest) {
      __syncthreads();
      const float pr = group_sum<kWaves>(a.m == -INFINITY ? a.r : a.r * f, part[0]) / total;
      float r = 1.f - mass;
      r = r > kRest ? r : 0.f;
      c = mass + r;
      outside = c;
      if (r > 0.f) {
        term += r * (lg2(r) - lg2(pr)) * kLn2;
        if (pr > 0.f) outside = c - r / pr;
      }
    }
    if (c == 0.f) term = 0.f;  // no entries
    if (tid == 0) {
      P.loss[row] = term;
      if (P.stats) P.stats[row] = make_float4(lse2, c, outside, n2);
    }
  }

  if constexpr (KIND != DISTILL_LOSS) {
    const float scale = gr * P.inv_tau;
    // rows that count nothing: zeros, whatever their logits are
    const bool none = scale == 0.f || c == 0.f;
    const float go = scale * outside;
    auto out = [&](float z) { return none ? 0.f : ex2(fmaf(z, s2, -lse2)) * go; };
    for (int v = v0 + tid; v < v1; v += kThreads) {
      if constexpr (VEC) {
        Vec16<E> t = {};
        if (!none) t = *(const Vec16<E>*)(xv + (int64_t)v * N);
#pragma unroll
        for (int i = 0; i < N; ++i) t.v[i] = E::put(out(E::get(t.v[i])));
        *(Vec16<E>*)(g - lead + (int64_t)v * N) = t;
      } else {
        g[v] = E::put(out(E::get(x[v])));
      }
    }
    if (VEC && tid < 2) {
      const int v = tid == 0 ? 0 : v1;
      if ((tid == 0 ? v0 == 1 : v1 < nvec && v1 >= v0))
        for (int i = 0; i < N; ++i) {
          const int e = v * N + i - lead;
          if (e >= 0 && e < P.V) g[e] = E::put(out(E::get(x[e])));
        }
    }
    if (none) return;
    __syncthreads();
    for (int k = tid; k < P.K; k += kThreads) {
      const int i = ti[k];
      if (i < 0 || i >= P.V) continue;
      float q = 0.f;
      if (!repeated) {
        q = ex2(tv[k] * s2 - n2);
      } else {
        for (int o = 0; o < P.K; ++o)
          if (ti[o] == i) q += ex2(tv[o] * s2 - n2);
      }
      g[i] = E::put(scale * (ex2(fmaf(E::get(x[i]), s2, -lse2)) * c - q));
    }
  }
}

template <class E, bool VEC>
const void* distill_ptr(int kind) {
  return kind == DISTILL_LOSS       ? (const void*)distill_kernel<E, DISTILL_LOSS, VEC>
         : kind == DISTILL_BACKWARD ? (const void*)distill_kernel<E, DISTILL_BACKWARD, VEC>
                                    : (const void*)distill_kernel<E, DISTILL_BOTH, VEC>;
}

}  // namespace

hipError_t launch_distill(const DistillParams& P, int dtype, int kind, hipStream_t stream) {
  const size_t es = dtype == 0 ? 4 : 2;
  // 16-byte loads and stores need input and output rows in step
  const bool vec = kind == DISTILL_LOSS ||
                   (((reinterpret_cast<uintptr_t>(P.logits) ^ reinterpret_cast<uintptr_t>(P.grad)) & 15) == 0 &&
                    (P.T == 1 || (P.ld - P.V) * (int64_t)es % 16 == 0));
  const void* fn = dtype == 0   ? (vec ? distill_ptr<F32, true>(kind) : distill_ptr<F32, false>(kind))
                   : dtype == 1 ? (vec ? distill_ptr<BF16, true>(kind) : distill_ptr<BF16, false>(kind))
                                : (vec ? distill_ptr<F16, true>(kind) : distill_ptr<F16, false>(kind));
  const size_t lds = ((size_t)P.V + 8 + 31) / 32 * 4 + 16;
  hipError_t e = hipSuccess;
  if (lds > 60000) e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (e != hipSuccess) return e;
  void* args[] = {(void*)&P};
  return hipLaunchKernel(fn, dim3((unsigned)P.T), dim3(kThreads), args, lds, stream);
}

}  // namespace bcjr
