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
// and sum per thread; its last wave does the teacher's K entries meanwhile, whose
// share of the loss needs the student's normaliser only as a factor.  The
// gradient reads the row again and writes it once, and overwrites the K entries
// behind a barrier; where loss and gradient are one call, a thread keeps its
// first C vectors of the row in registers between the two.
//
// Exponents are of differences from the row's maximum m, which are exact or nearly
// so; log2(e) / tau is held in two floats, since the rounding of one would move
// all terms the same way.  The row's sums are float32.  What is done K times or
// once a row is done in 64 bits: a divergence is a small difference of logarithms.
// stats[row] = (m, 1 / the sum, c, c - r / p_r; n as a double, 2 unused).
//
// Bound by the logits' bytes, at a copy's rate: 4,096 rows of 50,257 bfloat16, 64
// entries, take 83 us (loss, 4.9 TB/s) and 166 (gradient, 4.95), and in one call 197
// (4.2: a row's loads wait for its stores to begin, and the rows beside it on a
// compute unit cover only part of that).  8,192 rows of 131,072 take 389 (5.5), 785
// (5.5) and 915 (5.9, with the half of a row that is not kept and read twice).
#include "bcjr_moe_device.h"
#include "bcjr_moe_kernels.h"

namespace bcjr {

namespace {

constexpr int kUnroll = 4;  // vectors in flight per thread beside the kept ones
// A teacher's mass outside its entries below this is what float32 sums leave of
// 1 by rounding: none.
constexpr double kRest = 1e-6;

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float finite_or_0(float m) { return m == -INFINITY ? 0.f : m; }

// 2^(d log2(e) / tau); lo > 0, so that -inf stays -inf.
struct Scale {
  float hi, lo;
  __device__ __forceinline__ float exp(float d) const { return ex2(fmaf(d, lo, d * hi)); }
};

// Running maximum of logits, and sums of exponentials over it: all, and those
// outside the entries.
struct Run {
  float m = -INFINITY, l = 0.f, r = 0.f;
  __device__ __forceinline__ void raise(float to, Scale s2) {
    if (to > m) {
      const float f = s2.exp(m - to);  // 0 the first time
      l *= f;
      r *= f;
      m = to;
    }
  }
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// PAST: the gradient is stored past the caches.
template <class E, int KIND, bool VEC, int NT, int C, bool PAST = false>
__global__ __launch_bounds__(NT, C > 8 ? 4 : 8) void distill_kernel(DistillParams P) {
  constexpr int N = VEC ? Vec16<E>::N : 1, NW = NT / 64;
  using raw = typename E::raw;
  extern __shared__ __align__(16) uint32_t marked[];  // one bit per element, from `lead` on
  __shared__ float top[NW], part[2][NW];
  __shared__ double teacher[4];
  __shared__ int repeated;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const raw* x = (const raw*)P.logits + row * P.ld;
  raw* g = KIND == DISTILL_LOSS ? nullptr : (raw*)P.grad + row * P.V;
  const float* tv = P.values + row * P.K;
  const int32_t* ti = P.indices + row * P.K;
  const Scale s2 = {P.scale_hi, P.scale_lo};
  const bool rest = KIND != DISTILL_BACKWARD && P.teacher_lse != nullptr;
  // elements of the row's first 16-byte block that lie before the row
  const int lead = VEC ? (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(raw)) : 0;
  const int nvec = (P.V + lead + N - 1) / N;
  const int v0 = lead ? 1 : 0, v1 = (P.V + lead) / N;  // whole vectors
  const raw* xv = x - lead;
  // threads 0 and 1 take the row's ends, inside vectors that it shares with its neighbours
  const int edge = tid == 0 ? 0 : v1;
  const bool has_edge = VEC && (tid == 0 ? v0 == 1 : tid == 1 && v1 < nvec && v1 >= v0);
  auto entry = [&](int k) { return ti[k] >= 0 && ti[k] < P.V; };

  if (KIND != DISTILL_LOSS || rest) {
    const int words = (P.V + lead + 31) / 32;
    for (int i = tid; i < words; i += NT) marked[i] = 0;
    if (tid == 0) repeated = 0;
    __syncthreads();
    for (int k = tid; k < P.K; k += NT)
      if (entry(k)) {
        const int i = ti[k] + lead;
        if (atomicOr(&marked[i >> 5], 1u << (i & 31)) >> (i & 31) & 1) repeated = 1;
      }
    __syncthreads();
  }

  float m, inv, c, outside;  // m as it is subtracted
  double n;
  u32x4 keep[C > 0 ? C : 1];
  auto vector_at = [&](int v) { return *(const u32x4*)(xv + (int64_t)v * N); };
  if constexpr (KIND == DISTILL_BACKWARD) {
    const float4 s = P.stats[2 * row];
    m = s.x, inv = s.y, c = s.z, outside = s.w;
    n = *(const double*)&P.stats[2 * row + 1];
  } else {
    Run a;
    // exponentials over a vector, and the same without the entries
    auto add = [&](const float* z, int v) {
      const float ref = finite_or_0(a.m);
      float e[N], s = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) s += e[i] = s2.exp(z[i] - ref);
      a.l += s;
      if (rest) {
        const uint32_t bits = (marked[(v * N) >> 5] >> ((v * N) & 31)) & ((1u << N) - 1);
        if (bits) {
          s = 0.f;
#pragma unroll
          for (int i = 0; i < N; ++i) s += (bits >> i) & 1 ? 0.f : e[i];
        }
        a.r += s;
      }
    };
    // Vector by vector in the same order whatever is kept, so that the loss alone
    // and the loss beside its gradient have the same bits.
    auto take = [&](const float* z, int v) {
      float most = z[0];
#pragma unroll
      for (int i = 1; i < N; ++i) most = fmaxf(most, z[i]);
      a.raise(most, s2);
      add(z, v);
    };
    int v = v0 + tid;
    if constexpr (VEC) {
      if constexpr (C > 0) {
#pragma unroll
        for (int u = 0; u < C; ++u)
          if (v + u * NT < v1) keep[u] = vector_at(v + u * NT);
#pragma unroll
        for (int u = 0; u < C; ++u)
          if (v + u * NT < v1) {
            float z[N];
            unpack16<E>(keep[u], z);
            take(z, v + u * NT);
          }
        v += C * NT;
      }
      for (; v + (kUnroll - 1) * NT < v1; v += kUnroll * NT) {
        u32x4 t[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) t[u] = vector_at(v + u * NT);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          float z[N];
          unpack16<E>(t[u], z);
          take(z, v + u * NT);
        }
      }
      for (; v < v1; v += NT) {
        float z[N];
        unpack16<E>(vector_at(v), z);
        take(z, v);
      }
    } else {
      for (; v < v1; v += NT) {
        const float z = E::get(xv[v]);
        take(&z, v);
      }
    }
    if (has_edge) {
      float z[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = edge * N + i - lead;
        z[i] = e >= 0 && e < P.V ? E::get(x[e]) : -INFINITY;
      }
      take(z, edge);
    }

    // The entries, by one wave: n, sum q, the largest student logit x_k among
    // them and sum q (log q - (x - x_k) / tau).
    if (wave == NW - 1) {
      float most = -INFINITY;
      if (rest) {
        n = P.teacher_lse[row];
      } else {
        double l = 0.;
        for (int k = lane; k < P.K; k += 64)
          if (entry(k)) most = fmaxf(most, tv[k]);
        const double ref = finite_or_0(wave_max(most));
        for (int k = lane; k < P.K; k += 64)
          if (entry(k)) l += expf((float)((tv[k] - ref) * P.inv_tau));
        n = ref * P.inv_tau + log(wave_sum(l));  // -inf for a row without entries
      }
      most = -INFINITY;
      for (int k = lane; k < P.K; k += 64)
        if (entry(k)) most = fmaxf(most, E::get(x[ti[k]]));
      const double xk = finite_or_0(wave_max(most));
      double mass = 0., term = 0.;
      for (int k = lane; k < P.K; k += 64)
        if (entry(k)) {
          const double lq = tv[k] * P.inv_tau - n;
          const float q = expf((float)lq);
          mass += q;
          if (q != 0.f) term += q * (lq - (E::get(x[ti[k]]) - xk) * P.inv_tau);
        }
      mass = wave_sum(mass);
      term = wave_sum(term);
      if (lane == 0) teacher[0] = n, teacher[1] = mass, teacher[2] = term, teacher[3] = xk;
    }
    const float wm = wave_max(a.m);
    if (lane == 0) top[wave] = wm;
    __syncthreads();
    m = top[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) m = fmaxf(m, top[i]);
    m = finite_or_0(m);
    const float f = a.m == -INFINITY ? 1.f : s2.exp(a.m - m);
    const float wl = wave_sum(a.l * f), wr = rest ? wave_sum(a.r * f) : 0.f;
    if (lane == 0) part[0][wave] = wl, part[1][wave] = wr;
    __syncthreads();
    float total = 0.f, others = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      total += part[0][i];
      if (rest) others += part[1][i];
    }
    inv = 1.f / total;
    n = teacher[0];
    const double mass = teacher[1];
    double r = 0.;
    const float pr = others / total;
    if (rest) {
      r = 1. - mass;
      if (!(r > kRest)) r = 0.;
      outside = c = (float)(mass + r);
      if (r > 0. && pr > 0.f) outside = c - (float)r / pr;
    } else {
      outside = c = n == -INFINITY ? 0.f : 1.f;
    }
    if (tid == 0) {
      double loss = mass == 0. ? 0. : teacher[2] + mass * ((m - teacher[3]) * P.inv_tau + log((double)total));
      if (r > 0.) loss += r * (log(r) - log((double)pr));
      if (c == 0.f) loss = 0.;  // no entries
      P.loss[row] = (float)loss;
      if (P.stats) {
        P.stats[2 * row] = make_float4(m, inv, c, outside);
        *(double2*)&P.stats[2 * row + 1] = make_double2(n, 0.);
      }
    }
  }

  if constexpr (KIND != DISTILL_LOSS) {
    const float scale = (float)(P.g_rows[row] * P.inv_tau);
    // rows that count nothing: zeros, whatever their logits are
    const bool none = scale == 0.f || c == 0.f;
    const float go = scale * outside * inv;

    auto q_of = [&](int k) { return expf((float)(tv[k] * P.inv_tau - n)); };
    auto out = [&](float z) { return none ? 0.f : s2.exp(z - m) * go; };
    auto write = [&](int v, u32x4 t) {
      float z[N];
      unpack16<E>(t, z);
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = out(z[i]);
      u32x4* to = (u32x4*)(g - lead + (int64_t)v * N);
      if constexpr (PAST)
        __builtin_nontemporal_store(pack16<E>(z), to);
      else
        *to = pack16<E>(z);
    };
    int v = v0 + tid;
    if constexpr (VEC) {
      if constexpr (C > 0) {
        // (else the compiler keeps the 16-bit types' elements apart, in twice the registers)
#pragma unroll
        for (int u = 0; u < C; ++u) asm volatile("" : "+v"(keep[u]));
#pragma unroll
        for (int u = 0; u < C; ++u)
          if (v + u * NT < v1) write(v + u * NT, keep[u]);
        v += C * NT;
      }
      for (; v < v1; v += NT) {
        u32x4 t = {0, 0, 0, 0};
        if (!none) t = vector_at(v);
        write(v, t);
      }
    } else {
      for (; v < v1; v += NT) g[v] = E::put(out(E::get(x[v])));
    }
    if (has_edge)
      for (int i = 0; i < N; ++i) {
        const int e = edge * N + i - lead;
        if (e >= 0 && e < P.V) g[e] = E::put(out(E::get(x[e])));
      }
    if (none) return;
    __syncthreads();
    for (int k = tid; k < P.K; k += NT) {
      if (!entry(k)) continue;
      const int i = ti[k];
      float q = 0.f;
      if (!repeated) {
        q = q_of(k);
      } else {
        for (int o = 0; o < P.K; ++o)
          if (ti[o] == i) q += q_of(o);
      }
      g[i] = E::put(scale * (s2.exp(E::get(x[i]) - m) * inv * c - q));
    }
  }
}

// Threads of a row's workgroup, by its number of 16-byte vectors, for the loss and
// for the loss with its gradient (one rule, so that their bits agree).  Small
// workgroups let rows overlap their beginnings and ends; large ones keep more of a
// long row on the chip between its two uses.  Loss with gradient, microseconds,
// 256 threads keeping 12 vectors / 512 keeping 16 / 1,024 keeping 16:
//   8,192 rows of  8,000 float32  (2,000 vectors)   110 /  157 /  263
//   1,024 rows of 32,000 bfloat16 (4,000)            32 /   36 /   50
//     256 rows of 32,000 bfloat16 (4,000)            18 /   14 /   14
//   4,096 rows of 50,257 bfloat16 (6,282)           217 /  207 /  255
//   8,192 rows of 131,072 bfloat16 (16,384)       1,215 /  986 / 1,076
//   4,096 rows of 131,072 float32 (32,768)        1,212 / 1,112 /  920
// (Keeping none cost 140, 34, 14, 218, 1,055 and 1,166 at the best width of each.  All
// stored through the caches; large gradients go past them now, 197 and 915 for 207 and
// 986.)
int row_threads(int64_t nvec) { return nvec < 3000 ? 256 : nvec <= 16384 ? 512 : 1024; }

template <class E, bool PAST>
const void* distill_ptr(int kind, bool vec, int nt) {
  if (kind == DISTILL_BACKWARD)
    return vec ? (const void*)distill_kernel<E, DISTILL_BACKWARD, true, 1024, 0, PAST>
               : (const void*)distill_kernel<E, DISTILL_BACKWARD, false, 1024, 0>;
  if (kind == DISTILL_LOSS)
    return nt == 256   ? (const void*)distill_kernel<E, DISTILL_LOSS, true, 256, 0>
           : nt == 512 ? (const void*)distill_kernel<E, DISTILL_LOSS, true, 512, 0>
                       : (const void*)distill_kernel<E, DISTILL_LOSS, true, 1024, 0>;
  if (!vec) return (const void*)distill_kernel<E, DISTILL_BOTH, false, 1024, 0>;
  return nt == 256   ? (const void*)distill_kernel<E, DISTILL_BOTH, true, 256, 12, PAST>
         : nt == 512 ? (const void*)distill_kernel<E, DISTILL_BOTH, true, 512, 16, PAST>
                     : (const void*)distill_kernel<E, DISTILL_BOTH, true, 1024, 16, PAST>;
}
template <class E>
const void* distill_ptr(int kind, bool vec, int nt, bool past) {
  return past ? distill_ptr<E, true>(kind, vec, nt) : distill_ptr<E, false>(kind, vec, nt);
}

}  // namespace

hipError_t launch_distill(const DistillParams& P, int dtype, int kind, hipStream_t stream) {
  const size_t es = dtype == 0 ? 4 : 2;
  const bool past = P.T * P.V * (int64_t)es > kPastCaches;
  // 16-byte loads and stores need input and output rows in step
  const bool vec = kind == DISTILL_LOSS ||
                   (((reinterpret_cast<uintptr_t>(P.logits) ^ reinterpret_cast<uintptr_t>(P.grad)) & 15) == 0 &&
                    (P.T == 1 || (P.ld - P.V) * (int64_t)es % 16 == 0));
  const int nt = kind == DISTILL_BACKWARD || !vec ? 1024 : row_threads((int64_t)P.V * (int64_t)es / 16);
  const void* fn = dtype == 0   ? distill_ptr<F32>(kind, vec, nt, past)
                   : dtype == 1 ? distill_ptr<BF16>(kind, vec, nt, past)
                                : distill_ptr<F16>(kind, vec, nt, past);
  const size_t lds = kind == DISTILL_LOSS && !P.teacher_lse ? 0 : ((size_t)P.V + 8 + 31) / 32 * 4 + 16;
  hipError_t e = hipSuccess;
  if (lds > 60000) e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (e != hipSuccess) return e;
  void* args[] = {(void*)&P};
  return hipLaunchKernel(fn, dim3((unsigned)P.T), dim3(nt), args, lds, stream);
}

}  // namespace bcjr
