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
// take.  Four waves, 32 x 32 outputs each.  Bound by its two-byte loads: 512 rows
// on 64 experts of 1023 x 2047 take 145 us, 1.9 TB/s of the weights, and 2,048 rows
// 253, 34 TFLOP/s; what calls it first weighs a padded copy against that.
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
  const uint16_t* b = (const uint16_t*)P.b + (int64_t)t.e * (NK ? P.N : P.K) * P.ldb;
  f32x4 acc[2][2] = {};
  for (int64_t k0 = 0; k0 < P.K; k0 += kTk) {
    const int kc = (int)min((int64_t)kTk, P.K - k0);
    for (int i = tid; i < kT * kTk; i += 256) {
      const int m = i / kTk, k = i % kTk;
      const int64_t r = row_of[m];
      As[m][k] = r >= 0 && k < kc ? a[r * P.lda + k0 + k] : (uint16_t)0;
      if (NK) {
        Bs[m][k] = m < nc && k < kc ? b[(n0 + m) * P.ldb + k0 + k] : (uint16_t)0;
      } else {
        const int n = i % kT, kk = i / kT;
        Bs[n][kk] = n < nc && kk < kc ? b[(k0 + kk) * P.ldb + n0 + n] : (uint16_t)0;
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

// --------------------------------------------------- rows in 16-byte chunks
//
// BM x BN outputs per workgroup of eight waves, 64 of the reduction at a time:
// loads straight into LDS fill one of two buffers while the matrix instructions
// work from the other.  Lanes outside an operand read past the buffer
// descriptor's end, which gives zeros.
//
// An operand whose reduction runs along its rows (K tiles) lies in LDS as
// [row][64] and is read 16 bytes a lane; one whose reduction runs across its
// rows (the weights of the rows' gradient, both sides of the weights' gradient)
// as [64][column], read with the transposing LDS read: 16 lanes take a 4 x 16
// block, each ends with one column's four values.  The 16-byte chunks of a row
// are permuted by its number so that the 16 lanes of a read's pass meet
// distinct banks (counted conflicts: none).
//
// With many rows the matrix instructions bind, at the clock that the card's power
// allows under them: 64 groups of 512 rows, 2048 x 2048, take 245 us forward, 1.12
// PFLOP/s (a library's product of 8192 cubed 1.32), 1.75 GHz with the matrix units
// busy 56 % of the time; uneven groups add short tiles and a longer last round (0.82).
// The weights' gradient, 465 us, also writes E N K values in float32.  With few
// rows the weights' bytes bind: 32 rows on about 26 of 64 experts take 45 us, 4.9 TB/s.
// Side by side on the large products, 256 x 256 tiles beat 128 x 256 and 128 x 128
// (less data moved per instruction), and two buffers of 64 beat three to five of 32
// (64-byte pieces of rows).
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kBK = 64;
constexpr int kFastThreads = 512;

// Row tile: byte offset of 16-byte chunk c (of 8) of row r.
__device__ __forceinline__ int row_at(int r, int c) { return r * 128 + ((c ^ ((r >> 1) & 7)) << 4); }
// Column tile of width W: permutation of reduction row r's chunks, and byte
// offset of its chunk c.  (Rows of 64 columns are half of the banks.)
template <int W>
__device__ __forceinline__ int col_swizzle(int r) {
  return W >= 128 ? 2 * ((r & 3) | ((r >> 1) & 4)) : 2 * (((r >> 1) & 1) | ((r >> 2) & 2));
}
template <int W>
__device__ __forceinline__ int col_at(int r, int c) {
  return r * W * 2 + ((c ^ col_swizzle<W>(r)) << 4);
}

// Fragment of 16 outputs (from o on) x 32 of the reduction (step ks of 2).
template <bool COL, int W>
__device__ __forceinline__ u16x8 fragment(const char* lds, int o, int ks) {
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  if constexpr (!COL) {
    return *(const u16x8*)(lds + row_at(o + i, 4 * ks + g));
  } else {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int r = 32 * ks + 8 * g + (i >> 2);
    const char* p = lds + col_at<W>(r, (o >> 3) + ((i >> 1) & 1)) + (i & 1) * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * W * 2));
    return __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// w (E, N, K); w (E, K, N); the weights' gradient; float32 w (E, N, K)
enum { GM_NK, GM_KN, GM_WG, GM_NF };

struct Place {
  int e;
  int64_t r0, r1;  // rows of the tile (products), of the group (weights' gradient)
  int64_t n0;
  bool first;      // the first row tile of its group
};

// A value that all lanes have alike, in scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)x) | (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32);
}

// Rows [a, b) of group e (E: those behind the last group; beyond: none).
__device__ __forceinline__ void group_rows(const int32_t* offsets, int E, int M, int e, int* a, int* b) {
  *a = *b = 0;
  if (e <= E) {
    *a = e == 0 ? 0 : min(max(offsets[e], 0), M);
    *b = max(*a, e == E ? M : min(max(offsets[e + 1], 0), M));
  }
}

// The workgroup's output tile of a product.  Workgroups go to the chip's eight
// dies in turn, each with an L2 of its own, so each die takes a contiguous part
// of the tiles, ordered by expert, then column, then row: an expert's weights
// are read by one die (two at the seams), and neighbours share a column panel.
// (All tiles of full height before the short ones fill the last round better, but
// read the weights twice: 64 uneven groups of 32,768 rows, 2048 x 2048, 351 us for
// 336.  Parts by cost, a short tile half of a full one, 344; the search for them
// takes longer, 276 for 262 with even groups.)
template <int BM>
__device__ __forceinline__ bool find_place(const int32_t* offsets, int E, int M, int nt, int id, Place* out) {
  const int lane = threadIdx.x & 63;
  int a, b, n, upto;  // of this lane's group: rows, row tiles, row tiles up to its end
  auto groups = [&](int i) {
    group_rows(offsets, E, M, i + lane, &a, &b);
    upto = n = (b - a + BM - 1) / BM;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o);
      if (lane >= o) upto += x;
    }
  };
  int64_t total = 0;
  for (int i = 0; i <= E; i += 64) {
    groups(i);
    total += uniform(__shfl(upto, 63));
  }
  if (total > (int64_t)M / BM + E + 1) return false;  // offsets that do not ascend
  const int tiles = (int)total * nt, per = (tiles + 7) / 8, seq = id >> 3, at = (id & 7) * per + seq;
  if (seq >= per || at >= tiles) return false;
  int done = 0;
  for (int i = 0; i <= E; i += 64) {
    if (E >= 64) groups(i);
    const int first = (done + upto - n) * nt;
    const unsigned long long here = __ballot(at >= first && at < first + n * nt);
    if (here) {
      const int src = __ffsll(here) - 1;
      const int ea = uniform(__shfl(a, src)), eb = uniform(__shfl(b, src)), en = uniform(__shfl(n, src));
      const int local = at - uniform(__shfl(first, src)), r0 = ea + local % en * BM;
      out->e = i + src;
      out->r0 = r0;
      out->r1 = min(r0 + BM, eb);
      out->n0 = local / en;
      out->first = r0 == ea;
      return true;
    }
    done += uniform(__shfl(upto, 63));
  }
  return false;
}

// The workgroup's expert and output tile of the weights' gradient.  The tiles of
// every expert are spread over all dies, xa x xb of them (xa xb = 8) across its
// rows and columns, so that a die reads 1/xa of dy and 1/xb of x, and the dies
// have alike to do however the rows are shared; the groups with the most rows
// come first (up to 64 experts), so that the last to end are short.
__device__ __forceinline__ bool find_wgrad_place(const GroupedParams& P, int tm, int tn, int64_t id, Place* out) {
  const int lane = threadIdx.x & 63, die = (int)(id & 7);
  const int xa = P.split, xb = 8 / xa;
  const int pm = (tm + xa - 1) / xa, pn = (tn + xb - 1) / xb;
  const int64_t seq = id >> 3;
  int e = (int)(seq / (pm * pn));
  const int local = (int)(seq % (pm * pn));
  const int i = local / pn * xa + die / xb, j = local % pn * xb + die % xb;
  if (e >= P.E || i >= tm || j >= tn) return false;
  int a, b;
  if (P.E <= 64) {
    group_rows(P.offsets, P.E, (int)P.M, lane < P.E ? lane : P.E + 1, &a, &b);
    const int n = b - a;
    int rank = 0;
    for (int o = 0; o < P.E; ++o) {
      const int other = __builtin_amdgcn_readlane(n, o);
      rank += other > n || (other == n && o < lane);
    }
    e = __ffsll(__ballot(lane < P.E && rank == e)) - 1;
  }
  group_rows(P.offsets, P.E, (int)P.M, e, &a, &b);
  out->e = uniform(e);
  out->r0 = uniform(a);
  out->r1 = uniform(b);
  out->n0 = (int64_t)i * tn + j;
  return true;
}

typedef __attribute__((address_space(3))) char lds_char;
constexpr int kAhead = 2;  // groups of matrix instructions that a fragment is read ahead
constexpr uint32_t kOutside = 0xffffffffu;  // a buffer offset that loads zeros

// S times: loads 16 bytes a lane from `base` + off[s] into the KiB of LDS at `to`
// (uniform) + 8 KiB s, in lane order; no register receives data.  Written as
// instructions because the compiler lets the transposing LDS reads of the other
// buffer wait for every such load that it sees.  Whoever reads the LDS waits for
// vmcnt first.  Five wait states stand between a vector instruction that wrote a
// scalar of the descriptor and the load that reads it, one after m0 is written: the
// compiler counts none inside asm.
#define BCJR_NEXT_KIB(off) "\n\ts_add_u32 m0, m0, 0x2000\n\ts_nop 0\n\tbuffer_load_dwordx4 " off ", %1, 0 offen lds"
template <int S>
__device__ __forceinline__ void load_to_lds(const char* base, const uint32_t (&off)[S], char* to) {
  static_assert(S == 1 || S == 2 || S == 4);
  const uint64_t b = (uint64_t)uniform((int64_t)base);
  const u32x4 desc = {(uint32_t)b, (uint32_t)(b >> 32) & 0xffffu, 0xfffffff0u, 0x00027000u};
  const uint32_t at = (uint32_t)uniform((int)(uint32_t)(uintptr_t)(lds_char*)to);
#define BCJR_FIRST_KIB "s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %2, %1, 0 offen lds"
  if constexpr (S == 1)
    asm volatile(BCJR_FIRST_KIB ::"s"(at), "s"(desc), "v"(off[0]) : "memory", "m0");
  else if constexpr (S == 2)
    asm volatile(BCJR_FIRST_KIB BCJR_NEXT_KIB("%3")::"s"(at), "s"(desc), "v"(off[0]), "v"(off[1])
                 : "memory", "m0", "scc");
  else
    asm volatile(BCJR_FIRST_KIB BCJR_NEXT_KIB("%3") BCJR_NEXT_KIB("%4") BCJR_NEXT_KIB("%5")::"s"(at), "s"(desc),
                 "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3])
                 : "memory", "m0", "scc");
#undef BCJR_FIRST_KIB
}
#undef BCJR_NEXT_KIB

// LDS of a wave: what its lanes wrote before, all of them read after.  (The LDS
// works off a wave's instructions in order: only the compiler has to keep them.)
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <class E, class O, int MODE, int BM, int BN>
__global__ __launch_bounds__(kFastThreads, 2) void grouped_tile_kernel(GroupedParams P) {
  constexpr bool ACOL = MODE == GM_WG, BCOL = MODE == GM_KN || MODE == GM_WG, BF32 = MODE == GM_NF;
  constexpr int WM = 2, WN = 4;                             // waves along rows and columns
  static_assert(BM % 64 == 0 && BN % 64 == 0);
  constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;       // 16 x 16 blocks of a wave
  constexpr int kABytes = BM * kBK * 2, kBytes = kABytes + BN * kBK * 2;
  extern __shared__ __align__(16) char lds[];  // two buffers of kBytes
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  Place t;
  int K;  // the reduction's length
  if constexpr (MODE == GM_WG) {
    if (!find_wgrad_place(P, (int)((P.N + BM - 1) / BM), (int)((P.K + BN - 1) / BN), blockIdx.x, &t)) return;
    K = (int)(t.r1 - t.r0);
  } else {
    if (!find_place<BM>(P.offsets, P.E, (int)P.M, (int)((P.N + BN - 1) / BN), blockIdx.x, &t)) return;
    K = t.e == P.E ? 0 : (int)P.K;
  }
  // m0: first row (product) or column of dy (weights' gradient); n0: first column
  const int64_t m0 = MODE == GM_WG ? t.n0 / ((P.K + BN - 1) / BN) * BM : t.r0;
  const int64_t n0 = (MODE == GM_WG ? t.n0 % ((P.K + BN - 1) / BN) : t.n0) * BN;
  const int64_t mend = MODE == GM_WG ? P.N : t.r1, nend = MODE == GM_WG ? P.K : P.N;

  // Buffer s of a wave is 1 KiB of LDS: 8 rows of a row tile, 2 or 4 of a column
  // tile, wave by wave.  This thread's row, chunk and byte offset in the operand
  // (kOutside: none).
  constexpr int SA = BM * kBK * 2 / 8192, SB = BN * kBK * 2 / 8192;
  constexpr int AR = ACOL ? 512 / BM : 8, BR = BCOL ? 512 / BN : 8;  // rows of a KiB
  auto row_of = [&](int s, int per) { return (s * 8 + wave) * per + lane / (64 / per); };
  auto a_chunk = [&](int r) { return lane % (64 / AR) ^ (ACOL ? col_swizzle<BM>(r) : (r >> 1) & 7); };
  auto b_chunk = [&](int r) { return lane % (64 / BR) ^ (BCOL ? col_swizzle<BN>(r) : (r >> 1) & 7); };
  const char* abase = (const char*)P.a;
  const char* bbase = (const char*)P.b;
  constexpr int kBSize = BF32 ? 4 : 2;
  if constexpr (MODE != GM_WG) bbase += (int64_t)t.e * (BCOL ? P.K : P.N) * P.ldb * kBSize;
  uint32_t aoff[SA], boff[SB];
  if constexpr (!ACOL) {
    if (!P.rows) abase += m0 * P.lda * 2;
#pragma unroll
    for (int s = 0; s < SA; ++s) {
      const int r = row_of(s, AR);
      aoff[s] = kOutside;
      if (m0 + r < mend) {
        const int64_t x = P.rows ? P.rows[m0 + r] : r;
        if (!P.rows || (x >= 0 && x < P.a_rows)) aoff[s] = (uint32_t)((x * P.lda + a_chunk(r) * 8) * 2);
      }
    }
  } else {
    abase += (t.r0 * P.lda + m0) * 2;
#pragma unroll
    for (int s = 0; s < SA; ++s) {
      const int r = row_of(s, AR), c = a_chunk(r) * 8;
      aoff[s] = m0 + c < mend ? (uint32_t)((r * P.lda + c) * 2) : kOutside;
    }
  }
  if constexpr (BF32) {
    bbase += n0 * P.ldb * 4;
  } else if constexpr (!BCOL) {
    bbase += n0 * P.ldb * 2;
#pragma unroll
    for (int s = 0; s < SB; ++s) {
      const int r = row_of(s, BR);
      boff[s] = n0 + r < nend ? (uint32_t)((r * P.ldb + b_chunk(r) * 8) * 2) : kOutside;
    }
  } else {
    bbase += n0 * 2;
    if (MODE == GM_WG && !P.rows) bbase += t.r0 * P.ldb * 2;
#pragma unroll
    for (int s = 0; s < SB; ++s) {
      const int r = row_of(s, BR), c = b_chunk(r) * 8;
      boff[s] = n0 + c < nend ? (uint32_t)(((MODE == GM_WG && P.rows ? 0 : r * P.ldb) + c) * 2) : kOutside;
    }
  }
  // the gathered rows of the weights' gradient, known one step ahead
  uint32_t brow[SB];
  const uint32_t bmost = (uint32_t)min(P.b_rows, (int64_t)INT32_MAX);
  auto find_rows = [&](int k0) {
    if (!P.rows) return;
#pragma unroll
    for (int s = 0; s < SB; ++s) {
      const int r = min(k0 + row_of(s, BR), K - 1);  // rows past the end are not loaded
      brow[s] = (uint32_t)P.rows[t.r0 + r];
    }
  };
  // rows or chunks that a step's reduction still has
  const int acut = ACOL ? row_of(0, AR) : a_chunk(row_of(0, AR)) * 8;
  const int bcut = BCOL ? row_of(0, BR) : b_chunk(row_of(0, BR)) * 8;
  const bool gather = MODE == GM_WG && P.rows;
  auto load = [&](int k0, char* to) {
    const char* pa = abase + (ACOL ? k0 * P.lda : (int64_t)k0) * 2;
    const char* pb = bbase + (gather ? 0 : BCOL ? k0 * P.ldb : (int64_t)k0) * 2;
    uint32_t oa[SA];
#pragma unroll
    for (int s = 0; s < SA; ++s) oa[s] = k0 + acut + (ACOL ? s * 8 * AR : 0) < K ? aoff[s] : kOutside;
    load_to_lds(pa, oa, to + wave * 1024);
    if constexpr (!BF32) {
      uint32_t ob[SB];
#pragma unroll
      for (int s = 0; s < SB; ++s) {
        ob[s] = k0 + bcut + (BCOL ? s * 8 * BR : 0) < K ? boff[s] : kOutside;
        if constexpr (MODE == GM_WG)
          if (gather) ob[s] = ob[s] != kOutside && brow[s] < bmost ? ob[s] + brow[s] * (uint32_t)(P.ldb * 2) : kOutside;
      }
      load_to_lds(pb, ob, to + kABytes + wave * 1024);
    }
    if constexpr (MODE == GM_WG) find_rows(k0 + kBK);
  };

  // float32 weights go through registers: a step's 16-byte loads, 16 lanes a row,
  // wait in `wide` for the next step, and are rounded on their way into LDS.  The
  // first row tile of a group also leaves the rounded weights behind, if asked.
  // (32,768 rows, 64 experts, 2048 x 2048: 453 us, with the copy 553; a copy first
  // and then the product 343 + 336.  32 rows: 61, with the copy 124; 272 + 42.)
  constexpr int SW = BF32 ? 2 * SB : 1;
  u32x4 wide[SW];
  const int wr = tid >> 4, wc = (tid & 15) * 4;  // row (32 more for each load), column
  const bool leave = BF32 && P.b_copy && t.first;
  auto load_wide = [&](int k0) {
    const auto rb = __builtin_amdgcn_make_buffer_rsrc((void*)uniform((int64_t)(bbase + (int64_t)k0 * 4)), 0, 0xfffffff0u,
                                                      0x00027000);
#pragma unroll
    for (int s = 0; s < SW; ++s) {
      const int r = wr + 32 * s;
      const uint32_t off = n0 + r < nend && k0 + wc < K ? (uint32_t)((r * P.ldb + wc) * 4) : kOutside;
      wide[s] = __builtin_amdgcn_raw_buffer_load_b128(rb, off, 0, 0);
    }
  };
  auto store_wide = [&](int k0, char* to) {
#pragma unroll
    for (int s = 0; s < SW; ++s) {
      const int r = wr + 32 * s;
      u16x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = E::put(__uint_as_float(wide[s][i]));
      *(u16x4*)(to + kABytes + row_at(r, wc >> 3) + (wc & 4) * 2) = v;
      if (leave && n0 + r < nend && k0 + wc < K)
        *(u16x4*)((uint16_t*)P.b_copy + ((int64_t)t.e * P.N + n0 + r) * P.K + k0 + wc) = v;
    }
  };

  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const bool busy = m0 + wm < mend && n0 + wn < nend;  // whole waves
  f32x4 acc[MI][NJ] = {};
  const int steps = (K + kBK - 1) / kBK;
  if (steps) {
    if constexpr (MODE == GM_WG) find_rows(0);
    load(0, lds);
    if constexpr (BF32) {
      load_wide(0);
      store_wide(0, lds);
      load_wide(kBK);
    }
  }
  for (int it = 0; it < steps; ++it) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this step's tiles are in LDS
    __syncthreads();
    // past the end: zeros, where nothing is read
    if constexpr (BF32) store_wide((it + 1) * kBK, lds + (~it & 1) * kBytes);
    load((it + 1) * kBK, lds + (~it & 1) * kBytes);
    if constexpr (BF32) load_wide((it + 2) * kBK);
    if (!busy) continue;
    const char* from = lds + (it & 1) * kBytes;
    // MI groups of NJ matrix instructions for either half of the step; a group's
    // fragments are read kAhead groups before it
    u16x8 fa[kAhead + 1], fb[2][NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) fb[0][j] = fragment<BCOL, BN>(from + kABytes, wn + 16 * j, 0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fa[i] = fragment<ACOL, BM>(from, wm + 16 * (i % MI), i / MI);
#pragma unroll
    for (int i = 0; i < 2 * MI; ++i) {
      const int n = i + kAhead;
      if (n < 2 * MI) fa[n % (kAhead + 1)] = fragment<ACOL, BM>(from, wm + 16 * (n % MI), n / MI);
      if (i < MI) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          if (j * MI / NJ == i) fb[1][j] = fragment<BCOL, BN>(from + kABytes, wn + 16 * j, 1);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i % MI][j] = mfma16<E>(fb[i / MI][j], fa[i % (kAhead + 1)], acc[i % MI][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // no load is under way into LDS that the next workgroup owns
  __syncthreads();                     // nor any read of what is overwritten now
  if (!busy) return;

  // A lane has four neighbouring columns of row (lane & 15) of a block.  Through
  // LDS, 16 rows at a time, stores cover whole rows of the wave's columns instead
  // of 16 pieces (64 experts, 512 rows each, 2048 x 2048: 257 -> 245 us forward,
  // 492 -> 465 us weights' gradient).
  typename O::raw* out = (typename O::raw*)P.out + (MODE == GM_WG ? (int64_t)t.e * P.N * P.K : 0);
  constexpr int WC = BN / WN, kRow = WC * 4 + 16;  // columns of a wave; bytes of a row in LDS
  char* mine = lds + wave * (16 * kRow);
  const bool vec = nend % 4 == 0 && (reinterpret_cast<uintptr_t>(P.out) & 15) == 0;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      *(f32x4*)(mine + (lane & 15) * kRow + (16 * j + 4 * (lane >> 4)) * 4) = acc[i][j];
    wave_fence();
    if (vec) {
      constexpr int lanes = WC / 4, rows = 64 / lanes;  // lanes of a row, rows of an instruction
#pragma unroll
      for (int q = 0; q < 16 / rows; ++q) {
        const int r = q * rows + lane / lanes, c = lane % lanes * 4;
        const f32x4 v = *(const f32x4*)(mine + r * kRow + c * 4);
        const int64_t m = m0 + wm + 16 * i + r, n = n0 + wn + c;
        struct alignas(4 * sizeof(typename O::raw)) { typename O::raw v[4]; } o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.v[e] = O::put(v[e]);
        if (m < mend && n < nend) {
          if (MODE == GM_WG && P.past) {
            typedef uint32_t vec_t __attribute__((ext_vector_type(sizeof(o) / 4)));
            store_past((vec_t*)(out + m * nend + n), __builtin_bit_cast(vec_t, o));
          } else {
            *(decltype(o)*)(out + m * nend + n) = o;
          }
        }
      }
    } else {
      constexpr int lanes = WC < 64 ? WC : 64, rows = 64 / lanes;
#pragma unroll 4
      for (int q = 0; q < 16 / rows; ++q)
        for (int c = lane % lanes; c < WC; c += lanes) {
          const int r = q * rows + lane / lanes;
          const int64_t m = m0 + wm + 16 * i + r, n = n0 + wn + c;
          if (m < mend && n < nend) out[m * nend + n] = O::put(*(const float*)(mine + r * kRow + c * 4));
        }
    }
    wave_fence();
  }
}

template <class E, class O, int MODE, int BM, int BN>
hipError_t launch_tile(const GroupedParams& P, hipStream_t stream) {
  const void* fn = (const void*)grouped_tile_kernel<E, O, MODE, BM, BN>;
  constexpr int bytes = 2 * (BM + BN) * kBK * 2;
  hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return e;
  int64_t tiles;
  GroupedParams Q = P;
  if (MODE == GM_WG) {
    const int64_t tm = (P.N + BM - 1) / BM, tn = (P.K + BN - 1) / BN;
    // the split over the dies that leaves the fewest without a tile, of those the squarest
    int64_t best = INT64_MAX;
    for (int xa : {2, 4, 1, 8}) {
      const int64_t per = (tm + xa - 1) / xa * ((tn + 8 / xa - 1) / (8 / xa));
      if (per < best) best = per, Q.split = xa;
    }
    tiles = best * 8 * P.E;
    Q.past = (int64_t)P.E * P.N * P.K * (int64_t)sizeof(typename O::raw) > kPastCaches;
  } else {
    tiles = (max_tiles(P.M, P.E, BM) * ((P.N + BN - 1) / BN) + 7) / 8 * 8;
  }
  if (tiles > INT32_MAX) return hipErrorInvalidConfiguration;
  void* args[] = {(void*)&Q};
  return hipLaunchKernel(fn, dim3((unsigned)tiles), dim3(kFastThreads), args, bytes, stream);
}

// Rows in 16-byte chunks (an aligned base, a stride of whole chunks), within the
// 32-bit offsets of a buffer descriptor: of the whole operand where rows are
// gathered, else of the rows that a workgroup reads at a time.
bool chunked(const void* p, int64_t ld, int64_t rows) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && rows * ld * 2 < (int64_t)0xfffffff0;
}

// Side of the square output tiles.  Larger tiles load less for the same work and
// smaller ones leave fewer compute units idle; the counts below take every group
// to have a short tile.  Measured (microseconds at 256 / 128 / 64, bfloat16, the
// groups as a router with favourites fills them; M rows, E experts, K -> N; tiles):
//   products  32,768, 64, 2048 -> 2048 (1,536 of 256)   332 / 367 / 585
//             32,768, 64, 1024 -> 1024 (768)             97 / 106 / 169
//             16,384, 16, 2048 -> 2048 (640)            158 / 169 / 270
//             16,384, 64, 2048 -> 1024 (512)            115 / 117 / 166
//              8,192, 16, 2048 -> 2048 (384)            107 / 105 / 151
//              8,192,  8, 2048 -> 2048 (320)            102 /  94 / 139
//   and of groups that hardly fill a tile of 256:
//             12,000, 64, 2048 -> 2048 (888)            178 / 189 / 247
//              8,192, 64, 2048 -> 2048 (768)            169 / 163 / 196
//              2,048, 64, 2048 -> 2048 (576)            126 / 118 / 124
//              2,048,  8, 1024 -> 1024 (192 of 128)      29 /  15 /  15
//                512,  8,  512 ->  512 (48 of 128)       16 / 8.1 / 5.9
//   and of a few rows, where the weights' bytes count and not the row tiles:
//              1,024, 64, 1024 -> 2048 (1,152 of 128)    58 /  50 /  51
//                512, 64, 2048 -> 2048 (1,088)          114 / 104 / 101
//                256, 64, 2048 -> 2048 (1,056)          111 /  99 /  93
//                 32, 64, 2048 -> 2048 (512)             52 /  45 /  44
//                 16,  8, 4096 -> 4096 (256)             81 /  60 /  52
//   the same by w (E, K, N), whose tiles of 64 are read in pieces of 128 bytes:
//                512, 64, 2048 -> 1024 (576)              - /  42 /  49
//   weights' gradient  32,768 rows, 64 experts, 2048 x 2048 (4,096) 468 / 564 / 985
//              8,192, 16, 2048 x 2048 (1,024)                      129 / 130 / 205
//              16,384, 8, 2048 x 2048 (512)                        179 / 168 / 273
//              4,096, 8, 2048 x 2048 (512)                          55 / 55 / 91
//              4,096, 16, 1024 x 1024 (256; 1,024 of 128)           49 / 25 / 38
//              2,048, 4, 512 x 2048 (64; 256 of 128)                44 / 20 / 17
int product_side(const GroupedParams& P, bool b_is_nk) {
  const int64_t groups = P.E < P.M ? P.E : P.M;
  auto tiles = [&](int64_t s) { return (P.M / s + groups) * ((P.N + s - 1) / s); };
  if (P.M >= 160 * groups && tiles(256) >= 500) return 256;
  if (P.M <= 12 * groups && b_is_nk) return 64;
  return tiles(128) < (P.M <= 64 * groups ? 512 : 176) ? 64 : 128;
}
int wgrad_side(const GroupedParams& P) {
  auto tiles = [&](int64_t s) { return P.E * ((P.N + s - 1) / s) * ((P.K + s - 1) / s); };
  return tiles(256) >= 640 ? 256 : tiles(128) >= 400 ? 128 : 64;
}

template <class E, int MODE, class O>
hipError_t launch_side(const GroupedParams& P, hipStream_t stream) {
  const int side = MODE == GM_WG ? wgrad_side(P) : product_side(P, MODE != GM_KN);
  return side == 256   ? launch_tile<E, O, MODE, 256, 256>(P, stream)
         : side == 128 ? launch_tile<E, O, MODE, 128, 128>(P, stream)
                       : launch_tile<E, O, MODE, 64, 64>(P, stream);
}

}  // namespace

bool grouped_f32w_fits(const void* a, int64_t lda, int64_t gathered_rows, const void* b, int64_t ldb, int64_t K) {
  return K % 8 == 0 && chunked(a, lda, gathered_rows > 256 ? gathered_rows : 256) &&
         (reinterpret_cast<uintptr_t>(b) & 15) == 0 && ldb % 4 == 0 && 256 * ldb * 4 < (int64_t)0xfffffff0;
}

hipError_t launch_grouped(const GroupedParams& P, int dtype, bool b_is_nk, hipStream_t stream) {
  if (P.b_f32)
    return dtype == 1 ? launch_side<BF16, GM_NF, BF16>(P, stream) : launch_side<F16, GM_NF, F16>(P, stream);
  if ((P.zero_padded || (P.K % 8 == 0 && (b_is_nk || P.N % 8 == 0))) &&
      chunked(P.a, P.lda, P.rows ? P.a_rows : 256) && chunked(P.b, P.ldb, 256)) {
    if (dtype == 1)
      return b_is_nk ? launch_side<BF16, GM_NK, BF16>(P, stream) : launch_side<BF16, GM_KN, BF16>(P, stream);
    return b_is_nk ? launch_side<F16, GM_NK, F16>(P, stream) : launch_side<F16, GM_KN, F16>(P, stream);
  }
  const void* fn = dtype == 1 ? (b_is_nk ? (const void*)grouped_any_kernel<BF16, true>
                                         : (const void*)grouped_any_kernel<BF16, false>)
                              : (b_is_nk ? (const void*)grouped_any_kernel<F16, true>
                                         : (const void*)grouped_any_kernel<F16, false>);
  void* args[] = {(void*)&P};
  return hipLaunchKernel(fn, dim3((unsigned)max_tiles(P.M, P.E, kT), (unsigned)((P.N + kT - 1) / kT)), dim3(256), args,
                         0, stream);
}

hipError_t launch_grouped_wgrad(const GroupedParams& P, int dtype, bool out_f32, hipStream_t stream) {
  if ((P.zero_padded || (P.K % 8 == 0 && P.N % 8 == 0)) && chunked(P.a, P.lda, kBK) &&
      chunked(P.b, P.ldb, P.rows ? P.b_rows : kBK)) {
    if (dtype == 1)
      return out_f32 ? launch_side<BF16, GM_WG, F32>(P, stream) : launch_side<BF16, GM_WG, BF16>(P, stream);
    return out_f32 ? launch_side<F16, GM_WG, F32>(P, stream) : launch_side<F16, GM_WG, F16>(P, stream);
  }
  const void* fn = dtype == 1 ? (out_f32 ? (const void*)wgrad_any_kernel<BF16, F32>
                                         : (const void*)wgrad_any_kernel<BF16, BF16>)
                              : (out_f32 ? (const void*)wgrad_any_kernel<F16, F32>
                                         : (const void*)wgrad_any_kernel<F16, F16>);
  void* args[] = {(void*)&P};
  return hipLaunchKernel(fn, dim3((unsigned)((P.N + kT - 1) / kT), (unsigned)((P.K + kT - 1) / kT), (unsigned)P.E),
                         dim3(256), args, 0, stream);
}

// ------------------------------------------------------------- padded copies

// Rows of n elements, copied to rows of ldo with zeros behind them, float32
// rounded to the 16-bit type.  A thread writes one 16-byte chunk, from loads that
// need no alignment but the elements'.
template <class E, class I>
__global__ __launch_bounds__(256) void pad_rows_kernel(const typename I::raw* x, int64_t ld, int64_t rows, int64_t n,
                                                       uint16_t* out, int64_t ldo) {
  const int64_t per = ldo / 8, total = rows * per;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
    const int64_t r = q / per, c = q % per * 8;
    const typename I::raw* p = x + r * ld + c;
    Vec16<E> v;
    if (c + 8 <= n) {
      typename I::raw t[8];
      __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
      for (int i = 0; i < 8; ++i) v.v[i] = E::put(I::get(t[i]));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v.v[i] = c + i < n ? E::put(I::get(p[i])) : 0;
    }
    *(Vec16<E>*)(out + r * ldo + c) = v;
  }
}

hipError_t launch_pad_rows(const void* x, int dtype_in, int64_t ld, int64_t rows, int64_t n, int dtype, void* out,
                           int64_t ldo, hipStream_t stream) {
  const int64_t blocks = (rows * (ldo / 8) + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 16384 ? blocks : 16384);
  if (dtype_in == 0) {
    if (dtype == 1)
      pad_rows_kernel<BF16, F32><<<grid, 256, 0, stream>>>((const float*)x, ld, rows, n, (uint16_t*)out, ldo);
    else
      pad_rows_kernel<F16, F32><<<grid, 256, 0, stream>>>((const float*)x, ld, rows, n, (uint16_t*)out, ldo);
  } else if (dtype == 1) {
    pad_rows_kernel<BF16, BF16><<<grid, 256, 0, stream>>>((const uint16_t*)x, ld, rows, n, (uint16_t*)out, ldo);
  } else {
    pad_rows_kernel<F16, F16><<<grid, 256, 0, stream>>>((const uint16_t*)x, ld, rows, n, (uint16_t*)out, ldo);
  }
  return hipGetLastError();
}

}  // namespace bcjr
