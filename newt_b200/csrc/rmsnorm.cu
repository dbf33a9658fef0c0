// Root-mean-square norm of rows, with the addition of a residual before it and an output in the
// input's type or in 8 bits (e4m3) with scales:
//   h = x (+ residual)                      fp32
//   y = h * rsqrt(mean(h^2) + eps) * w      fp32
//   out = y, or y / s in e4m3 with s = max|y| / 448 over the row or over `group` columns
//   residual_out = h
// One rounding per output; nothing between the loads and the stores is narrower than fp32.  Rows whose
// squares leave fp32's range (values beyond 1e16 or so, or below 1e-14 with an eps as small) are summed
// again from scaled values; that the code is there takes 0.4 of the 38.5 us below.
//
// HBM-bound: 16-bit rows with a residual and an e4m3 output move 7 bytes per element for about
// ten instructions.  A row lives in registers, ITEMS 16-byte vectors of x and of the residual per
// thread, so both are read once and all of a row's loads are in flight before its first use.
// `threads` threads share a row (32: a warp per row, eight rows per CTA; more: one row per CTA): as
// many warps as the row's vectors fill.  8191 x 4096 fp16 with a residual, e4m3 by 128 columns: 38.5 us
// (6.0 TB/s); 8 x 4096 bf16: 2.6 us, one row's chain of loads and two reductions.
// Nothing is prefetched across rows: the loads of the other resident CTAs cover a row's
// reductions.  The weight is read through L1, where it stays: x and the residual do not allocate
// there.

#include <type_traits>

#include "common.cuh"
#include "elem.cuh"
#include "shifted_row.cuh"
#include "sm100.cuh"

namespace nb200 {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kLargestSum = 0x1p+120f, kLeastSum = 0x1p-80f;   // between them no square that counts leaves fp32's range
constexpr int kMaxColumns = 32768;     // 32 values per thread are what 1024 threads have registers for
constexpr int kMaxShifted = 16384;     // of shifted rows, which take a few registers more

// The scale of values of magnitude up to `most`, and what they are multiplied with: 1 where they are
// all zero, or so small that the scale is no normal number (they become zeros).  Neither is the
// correctly rounded quotient (2^-22 relative, against e4m3's 2^-4): a division per vector would be a
// third of the kernel's instructions.  A quarter of either side, as the quick division has no divisors
// above 2^126.
__device__ __forceinline__ float e4m3_scale(float most) {
  const float s = most * (1.0f / kE4m3Max);
  return s >= 1.17549435e-38f ? s : 1.0f;
}
__device__ __forceinline__ float e4m3_factor(float most) {
  return most * (1.0f / kE4m3Max) >= 1.17549435e-38f ? __fdividef(0.25f * kE4m3Max, 0.25f * most) : 1.0f;
}

struct RmsParams {
  const void* x;
  const void* residual;   // null: none
  const void* w;
  void* out;
  void* residual_out;     // null: not wanted
  float* scales;          // e4m3 only: [rows, ceil(n / group)]
  int rows, n;
  int group_shift;        // log2 of the columns per scale; 0: one scale per row
  int threads;            // per row
  int64_t stride_x, stride_residual, stride_out, stride_residual_out, stride_scales;
  float eps;
};

// Over the threads of one row, which is one warp or the whole CTA.
template <class Op>
__device__ __forceinline__ float reduce_row(float v, float* slots, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = Op::apply(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (warps > 1) {
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    v = slots[threadIdx.x & 31];      // slots beyond the last warp hold the operation's neutral 0
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = Op::apply(v, __shfl_xor_sync(0xffffffffu, v, o));
  }
  return v;
}
struct Add {
  __device__ static float apply(float a, float b) { return a + b; }
};
struct Max {   // of magnitudes: 0 is neutral
  __device__ static float apply(float a, float b) { return fmaxf(a, b); }
};

// How a row's columns are spread over its threads.
//   ALIGNED: every row of every tensor starts on a 16-byte boundary (8-byte or 4-byte for the e4m3
//     output) and n is a multiple of the vector: a thread's E columns are neighbours.
//   SHIFTED: the rows start anywhere, but at the same remainder `m` in all tensors but the weight, as rows
//     of odd length do: vectors from the row's first boundary on, the elements around them one to a thread.
//     The weight's vectors are put together from two each, the second of which ends inside the row too.
//     A thread's columns may lie in two groups, so the groups' maxima meet in shared memory.
//   SINGLE: neither.  A warp's 32 * E columns are the same but a thread's lie 32 apart, so that every access
//     of a warp is one run of elements.
// 8191 x 4097 fp16 with a residual, e4m3 by 128: 69 us SHIFTED (issue slots: 64 % busy), 160 SINGLE (five
// accesses an element); 8191 x 4096 ALIGNED 39.
enum Spread { ALIGNED, SHIFTED, SINGLE };

// E elements from `off` < E on of the 2 * E in lo and hi.
template <typename T>
__device__ __forceinline__ Vec<T> window(const uint4& lo, const uint4& hi, int off) {
  const int bits = off * (int)sizeof(T) * 8, q = bits >> 5;
  const uint32_t a[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t b[7], c[5];
#pragma unroll
  for (int k = 0; k < 7; ++k) b[k] = (q & 1) ? a[k + 1] : a[k];
#pragma unroll
  for (int k = 0; k < 5; ++k) c[k] = (q & 2) ? b[k + 2] : b[k];
  Vec<T> r;
  r.raw.x = __funnelshift_r(c[0], c[1], bits);
  r.raw.y = __funnelshift_r(c[1], c[2], bits);
  r.raw.z = __funnelshift_r(c[2], c[3], bits);
  r.raw.w = __funnelshift_r(c[3], c[4], bits);
  return r;
}

template <typename T, bool E4M3, int ITEMS, int SPREAD, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS) rms_kernel(const RmsParams p) {
  constexpr int E = Elem<T>::kPerVec;
  constexpr bool FAST = SPREAD == ALIGNED, WHOLE = SPREAD != SINGLE;
  __shared__ float slots[2][32];
  // SHIFTED: the groups' maxima, a row's behind the other's (eight rows of one warp have at most 33 groups each)
  __shared__ uint32_t group_most[SPREAD == SHIFTED && E4M3 ? kMaxShifted / 32 : 1];
  const int warps = p.threads >> 5;
  const int per_cta = blockDim.x / p.threads;
  const int lane = threadIdx.x % p.threads;       // of the row
  const int64_t row = (int64_t)blockIdx.x * per_cta + threadIdx.x / p.threads;
  if (warps > 1) {
    if (threadIdx.x < 64) slots[threadIdx.x >> 5][threadIdx.x & 31] = 0.0f;
    __syncthreads();
  }
  if (row >= p.rows) return;     // whole warps, and only where a row is a warp
  const int n = p.n;
  const int groups = (n + (1 << p.group_shift) - 1) >> p.group_shift;
  uint32_t* most_of = group_most + threadIdx.x / p.threads * groups;
  if (SPREAD == SHIFTED && E4M3 && p.group_shift) {
    for (int g = lane; g < groups; g += p.threads) most_of[g] = 0;   // the row's first reduction is the barrier
    if (warps == 1) __syncwarp();
  }
  const T* x = static_cast<const T*>(p.x) + row * p.stride_x;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.stride_residual : nullptr;
  const T* w = static_cast<const T*>(p.w);
  const int m = SPREAD == SHIFTED ? (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)) : 0;
  const ShiftedRow at(n, m, E);
  const int head = at.head, end = SPREAD == SHIFTED ? at.end : n;     // of the vectors
  // vectors from m columns before the row on, the first of them left out where m is not 0
  const int col0 = WHOLE ? lane * E - m : (lane >> 5) * 32 * E + (lane & 31), col_step = p.threads * E;
  auto column = [&](int i, int j) { return col0 + i * col_step + (WHOLE ? j : 32 * j); };
  auto whole = [&](int i) { return (unsigned)column(i, 0) < (unsigned)end; };
  // this thread's element outside of the vectors: at most 2 E - 1 threads of a row have one
  const int alone = SPREAD != SHIFTED ? n : at.single(lane);
  const bool has_alone = SPREAD == SHIFTED && lane < at.singles();

  // this thread's part of a row; columns outside of it are 0
  auto read = [&](const T* from, Vec<T> (&to)[ITEMS]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      to[i].raw = make_uint4(0, 0, 0, 0);
      if constexpr (WHOLE) {
        if (whole(i)) to[i].raw = ld_once(from + column(i, 0));
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (column(i, j) < n) to[i].e[j] = from[column(i, j)];
      }
    }
  };
  auto read_weight = [&](Vec<T> (&to)[ITEMS]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      to[i].raw = make_uint4(0, 0, 0, 0);
      if constexpr (WHOLE) {
        if (!whole(i)) continue;
        const uint4* from = reinterpret_cast<const uint4*>(w + column(i, 0) - head);
        to[i].raw = __ldg(from);
        if (SPREAD == SHIFTED && m) to[i] = window<T>(to[i].raw, __ldg(from + 1), head);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (column(i, j) < n) to[i].e[j] = w[column(i, j)];
      }
    }
  };
  auto write = [&](T* to, const float (&from)[ITEMS * E], float from_alone) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if constexpr (WHOLE) {
        if (whole(i)) st_once(to + column(i, 0), round_elems<T>(&from[i * E]).raw);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (column(i, j) < n) to[column(i, j)] = Elem<T>::from_f32(from[i * E + j]);
      }
    }
    if (has_alone) to[alone] = Elem<T>::from_f32(from_alone);
  };

  Vec<T> xv[ITEMS], rv[ITEMS];
  read(x, xv);
  if (res) read(res, rv);
  float single = has_alone ? Elem<T>::to_f32(x[alone]) : 0.0f;
  if (res && has_alone) single += Elem<T>::to_f32(res[alone]);
  float v[ITEMS * E];
#pragma unroll
  for (int k = 0; k < ITEMS * E; ++k) v[k] = Elem<T>::to_f32(xv[k / E].e[k % E]);
  if (res) {
#pragma unroll
    for (int k = 0; k < ITEMS * E; ++k) v[k] += Elem<T>::to_f32(rv[k / E].e[k % E]);
  }
  float sum = single * single;
#pragma unroll
  for (int k = 0; k < ITEMS * E; ++k) sum = fmaf(v[k], v[k], sum);
  if (p.residual_out) write(static_cast<T*>(p.residual_out) + row * p.stride_residual_out, v, single);
  sum = reduce_row<Add>(sum, slots[0], warps);
  float eps = p.eps;
  // the same in all threads of the row
  if (__builtin_expect(!(sum < kLargestSum && (sum >= kLeastSum || eps >= kLeastSum)), 0)) {
    // squares that left fp32's range, or a row of zeros, or one that is not finite: once more, scaled
    const float f = sum < 1.0f ? 0x1p+96f : 0x1p-80f;
    eps = eps * f * f;
    single *= f;
    sum = single * single;
#pragma unroll
    for (int k = 0; k < ITEMS * E; ++k) {
      v[k] *= f;
      sum = fmaf(v[k], v[k], sum);
    }
    if (warps > 1) __syncthreads();                         // the slots have been read
    sum = reduce_row<Add>(sum, slots[0], warps);
  }
  const float rstd = rsqrtf(sum / (float)n + eps);
  read_weight(xv);
  if (has_alone) single = single * rstd * Elem<T>::to_f32(w[alone]);
#pragma unroll
  for (int k = 0; k < ITEMS * E; ++k) v[k] = v[k] * rstd * Elem<T>::to_f32(xv[k / E].e[k % E]);

  if constexpr (!E4M3) {
    write(static_cast<T*>(p.out) + row * p.stride_out, v, single);
  } else {
    // of a thread's columns: one scale for all of them, one for those before column m and one for those
    // from it on, or one for each
    constexpr int SCALES = FAST ? 1 : SPREAD == SHIFTED ? 2 : E;
    float amax[ITEMS][SCALES];
    float most_alone = 0.0f;                    // of the group of the element outside of the vectors
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      amax[i][0] = 0.0f;
#pragma unroll
      for (int j = 0; j < E; ++j) amax[i][0] = fmaxf(amax[i][0], fabsf(v[i * E + j]));
    }
    float* scales = p.scales + row * p.stride_scales;
    if (p.group_shift == 0) {
      float most = fmaxf(amax[0][0], fabsf(single));
#pragma unroll
      for (int i = 1; i < ITEMS; ++i) most = fmaxf(most, amax[i][0]);
      most = reduce_row<Max>(most, slots[1], warps);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < SCALES; ++j) amax[i][j] = most;
      most_alone = most;
      if (lane == 0) scales[0] = e4m3_scale(most);
    } else if constexpr (FAST) {
      // a group is 32, 64 or 128 columns: 4 to 32 neighbouring lanes
      const int lanes = (1 << p.group_shift) / E;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        for (int o = lanes >> 1; o > 0; o >>= 1)
          amax[i][0] = fmaxf(amax[i][0], __shfl_xor_sync(0xffffffffu, amax[i][0], o));
        const int col = column(i, 0);
        if ((lane & (lanes - 1)) == 0 && col < n) scales[col >> p.group_shift] = e4m3_scale(amax[i][0]);
      }
    } else if constexpr (SPREAD == SHIFTED) {
      // A vector's columns from its m-th on and those before the m-th of the thread behind are E neighbours
      // from a multiple of E on, in one group; a warp's last thread leaves the thread behind to that
      // one's warp.
      const int lanes = (1 << p.group_shift) / E, in_warp = threadIdx.x & 31;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        float before = 0.0f, from = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float a = fabsf(v[i * E + j]);
          if (j < m) before = fmaxf(before, a); else from = fmaxf(from, a);
        }
        const float behind = __shfl_down_sync(0xffffffffu, before, 1);
        if (in_warp < 31) from = fmaxf(from, behind);
        for (int o = lanes >> 1; o > 0; o >>= 1) from = fmaxf(from, __shfl_xor_sync(0xffffffffu, from, o));
        // magnitudes are ordered as their bits are
        const int group_before = at.group_before(column(i, 0), p.group_shift), group_from = at.group_from(column(i, 0), p.group_shift);
        if (in_warp == 0 && group_before >= 0) atomicMax(&most_of[group_before], __float_as_uint(before));
        if ((in_warp & (lanes - 1)) == 0 && group_from >= 0) atomicMax(&most_of[group_from], __float_as_uint(from));
      }
      if (has_alone) atomicMax(&most_of[alone >> p.group_shift], __float_as_uint(fmaxf(fabsf(single), 0.0f)));
      if (warps > 1) __syncthreads(); else __syncwarp();
      if (has_alone) most_alone = __uint_as_float(most_of[alone >> p.group_shift]);
      for (int g = lane; g < groups; g += p.threads) scales[g] = e4m3_scale(__uint_as_float(most_of[g]));
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int col = column(i, 0) + m;
        amax[i][0] = __uint_as_float(most_of[min(max(col - 1, 0) >> p.group_shift, groups - 1)]);
        amax[i][1] = __uint_as_float(most_of[min(col >> p.group_shift, groups - 1)]);
      }
    } else {
      // a group is one, two or four neighbouring runs of 32 columns
      const int runs = 1 << (p.group_shift - 5);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
        for (int j = 0; j < E; ++j) amax[i][j] = sm100::warp_max(fabsf(v[i * E + j]));
#pragma unroll
        for (int step = 1; step < 4; step *= 2) {
          if (step >= runs) break;
#pragma unroll
          for (int j = 0; j < E; j += 2 * step) {
            const float most = fmaxf(amax[i][j], amax[i][j + step]);
#pragma unroll
            for (int k = 0; k < 2 * step; ++k) amax[i][j + k] = most;
          }
        }
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const int col = column(i, j) - (lane & 31);
          if ((lane & 31) == 0 && (j & (runs - 1)) == 0 && col < n) scales[col >> p.group_shift] = e4m3_scale(amax[i][j]);
        }
      }
    }
    uint8_t* out = static_cast<uint8_t*>(p.out) + row * p.stride_out;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if constexpr (WHOLE) {
        if (!whole(i)) continue;
        const float factor = e4m3_factor(amax[i][0]);
        if constexpr (SPREAD == SHIFTED) {
          const float from = e4m3_factor(amax[i][1]);
#pragma unroll
          for (int j = 0; j < E; ++j) v[i * E + j] *= j < m ? factor : from;
        }
        store_e4m3<E>(out + column(i, 0), &v[i * E], SPREAD == SHIFTED ? 1.0f : factor);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (column(i, j) < n) out[column(i, j)] = (uint8_t)e4m3x2(v[i * E + j] * e4m3_factor(amax[i][j]), 0.0f);
      }
    }
    if (has_alone) out[alone] = (uint8_t)e4m3x2(single * e4m3_factor(most_alone), 0.0f);
  }
}

template <typename T, bool E4M3, int ITEMS>
int launch_rms(const RmsParams& p, Spread spread, cudaStream_t stream) {
  const int threads = p.threads == 32 ? 256 : p.threads;
  const int64_t grid = cdiv64(p.rows, threads / p.threads);
  auto go = [&](auto kern) {
    kern<<<(int)grid, threads, 0, stream>>>(p);
    return cuda_check(cudaGetLastError(), "rmsnorm launch");
  };
  // Registers a thread: 64 fit 1024 threads.  Aligned rows do with that (bounds of 256 threads give them 68
  // and seven CTAs of 128 instead of eight: 39.1 us, not 38.8), shifted ones spill (rows of 4097 columns with bounds
  // of 512: 76 us, of 256: 69).
  auto of = [&](auto spread) {
    constexpr int S = decltype(spread)::value;
    constexpr int SMALL = S == ALIGNED ? 512 : 256;
    return threads <= SMALL ? go(rms_kernel<T, E4M3, ITEMS, S, SMALL>) : go(rms_kernel<T, E4M3, ITEMS, S, 1024>);
  };
  if (spread == ALIGNED) return of(std::integral_constant<int, ALIGNED>());
  if constexpr (ITEMS <= 4)            // what kMaxShifted columns come to
    if (spread == SHIFTED) return of(std::integral_constant<int, SHIFTED>());
  return of(std::integral_constant<int, SINGLE>());
}

template <typename T, bool E4M3>
int dispatch_rms(RmsParams p, cudaStream_t stream) {
  constexpr int E = Elem<T>::kPerVec;
  // whether all rows of a tensor start where x's do, modulo the vector; `bytes` per element
  auto with_x = [&](const void* t, int64_t stride, int bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(t), x = reinterpret_cast<uintptr_t>(p.x);
    return (at / bytes - x / sizeof(T)) % E == 0 && (stride - p.stride_x) % E == 0;
  };
  bool together = at16(p.w);
  if (p.residual) together = together && with_x(p.residual, p.stride_residual, sizeof(T));
  if (p.residual_out) together = together && with_x(p.residual_out, p.stride_residual_out, sizeof(T));
  together = together && with_x(p.out, p.stride_out, E4M3 ? 1 : sizeof(T));
  const bool aligned = p.n % E == 0 && at16(p.x) && p.stride_x % E == 0;
  const Spread spread = together && aligned ? ALIGNED
                        : together && p.n <= kMaxShifted ? SHIFTED : SINGLE;

  if (p.n > kMaxColumns)
    return fail(NB200_E_UNSUPPORTED, "rmsnorm: rows of %d elements (at most %d)", p.n, kMaxColumns);
  const int64_t vectors = spread == SHIFTED ? (p.n >= E ? p.n / E : 1) : cdiv64(p.n > 0 ? p.n : 1, E);
  int items = 1;
  // Few rows: as many threads as there are vectors, the row's latency counts (8 rows of 4096 bf16:
  // 2.6 us).  Rows for every SM: four vectors of x and of the residual in flight per thread (8191
  // rows of 4096 fp16: 41.1 us with two, 38.5 with four; of 4097: 70.7 with two, 69.1).
  const int most = p.rows < 2 * device_info().sm_count ? 1 : 4;
  while (32 * items < vectors && items < most) items *= 2;
  while (1024 * items < vectors) items *= 2;
  p.threads = 32 * (int)cdiv64(vectors, 32 * items);
  switch (items) {
    case 1: return launch_rms<T, E4M3, 1>(p, spread, stream);
    case 2: return launch_rms<T, E4M3, 2>(p, spread, stream);
    case 4: return launch_rms<T, E4M3, 4>(p, spread, stream);
  }
  if constexpr (E == 4) return launch_rms<T, E4M3, 8>(p, spread, stream);
  return fail(NB200_E_INVALID, "rmsnorm: no kernel for %d vectors per thread", items);
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" int nb200_rmsnorm(const void* x, const void* residual, const void* w, void* out,
                             void* residual_out, float* scales, int64_t rows, int64_t n,
                             int64_t stride_x, int64_t stride_residual, int64_t stride_out,
                             int64_t stride_residual_out, int64_t stride_scales, int64_t group,
                             float eps, int dtype, int out_dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (rows < 0 || n < 0)
    return fail(NB200_E_INVALID, "rmsnorm: negative size (rows=%lld n=%lld)", (long long)rows, (long long)n);
  if (rows > INT32_MAX || n > INT32_MAX)
    return fail(NB200_E_INVALID, "rmsnorm: rows / n beyond int32 (rows=%lld n=%lld)", (long long)rows,
                (long long)n);
  if (dtype != NB200_F32 && dtype != NB200_F16 && dtype != NB200_BF16)
    return fail(NB200_E_INVALID, "rmsnorm: unknown dtype code %d", dtype);
  const bool e4m3 = out_dtype == NB200_E4M3;
  if (!e4m3 && out_dtype != dtype)
    return fail(NB200_E_INVALID, "rmsnorm: the output has the input's type or e4m3 (out_dtype code %d)",
                out_dtype);
  if (e4m3 && group != 0 && group != 32 && group != 64 && group != 128)
    return fail(NB200_E_INVALID, "rmsnorm: group %lld (0: one scale per row; 32, 64, 128 columns)",
                (long long)group);
  if (!e4m3 && group != 0)
    return fail(NB200_E_INVALID, "rmsnorm: a group of columns goes with an e4m3 output");
  if (!(eps >= 0.0f)) return fail(NB200_E_INVALID, "rmsnorm: eps must not be negative");
  if (rows == 0 || (n == 0 && !(e4m3 && group == 0))) return 0;     // rows without columns still have a scale each
  if ((n > 0 && (!x || !w || !out)) || (e4m3 && !scales))
    return fail(NB200_E_INVALID, "rmsnorm: null tensor pointer");
  if (!aligned_to(bytes_of(dtype), x, residual, w, residual_out) || !aligned_to(bytes_of(out_dtype), out) || !aligned_to(4, scales))
    return fail(NB200_E_INVALID, "rmsnorm: a tensor does not start on a multiple of its element");
  RmsParams p;
  p.x = x;
  p.residual = residual;
  p.w = w;
  p.out = out;
  p.residual_out = residual_out;
  p.scales = scales;
  p.rows = (int)rows;
  p.n = (int)n;
  p.group_shift = group == 0 ? 0 : group == 32 ? 5 : group == 64 ? 6 : 7;
  p.threads = 0;
  p.stride_x = stride_x;
  p.stride_residual = stride_residual;
  p.stride_out = stride_out;
  p.stride_residual_out = stride_residual_out;
  p.stride_scales = stride_scales;
  p.eps = eps;
  switch (dtype) {
    case NB200_F32:
      return e4m3 ? dispatch_rms<float, true>(p, stream) : dispatch_rms<float, false>(p, stream);
    case NB200_F16:
      return e4m3 ? dispatch_rms<__half, true>(p, stream) : dispatch_rms<__half, false>(p, stream);
    default:
      return e4m3 ? dispatch_rms<__nv_bfloat16, true>(p, stream)
                  : dispatch_rms<__nv_bfloat16, false>(p, stream);
  }
}
