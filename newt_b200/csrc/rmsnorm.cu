// Root-mean-square norm of rows, with the addition of a residual before it and an output in the
// input's type or in 8 bits (e4m3) with scales:
//   h = x (+ residual)                      fp32
//   y = h * rsqrt(mean(h^2) + eps) * w      fp32
//   out = y, or y / s in e4m3 with s = max|y| / 448 over the row or over `group` columns
//   residual_out = h
// One rounding per output; nothing between the loads and the stores is narrower than fp32.
//
// HBM-bound: 16-bit rows with a residual and an e4m3 output move 7 bytes per element for about
// ten instructions.  A row lives in registers, ITEMS 16-byte vectors of x and of the residual per
// thread, so both are read once and all of a row's loads are in flight before its first use.
// `threads` threads share a row (32: a warp per row, eight rows per CTA; more: one row per CTA).
// Nothing is prefetched across rows: the loads of the other resident CTAs cover a row's
// reductions.  The weight is read through L1, where it stays: x and the residual do not allocate
// there.

#include "common.cuh"
#include "elem.cuh"
#include "sm100.cuh"

namespace nb200 {
namespace {

constexpr float kE4m3Max = 448.0f;

// The scale of values of magnitude up to `most`, and what they are multiplied with: 1 where they are
// all zero, or so small that the scale is no normal number (they become zeros).  Neither is the
// correctly rounded quotient (2^-22 relative, against e4m3's 2^-4): a division per vector would be a
// third of the kernel's instructions.
__device__ __forceinline__ float e4m3_scale(float most) {
  const float s = most * (1.0f / kE4m3Max);
  return s >= 1.17549435e-38f ? s : 1.0f;
}
__device__ __forceinline__ float e4m3_factor(float most) {
  return most * (1.0f / kE4m3Max) >= 1.17549435e-38f ? __fdividef(kE4m3Max, most) : 1.0f;
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

// FAST: every row of every tensor starts on a 16-byte boundary (8-byte for the e4m3 output of a
// 16-bit type) and n is a multiple of the vector: a thread's E columns are neighbours.  Otherwise a
// warp's 32 * E columns are the same but a thread's lie 32 apart, so that every access of a warp is
// one run of elements whatever the row's alignment (8191 x 4097 fp16: 162 us with E neighbours read
// one by one and as many stores of a byte or two, 160 like this: the count of accesses is what is left).
template <typename T, bool E4M3, int ITEMS, bool FAST, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS) rms_kernel(const RmsParams p) {
  constexpr int E = Elem<T>::kPerVec;
  __shared__ float slots[2][32];
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
  const T* x = static_cast<const T*>(p.x) + row * p.stride_x;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.stride_residual : nullptr;
  const T* w = static_cast<const T*>(p.w);
  const int col0 = FAST ? lane * E : (lane >> 5) * 32 * E + (lane & 31), col_step = p.threads * E;
  auto column = [&](int i, int j) { return col0 + i * col_step + (FAST ? j : 32 * j); };

  // this thread's part of a row; columns past n are 0
  auto read = [&](const T* from, bool once, Vec<T> (&to)[ITEMS]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if constexpr (FAST) {
        to[i].raw = make_uint4(0, 0, 0, 0);
        if (column(i, 0) < n)
          to[i].raw = once ? ld_once(from + column(i, 0)) : __ldg(reinterpret_cast<const uint4*>(from + column(i, 0)));
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          to[i].e[j] = column(i, j) < n ? from[column(i, j)] : Elem<T>::from_f32(0.0f);
      }
    }
  };
  auto write = [&](T* to, const float (&from)[ITEMS * E]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if constexpr (FAST) {
        if (column(i, 0) < n) st_once(to + column(i, 0), round_elems<T>(&from[i * E]).raw);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (column(i, j) < n) to[column(i, j)] = Elem<T>::from_f32(from[i * E + j]);
      }
    }
  };

  Vec<T> xv[ITEMS], rv[ITEMS];
  read(x, true, xv);
  if (res) read(res, true, rv);
  float v[ITEMS * E];
#pragma unroll
  for (int k = 0; k < ITEMS * E; ++k) v[k] = Elem<T>::to_f32(xv[k / E].e[k % E]);
  if (res) {
#pragma unroll
    for (int k = 0; k < ITEMS * E; ++k) v[k] += Elem<T>::to_f32(rv[k / E].e[k % E]);
  }
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < ITEMS * E; ++k) sum = fmaf(v[k], v[k], sum);
  if (p.residual_out) write(static_cast<T*>(p.residual_out) + row * p.stride_residual_out, v);
  sum = reduce_row<Add>(sum, slots[0], warps);
  const float rstd = rsqrtf(sum / (float)n + p.eps);
  read(w, false, xv);
#pragma unroll
  for (int k = 0; k < ITEMS * E; ++k) v[k] = v[k] * rstd * Elem<T>::to_f32(xv[k / E].e[k % E]);

  if constexpr (!E4M3) {
    write(static_cast<T*>(p.out) + row * p.stride_out, v);
  } else {
    float amax[ITEMS][FAST ? 1 : E];      // of a thread's columns: one scale for all of them, or for each
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      amax[i][0] = 0.0f;
#pragma unroll
      for (int j = 0; j < E; ++j) amax[i][0] = fmaxf(amax[i][0], fabsf(v[i * E + j]));
    }
    float* scales = p.scales + row * p.stride_scales;
    if (p.group_shift == 0) {
      float most = amax[0][0];
#pragma unroll
      for (int i = 1; i < ITEMS; ++i) most = fmaxf(most, amax[i][0]);
      most = reduce_row<Max>(most, slots[1], warps);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < (FAST ? 1 : E); ++j) amax[i][j] = most;
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
      if constexpr (FAST) {
        if (column(i, 0) < n) store_e4m3<E>(out + column(i, 0), &v[i * E], e4m3_factor(amax[i][0]));
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (column(i, j) < n) out[column(i, j)] = (uint8_t)e4m3x2(v[i * E + j] * e4m3_factor(amax[i][j]), 0.0f);
      }
    }
  }
}

template <typename T, bool E4M3, int ITEMS>
int launch_rms(const RmsParams& p, bool fast, cudaStream_t stream) {
  const int threads = p.threads == 32 ? 256 : p.threads;
  const int64_t grid = cdiv64(p.rows, threads / p.threads);
  auto go = [&](auto kern) {
    kern<<<(int)grid, threads, 0, stream>>>(p);
    return cuda_check(cudaGetLastError(), "rmsnorm launch");
  };
  // up to 256 threads a CTA may have 255 registers a thread, 1024 have 64
  if (threads <= 256)
    return fast ? go(rms_kernel<T, E4M3, ITEMS, true, 256>) : go(rms_kernel<T, E4M3, ITEMS, false, 256>);
  return fast ? go(rms_kernel<T, E4M3, ITEMS, true, 1024>) : go(rms_kernel<T, E4M3, ITEMS, false, 1024>);
}

template <typename T, bool E4M3>
int dispatch_rms(RmsParams p, cudaStream_t stream) {
  constexpr int E = Elem<T>::kPerVec;
  bool fast = p.n % E == 0 && at16(p.x) && at16(p.w) && p.stride_x % E == 0;
  if (p.residual) fast = fast && at16(p.residual) && p.stride_residual % E == 0;
  if (p.residual_out) fast = fast && at16(p.residual_out) && p.stride_residual_out % E == 0;
  if (E4M3) fast = fast && reinterpret_cast<uintptr_t>(p.out) % E == 0 && p.stride_out % E == 0;
  else fast = fast && at16(p.out) && p.stride_out % E == 0;

  // 32 values per thread are what 1024 threads have registers for
  if (p.n > 1024 * 32)
    return fail(NB200_E_UNSUPPORTED, "rmsnorm: rows of %d elements (at most 32768)", p.n);
  const int64_t vectors = cdiv64(p.n, E);
  int items = 1;
  p.threads = 32;
  // Few rows: as many threads as there are vectors, the row's latency counts (8 rows of 4096 bf16:
  // 2.7 us).  Rows for every SM: four vectors of x and of the residual in flight per thread (8191
  // rows of 4096 fp16: 49.7 us with one, 41.5 with two, 40.2 with four).
  const int most = p.rows >= 2 * device_info().sm_count ? 4 : 1;
  while ((int64_t)p.threads * items < vectors) {
    if (items < most) items *= 2;
    else if (p.threads < 1024) p.threads *= 2;
    else items *= 2;
  }
  switch (items) {
    case 1: return launch_rms<T, E4M3, 1>(p, fast, stream);
    case 2: return launch_rms<T, E4M3, 2>(p, fast, stream);
    case 4: return launch_rms<T, E4M3, 4>(p, fast, stream);
  }
  if constexpr (E == 4) return launch_rms<T, E4M3, 8>(p, fast, stream);
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
  if (rows == 0 || n == 0) return 0;
  if (!x || !w || !out || (e4m3 && !scales)) return fail(NB200_E_INVALID, "rmsnorm: null tensor pointer");
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
