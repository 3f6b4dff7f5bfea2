// Typed loads, stores and conversions shared by the differentiable operators
// (gated_scan.cu, layer_norm.cu, linear_act.cu): vectors of VEC elements of fp32, bf16
// or fp16 that travel as one aligned access of VEC * sizeof(T) bytes.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace vdn {

template <int BYTES> struct RawOf;
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };
template <typename T, int VEC> using Raw = typename RawOf<sizeof(T) * VEC>::type;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Raw<T, VEC>& raw, float (&v)[VEC]) {
  T e[VEC];
  *reinterpret_cast<Raw<T, VEC>*>(e) = raw;
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = to_f32(e[i]);
}

template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> pack(const float (&v)[VEC]) {
  alignas(16) T e[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(v[i]);
  return *reinterpret_cast<Raw<T, VEC>*>(e);
}

template <typename R> __device__ __forceinline__ R raw_zero() { return R{}; }

// Streaming accesses: each element is read once, so it need not stay in L1.
template <typename R> __device__ __forceinline__ R load_once(const void* p) { return __ldcs(static_cast<const R*>(p)); }
template <typename R> __device__ __forceinline__ void store_once(void* p, const R& v) { __stcs(static_cast<R*>(p), v); }

inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Sums `lines` lines of `cols` fp32 partial sums in a fixed order: 32 columns by 8 line
// groups a block.  Columns below `split` go to `a`, the others to `b` (either may be null).
template <typename T>
__global__ void __launch_bounds__(256) lines_kernel(const float* part, int lines, int64_t cols, T* a, int64_t split,
                                                    T* b) {
  __shared__ float sums[8][33];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < cols)
    for (int l = g; l < lines; l += 8) s += part[l * cols + c];
  sums[g][lane] = s;
  __syncthreads();
  if (g == 0 && c < cols) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sums[k][lane];
    if (c < split) {
      if (a) a[c] = from_f32<T>(s);
    } else if (b) {
      b[c - split] = from_f32<T>(s);
    }
  }
}
template <typename T>
inline int add_lines(const float* part, int lines, int64_t cols, T* a, int64_t split, T* b, cudaStream_t stream) {
  lines_kernel<T><<<(unsigned)((cols + 31) / 32), 256, 0, stream>>>(part, lines, cols, a, split, b);
  VDN_LAUNCH_CHECK("line sums");
  return VDN_OK;
}

inline int dtype_bytes(int code) { return code == VDN_DTYPE_F32 ? 4 : 2; }
inline bool dtype_known(int code) { return code == VDN_DTYPE_F32 || code == VDN_DTYPE_BF16 || code == VDN_DTYPE_F16; }

}  // namespace vdn
