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

// A 32-bit word of two 16-bit values (the lower in the low half), and back with one conversion.
template <typename T> __device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi);
template <> __device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t w, float& lo, float& hi) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xFFFF0000u);
}
template <> __device__ __forceinline__ void unpack2<__half>(uint32_t w, float& lo, float& hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  lo = f.x;
  hi = f.y;
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void words(uint32_t r, uint32_t (&w)[1]) { w[0] = r; }
__device__ __forceinline__ void words(const uint2& r, uint32_t (&w)[2]) { w[0] = r.x; w[1] = r.y; }
__device__ __forceinline__ void words(const uint4& r, uint32_t (&w)[4]) { w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w; }
__device__ __forceinline__ uint32_t join(const uint32_t (&w)[1]) { return w[0]; }
__device__ __forceinline__ uint2 join(const uint32_t (&w)[2]) { return make_uint2(w[0], w[1]); }
__device__ __forceinline__ uint4 join(const uint32_t (&w)[4]) { return make_uint4(w[0], w[1], w[2], w[3]); }

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Raw<T, VEC>& raw, float (&v)[VEC]) {
  if constexpr (VEC == 1 && sizeof(T) == 2) {
    T e;
    *reinterpret_cast<uint16_t*>(&e) = raw;
    v[0] = to_f32(e);
  } else {
    uint32_t w[VEC * sizeof(T) / 4];
    words(raw, w);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> pack(const float (&v)[VEC]) {
  if constexpr (VEC == 1 && sizeof(T) == 2) {
    const T e = from_f32<T>(v[0]);
    return *reinterpret_cast<const uint16_t*>(&e);
  } else {
    uint32_t w[VEC * sizeof(T) / 4];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
    return join(w);
  }
}

// Arithmetic on one value (float) or two (f2, packed fp32 pairs: one instruction for both).
__device__ __forceinline__ float vset(float, float c) { return c; }
__device__ __forceinline__ f2 vset(f2, float c) { return f2_pack(c, c); }
__device__ __forceinline__ float vadd(float a, float b) { return a + b; }
__device__ __forceinline__ f2 vadd(f2 a, f2 b) { return f2_add(a, b); }
__device__ __forceinline__ float vmul(float a, float b) { return a * b; }
__device__ __forceinline__ f2 vmul(f2 a, f2 b) { return f2_mul(a, b); }
__device__ __forceinline__ float vfma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ f2 vfma(f2 a, f2 b, f2 c) { return f2_fma(a, b, c); }
template <int VEC> struct Lanes { using V = f2; static constexpr int N = VEC / 2; };
template <> struct Lanes<1> { using V = float; static constexpr int N = 1; };

__device__ __forceinline__ void spread(float a, float& v) { v = a; }
__device__ __forceinline__ void spread(float a, f2& v) { v = f2_pack(a, a); }
__device__ __forceinline__ void spread(f2 a, f2& v) { v = a; }

__device__ __forceinline__ void to_lanes(const float (&e)[1], float (&v)[1]) { v[0] = e[0]; }
template <int VEC> __device__ __forceinline__ void to_lanes(const float (&e)[VEC], f2 (&v)[VEC / 2]) {
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) v[i] = f2_pack(e[2 * i], e[2 * i + 1]);
}
__device__ __forceinline__ void from_lanes(const float (&v)[1], float (&e)[1]) { e[0] = v[0]; }
template <int VEC> __device__ __forceinline__ void from_lanes(const f2 (&v)[VEC / 2], float (&e)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) f2_unpack(v[i], e[2 * i], e[2 * i + 1]);
}
template <typename T, int VEC, typename V, int N>
__device__ __forceinline__ void unpack_lanes(const Raw<T, VEC>& raw, V (&v)[N]) {
  float e[VEC];
  unpack<T, VEC>(raw, e);
  to_lanes(e, v);
}
template <typename T, int VEC, typename V, int N>
__device__ __forceinline__ Raw<T, VEC> pack_lanes(const V (&v)[N]) {
  float e[VEC];
  from_lanes(v, e);
  return pack<T, VEC>(e);
}

template <typename R> __device__ __forceinline__ R raw_zero() { return R{}; }

// Streaming accesses: each element is read once, so it need not stay in L1.
template <typename R> __device__ __forceinline__ R load_once(const void* p) { return __ldcs(static_cast<const R*>(p)); }
template <typename R> __device__ __forceinline__ void store_once(void* p, const R& v) { __stcs(static_cast<R*>(p), v); }

inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Sums `lines` lines of `cols` fp32 partial sums in a fixed order: 8 columns (a 32-byte sector a
// line) by 128 line groups a block, so that few columns still have many loads in flight.
// Columns below `split` go to `a`, the others to `b` (either may be null).
template <typename T>
__global__ void __launch_bounds__(1024) lines_kernel(const float* part, int lines, int64_t cols, T* a, int64_t split,
                                                     T* b) {
  __shared__ float sums[8][129];
  const int col = threadIdx.x & 7, group = threadIdx.x >> 3;
  const int64_t c = (int64_t)blockIdx.x * 8 + col;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int l = group; l < lines; l += 128) s += part[l * cols + c];
  }
  sums[col][group] = s;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;   // a warp per column
  if (warp >= 8) return;
  s = sums[warp][lane];
#pragma unroll
  for (int k = 32; k < 128; k += 32) s += sums[warp][lane + k];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int64_t at = (int64_t)blockIdx.x * 8 + warp;
  if (lane == 0 && at < cols) {
    if (at < split) {
      if (a) a[at] = from_f32<T>(s);
    } else if (b) {
      b[at - split] = from_f32<T>(s);
    }
  }
}
template <typename T>
inline int add_lines(const float* part, int lines, int64_t cols, T* a, int64_t split, T* b, cudaStream_t stream) {
  lines_kernel<T><<<(unsigned)((cols + 7) / 8), 1024, 0, stream>>>(part, lines, cols, a, split, b);
  VDN_LAUNCH_CHECK("line sums");
  return VDN_OK;
}

inline int dtype_bytes(int code) { return code == VDN_DTYPE_F32 ? 4 : 2; }
inline bool dtype_known(int code) { return code == VDN_DTYPE_F32 || code == VDN_DTYPE_BF16 || code == VDN_DTYPE_F16; }

}  // namespace vdn
