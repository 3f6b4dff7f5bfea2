// Layer norm over the last dimension, forward and backward, sm_100a.
//
//   forward   y = (x - mean) rstd w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   backward  xh = (x - mean) rstd,  t = w dy
//             dx = rstd (t - mean(t) - xh mean(t xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// HBM is the bound: the forward moves two elements per value, the backward three.  A row is
// read once and stays in registers between its statistics and its result: a group of 8,
// 16 or 32 lanes per short row, a CTA per long one, in 16-byte vectors; rows whose width, stride
// or address does not allow those take one element per lane.  The variance is the mean
// square of the centred values (a second pass over registers), all sums in fp32.
//
// The backward's CTAs each walk a fixed set of rows (blockIdx.x, + gridDim.x, ...) with the next
// row's loads issued ahead, and keep their columns' dw and db in fp32 registers over all of
// them; one line of partial sums per CTA goes to the caller's workspace, and a second
// kernel adds the lines in a fixed order.  No atomics: the same bits on every run.
// Widths that fit no register form take `wide` kernels, which read a row again for each pass.
#include "train_common.cuh"

namespace vdn {
namespace lnorm {

struct Fwd {
  const void* x;
  const void* w;
  const void* b;
  void* y;
  float *mean, *rstd;   // optional
  int64_t rows, x_ld, y_ld;
  int width;
  float eps;
};

struct Bwd {
  const void* dy;
  const void* x;
  const void* w;
  const float *mean, *rstd;
  void* dx;
  float* part;          // [gridDim.x, 2, width]
  int64_t rows, dy_ld, x_ld, dx_ld;
  int width;
};

// Sum over the `lanes` threads of a row: a lane group, or the whole block (0).
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
  if constexpr (LANES > 0) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  } else {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < warps; ++w) v += scratch[w];
    return v;             // the caller alternates scratch halves, so no barrier after the reads
  }
}

template <typename TW, int VEC>
__device__ __forceinline__ void load_weight(const void* w, int col, float fill, float (&v)[VEC]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = fill;
    return;
  }
  constexpr int STEP = sizeof(TW) * VEC > 16 ? 16 / sizeof(TW) : VEC;
#pragma unroll
  for (int i = 0; i < VEC; i += STEP) {
    float part[STEP];
    unpack<TW, STEP>(*reinterpret_cast<const Raw<TW, STEP>*>(static_cast<const TW*>(w) + col + i), part);
#pragma unroll
    for (int j = 0; j < STEP; ++j) v[i + j] = part[j];
  }
}

template <typename T, typename TW, int VEC, int NV, int LANES, int MAXT>
__global__ void __launch_bounds__(MAXT) forward_kernel(const Fwd p) {
  using R = Raw<T, VEC>;
  __shared__ float scratch[2][32];
  const int lanes = LANES ? LANES : blockDim.x;
  const int t = LANES ? threadIdx.x % (LANES ? LANES : 1) : threadIdx.x;
  const int64_t row = LANES ? (int64_t)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes : blockIdx.x;
  const bool on = row < p.rows;                      // uniform over the row's lanes
  const T* x = static_cast<const T*>(p.x) + (on ? row : 0) * p.x_ld;
  R raw[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int col = (t + k * lanes) * VEC;
    raw[k] = on && col < p.width ? load_once<R>(x + col) : raw_zero<R>();
  }
  float v[NV][VEC], sum = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    unpack<T, VEC>(raw[k], v[k]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += v[k][i];
  }
  const float inv = 1.0f / (float)p.width;
  const float mean = row_sum<LANES>(sum, scratch[0]) * inv;
  float sq = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const bool in = (t + k * lanes) * VEC < p.width;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[k][i] -= mean;
      if (in) sq = fmaf(v[k][i], v[k][i], sq);
    }
  }
  const float rstd = rsqrtf(row_sum<LANES>(sq, scratch[1]) * inv + p.eps);
  if (!on) return;
  if (t == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(p.y) + row * p.y_ld;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int col = (t + k * lanes) * VEC;
    if (col >= p.width) continue;
    float w[VEC], b[VEC];
    load_weight<TW, VEC>(p.w, col, 1.f, w);
    load_weight<TW, VEC>(p.b, col, 0.f, b);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[k][i] = fmaf(v[k][i] * rstd, w[i], b[i]);
    store_once(y + col, pack<T, VEC>(v[k]));
  }
}

// Any width: a CTA per row that reads its row three times (from L2 after the first).
template <typename T, typename TW>
__global__ void __launch_bounds__(1024) forward_wide_kernel(const Fwd p) {
  __shared__ float scratch[2][32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  float sum = 0.f, sq = 0.f;
  for (int c = threadIdx.x; c < p.width; c += blockDim.x) sum += to_f32(x[c]);
  const float inv = 1.0f / (float)p.width;
  const float mean = row_sum<0>(sum, scratch[0]) * inv;
  for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
    const float d = to_f32(x[c]) - mean;
    sq = fmaf(d, d, sq);
  }
  const float rstd = rsqrtf(row_sum<0>(sq, scratch[1]) * inv + p.eps);
  if (threadIdx.x == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(p.y) + row * p.y_ld;
  for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
    const float w = p.w ? to_f32(static_cast<const TW*>(p.w)[c]) : 1.f;
    const float b = p.b ? to_f32(static_cast<const TW*>(p.b)[c]) : 0.f;
    y[c] = from_f32<T>(fmaf((to_f32(x[c]) - mean) * rstd, w, b));
  }
}

template <typename T, typename TW, int VEC, int NV, int LANES, int MAXT, int PER_SM>
__global__ void __launch_bounds__(MAXT, PER_SM) backward_kernel(const Bwd p) {
  using R = Raw<T, VEC>;
  __shared__ float scratch[2][2][32];
  const int lanes = LANES ? LANES : blockDim.x;
  const int t = LANES ? threadIdx.x % (LANES ? LANES : 1) : threadIdx.x;
  const int groups = LANES ? blockDim.x / lanes : 1;       // rows a CTA walks side by side
  const int group = LANES ? threadIdx.x / lanes : 0;
  const float inv = 1.0f / (float)p.width;
  float dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k][i] = db[k][i] = 0.f;

  R rx[NV], rd[NV];
  float mean = 0.f, rstd = 0.f;
  auto load = [&](int64_t row) {
    const bool on = row < p.rows;
    const T* x = static_cast<const T*>(p.x) + (on ? row : 0) * p.x_ld;
    const T* d = static_cast<const T*>(p.dy) + (on ? row : 0) * p.dy_ld;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (t + k * lanes) * VEC;
      const bool in = on && col < p.width;
      rx[k] = in ? load_once<R>(x + col) : raw_zero<R>();
      rd[k] = in ? load_once<R>(d + col) : raw_zero<R>();
    }
    mean = on ? p.mean[row] : 0.f;
    rstd = on ? p.rstd[row] : 0.f;
  };
  // Every group takes the same number of turns, so the block's barriers match.
  const int64_t stride = (int64_t)gridDim.x * groups;
  int64_t row = (int64_t)blockIdx.x * groups + group;
  load(row);
  int half = 0;
  for (int64_t base = (int64_t)blockIdx.x * groups; base < p.rows; base += stride, row += stride, half ^= 1) {
    R cx[NV], cd[NV];
    const float m = mean, r = rstd;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      cx[k] = rx[k];
      cd[k] = rd[k];
    }
    load(row + stride);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (t + k * lanes) * VEC;
      if (col >= p.width) continue;
      float x[VEC], d[VEC], w[VEC];
      unpack<T, VEC>(cx[k], x);
      unpack<T, VEC>(cd[k], d);
      load_weight<TW, VEC>(p.w, col, 1.f, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float xh = (x[i] - m) * r, td = w[i] * d[i];
        s1 += td;
        s2 = fmaf(td, xh, s2);
        dw[k][i] = fmaf(d[i], xh, dw[k][i]);
        db[k][i] += d[i];
      }
    }
    if constexpr (LANES > 0) {
      s1 = row_sum<LANES>(s1, nullptr);
      s2 = row_sum<LANES>(s2, nullptr);
    } else {              // both sums behind one barrier
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        s1 += __shfl_xor_sync(0xffffffffu, s1, o);
        s2 += __shfl_xor_sync(0xffffffffu, s2, o);
      }
      if ((threadIdx.x & 31) == 0) {
        scratch[half][0][threadIdx.x >> 5] = s1;
        scratch[half][1][threadIdx.x >> 5] = s2;
      }
      __syncthreads();
      s1 = s2 = 0.f;
      const int warps = blockDim.x >> 5;
      for (int w = 0; w < warps; ++w) {
        s1 += scratch[half][0][w];
        s2 += scratch[half][1][w];
      }
    }
    if (row >= p.rows) continue;
    s1 *= inv;
    s2 *= inv;
    T* dx = static_cast<T*>(p.dx) + row * p.dx_ld;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (t + k * lanes) * VEC;
      if (col >= p.width) continue;
      float x[VEC], d[VEC], w[VEC];
      unpack<T, VEC>(cx[k], x);
      unpack<T, VEC>(cd[k], d);
      load_weight<TW, VEC>(p.w, col, 1.f, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float xh = (x[i] - m) * r;
        x[i] = r * (fmaf(w[i], d[i], -s1) - xh * s2);
      }
      store_once(dx + col, pack<T, VEC>(x));
    }
  }

  float* part = p.part + (int64_t)blockIdx.x * 2 * p.width;
  if constexpr (LANES == 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (t + k * lanes) * VEC;
      if (col >= p.width) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        part[col + i] = dw[k][i];
        part[p.width + col + i] = db[k][i];
      }
    }
  } else {                // join the lane groups: column by column, groups in order
    extern __shared__ float lines[];                 // [groups][width]
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (t + k * lanes) * VEC;
        if (col >= p.width) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) lines[group * p.width + col + i] = which ? db[k][i] : dw[k][i];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
        float s = 0.f;
        for (int g = 0; g < groups; ++g) s += lines[g * p.width + c];
        part[which * p.width + c] = s;
      }
    }
  }
}

// Any width: dx by a CTA per row, and the column sums by a CTA per 256 columns and row chunk.
template <typename T, typename TW>
__global__ void __launch_bounds__(1024) backward_wide_kernel(const Bwd p) {
  __shared__ float scratch[2][32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* d = static_cast<const T*>(p.dy) + row * p.dy_ld;
  const TW* w = static_cast<const TW*>(p.w);
  const float m = p.mean[row], r = p.rstd[row], inv = 1.0f / (float)p.width;
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
    const float td = (w ? to_f32(w[c]) : 1.f) * to_f32(d[c]);
    s1 += td;
    s2 = fmaf(td, (to_f32(x[c]) - m) * r, s2);
  }
  s1 = row_sum<0>(s1, scratch[0]) * inv;
  s2 = row_sum<0>(s2, scratch[1]) * inv;
  T* dx = static_cast<T*>(p.dx) + row * p.dx_ld;
  for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
    const float xh = (to_f32(x[c]) - m) * r;
    dx[c] = from_f32<T>(r * (fmaf(w ? to_f32(w[c]) : 1.f, to_f32(d[c]), -s1) - xh * s2));
  }
}

template <typename T>
__global__ void __launch_bounds__(256) columns_wide_kernel(const Bwd p) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.width) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float d = to_f32(static_cast<const T*>(p.dy)[row * p.dy_ld + c]);
    const float x = to_f32(static_cast<const T*>(p.x)[row * p.x_ld + c]);
    dw = fmaf(d, (x - p.mean[row]) * p.rstd[row], dw);
    db += d;
  }
  float* part = p.part + (int64_t)blockIdx.y * 2 * p.width;
  part[c] = dw;
  part[p.width + c] = db;
}

template <typename T, typename TW, int VEC, int NV, int LANES, int MAXT>
static int launch_forward(const Fwd& p, int block, cudaStream_t stream) {
  const int64_t per = LANES ? block / (LANES ? LANES : 1) : 1;
  forward_kernel<T, TW, VEC, NV, LANES, MAXT><<<(unsigned)((p.rows + per - 1) / per), block, 0, stream>>>(p);
  VDN_LAUNCH_CHECK("layer norm");
  return VDN_OK;
}

template <typename T, typename TW>
static int forward(const Fwd& p, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const size_t wv = sizeof(TW) * V > 16 ? 16 : sizeof(TW) * V;
  const bool vec = p.width % V == 0 && p.x_ld % V == 0 && p.y_ld % V == 0 && aligned16(p.x) && aligned16(p.y) &&
                   (!p.w || aligned_to(p.w, wv)) && (!p.b || aligned_to(p.b, wv));
  if (vec) {
    const int n = p.width / V;
    if (n <= 8) return launch_forward<T, TW, V, 1, 8, 256>(p, 256, stream);
    if (n <= 16) return launch_forward<T, TW, V, 1, 16, 256>(p, 256, stream);
    if (n <= 32) return launch_forward<T, TW, V, 1, 32, 256>(p, 256, stream);
    if (n <= 64) return launch_forward<T, TW, V, 2, 32, 256>(p, 256, stream);
    if (n <= 128) return launch_forward<T, TW, V, 4, 32, 256>(p, 256, stream);
    if (n <= 2 * 512) return launch_forward<T, TW, V, 2, 0, 512>(p, (n + 63) / 64 * 32, stream);
    if (n <= 4 * 1024) return launch_forward<T, TW, V, 4, 0, 1024>(p, (n + 127) / 128 * 32, stream);
  } else {
    if (p.width <= 128) return launch_forward<T, TW, 1, 4, 32, 256>(p, 256, stream);
    if (p.width <= 8 * 512) return launch_forward<T, TW, 1, 8, 0, 512>(p, (p.width + 255) / 256 * 32, stream);
    if (p.width <= 16 * 1024) return launch_forward<T, TW, 1, 16, 0, 1024>(p, (p.width + 511) / 512 * 32, stream);
  }
  forward_wide_kernel<T, TW><<<(unsigned)p.rows, 1024, 0, stream>>>(p);
  VDN_LAUNCH_CHECK("layer norm (wide)");
  return VDN_OK;
}

// CTAs of the backward, one line of partial sums each: enough to fill 148 SMs a few times
// over for short rows; the count depends on the shape alone, so results do not vary.
constexpr int kLines = 296;

template <typename T, typename TW, int VEC, int NV, int LANES, int MAXT, int PER_SM>
static int launch_backward(const Bwd& p, int block, int lines, cudaStream_t stream) {
  const size_t smem = LANES ? sizeof(float) * (block / (LANES ? LANES : 1)) * (size_t)p.width : 0;
  backward_kernel<T, TW, VEC, NV, LANES, MAXT, PER_SM><<<lines, block, smem, stream>>>(p);
  VDN_LAUNCH_CHECK("layer norm backward");
  return VDN_OK;
}

template <typename T, typename TW>
static int backward(const Bwd& p, int lines, void* dw, void* db, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T), M = sizeof(T) / 2;   // M: fp32 holds half the values per vector
  const size_t wv = sizeof(TW) * V > 16 ? 16 : sizeof(TW) * V;
  const bool vec = p.width % V == 0 && p.x_ld % V == 0 && p.dy_ld % V == 0 && p.dx_ld % V == 0 && aligned16(p.x) &&
                   aligned16(p.dy) && aligned16(p.dx) && (!p.w || aligned_to(p.w, wv));
  const int n = p.width / V;
  int rc = -1;
  if (vec) {
    if (n <= 8) rc = launch_backward<T, TW, V, 1, 8, 256, 2>(p, 256, lines, stream);
    else if (n <= 16) rc = launch_backward<T, TW, V, 1, 16, 256, 2>(p, 256, lines, stream);
    else if (n <= 32) rc = launch_backward<T, TW, V, 1, 32, 256, 2>(p, 256, lines, stream);
    else if (n <= 64) rc = launch_backward<T, TW, V, 2, 32, 128, 4>(p, 128, lines, stream);
    else if (n <= 2 * M * 384) rc = launch_backward<T, TW, V, 2 * M, 0, 384, 2>(p, (n + 64 * M - 1) / (64 * M) * 32, lines, stream);
    else if (n <= 4 * M * 512) rc = launch_backward<T, TW, V, 4 * M, 0, 512, 1>(p, (n + 128 * M - 1) / (128 * M) * 32, lines, stream);
  } else {
    if (p.width <= 128) rc = launch_backward<T, TW, 1, 4, 32, 128, 4>(p, 128, lines, stream);
    else if (p.width <= 16 * 512) rc = launch_backward<T, TW, 1, 16, 0, 512, 1>(p, (p.width + 511) / 512 * 32, lines, stream);
  }
  if (rc > 0) return rc;
  if (rc < 0) {
    backward_wide_kernel<T, TW><<<(unsigned)p.rows, 1024, 0, stream>>>(p);
    VDN_LAUNCH_CHECK("layer norm backward (wide)");
    columns_wide_kernel<T><<<dim3((p.width + 255) / 256, lines), 256, 0, stream>>>(p);
    VDN_LAUNCH_CHECK("layer norm backward (wide columns)");
  }
  if (!dw && !db) return VDN_OK;
  return add_lines<TW>(p.part, lines, 2 * (int64_t)p.width, static_cast<TW*>(dw), p.width, static_cast<TW*>(db), stream);
}

static int check(int dtype, int w_dtype, int64_t rows, int64_t width) {
  if (!dtype_known(dtype) || !dtype_known(w_dtype)) return set_error(VDN_ERR_TYPE, "unknown dtype code");
  if (w_dtype != dtype && w_dtype != VDN_DTYPE_F32)
    return set_error(VDN_ERR_TYPE, "the weight must have x's dtype or be fp32");
  VDN_CHECK_ARG(rows >= 0 && rows < (1ll << 31) && width >= 1 && width < (1ll << 30), "bad layer norm extents");
  return VDN_OK;
}

#define VDN_LN_DISPATCH(fn, ...)                                                               \
  if (dtype == VDN_DTYPE_F32) return fn<float, float>(__VA_ARGS__);                            \
  if (dtype == VDN_DTYPE_BF16)                                                                 \
    return w_dtype == VDN_DTYPE_F32 ? fn<__nv_bfloat16, float>(__VA_ARGS__)                    \
                                    : fn<__nv_bfloat16, __nv_bfloat16>(__VA_ARGS__);           \
  return w_dtype == VDN_DTYPE_F32 ? fn<__half, float>(__VA_ARGS__) : fn<__half, __half>(__VA_ARGS__);

}  // namespace lnorm
}  // namespace vdn

using namespace vdn;

extern "C" int vdn_layer_norm(const void* x, int dtype, int64_t rows, int64_t width, int64_t x_stride,
                              const void* weight, const void* bias, int w_dtype, float eps, void* y,
                              int64_t y_stride, float* mean, float* rstd, cudaStream_t stream) {
  using namespace vdn::lnorm;
  if (int rc = check(dtype, w_dtype, rows, width)) return rc;
  if (rows == 0) return VDN_OK;
  VDN_CHECK_ARG(x && y, "null pointer");
  VDN_CHECK_ARG(rows == 1 || (x_stride >= 0 && y_stride >= width), "bad row stride");
  const Fwd p = {x, weight, bias, y, mean, rstd, rows, x_stride, y_stride, (int)width, eps};
  VDN_LN_DISPATCH(forward, p, stream)
}

extern "C" size_t vdn_layer_norm_backward_workspace_size(int64_t rows, int64_t width) {
  if (rows < 1 || width < 1) return 0;
  const int64_t lines = rows < vdn::lnorm::kLines ? rows : vdn::lnorm::kLines;
  return sizeof(float) * 2 * (size_t)lines * (size_t)width;
}

extern "C" int vdn_layer_norm_backward(const void* dy, int dtype, int64_t rows, int64_t width, int64_t dy_stride,
                                       const void* x, int64_t x_stride, const void* weight, int w_dtype,
                                       const float* mean, const float* rstd, void* dx, int64_t dx_stride,
                                       void* d_weight, void* d_bias, void* workspace, size_t workspace_bytes,
                                       cudaStream_t stream) {
  using namespace vdn::lnorm;
  if (int rc = check(dtype, w_dtype, rows, width)) return rc;
  if (rows == 0) {
    const size_t bytes = (size_t)width * dtype_bytes(w_dtype);
    if (d_weight) VDN_CUDA_TRY(cudaMemsetAsync(d_weight, 0, bytes, stream));
    if (d_bias) VDN_CUDA_TRY(cudaMemsetAsync(d_bias, 0, bytes, stream));
    return VDN_OK;
  }
  VDN_CHECK_ARG(dy && x && mean && rstd && dx && workspace, "null pointer");
  VDN_CHECK_ARG(rows == 1 || (dy_stride >= 0 && x_stride >= 0 && dx_stride >= width), "bad row stride");
  VDN_CHECK_ARG(workspace_bytes >= vdn_layer_norm_backward_workspace_size(rows, width),
                "workspace smaller than vdn_layer_norm_backward_workspace_size");
  const int lines = (int)(rows < kLines ? rows : kLines);
  const Bwd p = {dy, x, weight, mean, rstd, dx, static_cast<float*>(workspace), rows, dy_stride, x_stride, dx_stride,
                 (int)width};
  VDN_LN_DISPATCH(backward, p, lines, d_weight, d_bias, stream)
}
