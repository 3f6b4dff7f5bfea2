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
// Bound by HBM: 32760 x 5120 in bf16 forward 124 us (5.4 TB/s, a copy reaches 6.5), backward 204
// (4.9 TB/s, some 10 us of it the sum of the lines).
#include <initializer_list>

#include "train_common.cuh"
#include "sm100.cuh"

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
  int* status;
};

// The sums of N values over a row's threads: a lane group, or the whole block (LANES = 0: one
// barrier; callers alternate between two `scratch` areas, so none is needed after the reads).
template <int LANES, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*scratch)[32]) {
#pragma unroll
  for (int o = (LANES ? LANES : 32) / 2; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (LANES == 0) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane < N) {
      float mine = v[0];
#pragma unroll
      for (int i = 1; i < N; ++i) mine = lane == i ? v[i] : mine;
      scratch[lane][threadIdx.x >> 5] = mine;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lane < warps ? scratch[i][lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float (*scratch)[32]) {
  float one[1] = {v};
  row_sums<LANES>(one, scratch);
  return one[0];
}
__device__ __forceinline__ float hsum(float v) { return v; }
__device__ __forceinline__ float hsum(f2 v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

// VEC weights (or biases) as they lie in memory, in 16-byte pieces or one smaller one.
template <typename TW, int VEC>
struct Weights {
  static constexpr int STEP = sizeof(TW) * VEC > 16 ? 16 / (int)sizeof(TW) : VEC, N = VEC / STEP;
  Raw<TW, STEP> raw[N];
  __device__ __forceinline__ void load(const void* w, int col) {
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = *reinterpret_cast<const Raw<TW, STEP>*>(static_cast<const TW*>(w) + col + i * STEP);
  }
  template <typename V, int M>
  __device__ __forceinline__ void get(V (&v)[M]) const {
    float e[VEC];
    values(e);
    to_lanes(e, v);
  }
  __device__ __forceinline__ void values(float (&v)[VEC]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float part[STEP];
      unpack<TW, STEP>(raw[i], part);
#pragma unroll
      for (int j = 0; j < STEP; ++j) v[i * STEP + j] = part[j];
    }
  }
};

// Short rows, one vector a lane: a group of LANES lanes walks rows (its CTA's blockIdx.x, + gridDim.x, ..) with the
// next row's load in flight and its columns' weights in registers.
template <typename T, typename TW, int VEC, int LANES>
__global__ void __launch_bounds__(256, 5) forward_kernel(const Fwd p) {
  using R = Raw<T, VEC>;
  using V = typename Lanes<VEC>::V;
  constexpr int NP = Lanes<VEC>::N, GROUPS = 256 / LANES;   // rows a CTA walks side by side
  const int64_t stride = (int64_t)gridDim.x * GROUPS;
  const float inv = 1.0f / (float)p.width;
  const int col = threadIdx.x % LANES * VEC;
  const bool in = col < p.width;
  Weights<TW, VEC> w, b;
  if (in && p.w) w.load(p.w, col);
  if (in && p.b) b.load(p.b, col);
  auto load = [&](int64_t row) {
    return in && row < p.rows ? load_once<R>(static_cast<const T*>(p.x) + row * p.x_ld + col) : raw_zero<R>();
  };
  int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES;
  R raw = load(row);
  // Every group takes the same number of turns, so a warp's shuffles match.
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < p.rows; base += stride, row += stride) {
    V v[NP], acc = vset(V{}, 0.f);
    unpack_lanes<T, VEC>(raw, v);
#pragma unroll
    for (int i = 0; i < NP; ++i) acc = vadd(acc, v[i]);
    raw = load(row + stride);
    const float mean = row_sum<LANES>(hsum(acc), nullptr) * inv;
    const V minus = vset(V{}, -mean);
    acc = vset(V{}, 0.f);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      v[i] = vadd(v[i], minus);
      if (in) acc = vfma(v[i], v[i], acc);
    }
    const float rstd = rsqrtf(row_sum<LANES>(hsum(acc), nullptr) * inv + p.eps);
    if (row >= p.rows || !in) continue;
    if (col == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
    const V scale = vset(V{}, rstd);
    V f[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) v[i] = vmul(v[i], scale);
    if (p.w) {
      w.get(f);
#pragma unroll
      for (int i = 0; i < NP; ++i) v[i] = vmul(v[i], f[i]);
    }
    if (p.b) {
      b.get(f);
#pragma unroll
      for (int i = 0; i < NP; ++i) v[i] = vadd(v[i], f[i]);
    }
    store_once(static_cast<T*>(p.y) + row * p.y_ld + col, pack_lanes<T, VEC>(v));
  }
}

// Longer rows: a warp per row (LANES = 32), or a CTA of a few warps (0), that holds its row as it
// lies in memory, up to NV vectors a lane, and unpacks it for each of the three passes.  With
// a whole row per warp the sums cost ten shuffles for up to 160 values a lane and there
// are no barriers (5120 columns: 23 instructions a value with a CTA per row, about 8 here).
// ROWS rows at a time share the weights' loads (which cost more than a 16-bit row's own, from L1)
// and the barriers.
template <typename T, typename TW, int VEC, int NV, int ROWS, int LANES, int MAXT, int PER_SM>
__global__ void __launch_bounds__(MAXT, PER_SM) forward_row_kernel(const Fwd p) {
  using R = Raw<T, VEC>;
  using V = typename Lanes<VEC>::V;
  constexpr int NP = Lanes<VEC>::N;
  __shared__ float scratch[2 * ROWS][32];
  const int lanes = LANES ? LANES : blockDim.x;
  const int t = LANES ? threadIdx.x % (LANES ? LANES : 1) : threadIdx.x;
  const int groups = LANES ? blockDim.x / lanes : 1;
  const float inv = 1.0f / (float)p.width;
  const int64_t row = ((int64_t)blockIdx.x * groups + (LANES ? threadIdx.x / lanes : 0)) * ROWS;
  if (LANES && row >= p.rows) return;                // a whole warp
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  R raw[ROWS][NV];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (t + k * lanes) * VEC;
      raw[r][k] = col < p.width && (r == 0 || row + r < p.rows) ? load_once<R>(x + r * p.x_ld + col) : raw_zero<R>();
    }
  float mean[ROWS], rstd[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    V acc = vset(V{}, 0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      V v[NP];
      unpack_lanes<T, VEC>(raw[r][k], v);
#pragma unroll
      for (int i = 0; i < NP; ++i) acc = vadd(acc, v[i]);
    }
    mean[r] = hsum(acc);
  }
  row_sums<LANES>(mean, scratch);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    mean[r] *= inv;
    const V minus = vset(V{}, -mean[r]);
    V acc = vset(V{}, 0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      V v[NP];
      unpack_lanes<T, VEC>(raw[r][k], v);
      if ((t + k * lanes) * VEC < p.width) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const V d = vadd(v[i], minus);
          acc = vfma(d, d, acc);
        }
      }
    }
    rstd[r] = hsum(acc);
  }
  row_sums<LANES>(rstd, scratch + ROWS);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    rstd[r] = rsqrtf(rstd[r] * inv + p.eps);
    if (t == 0 && row + r < p.rows) {
      if (p.mean) p.mean[row + r] = mean[r];
      if (p.rstd) p.rstd[row + r] = rstd[r];
    }
  }
  T* y = static_cast<T*>(p.y) + row * p.y_ld;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int col = (t + k * lanes) * VEC;
    if (col >= p.width) break;
    Weights<TW, VEC> w, b;
    if (p.w) w.load(p.w, col);
    if (p.b) b.load(p.b, col);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (r > 0 && row + r >= p.rows) break;
      const V minus = vset(V{}, -mean[r]), scale = vset(V{}, rstd[r]);
      V v[NP], f[NP];
      unpack_lanes<T, VEC>(raw[r][k], v);
#pragma unroll
      for (int i = 0; i < NP; ++i) v[i] = vmul(vadd(v[i], minus), scale);
      if (p.w) {
        w.get(f);
#pragma unroll
        for (int i = 0; i < NP; ++i) v[i] = vmul(v[i], f[i]);
      }
      if (p.b) {
        b.get(f);
#pragma unroll
        for (int i = 0; i < NP; ++i) v[i] = vadd(v[i], f[i]);
      }
      store_once(y + r * p.y_ld + col, pack_lanes<T, VEC>(v));
    }
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
  const float mean = row_sum<0>(sum, scratch) * inv;
  for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
    const float d = to_f32(x[c]) - mean;
    sq = fmaf(d, d, sq);
  }
  const float rstd = rsqrtf(row_sum<0>(sq, scratch + 1) * inv + p.eps);
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

template <typename T, typename TW, int VEC, int NV, int LANES, int MAXT, int PER_SM, bool HELD>
__global__ void __launch_bounds__(MAXT, PER_SM) backward_kernel(const Bwd p) {
  using R = Raw<T, VEC>;
  __shared__ float scratch[2][2][32];
  const int lanes = LANES ? LANES : blockDim.x;
  const int t = LANES ? threadIdx.x % (LANES ? LANES : 1) : threadIdx.x;
  const int groups = LANES ? blockDim.x / lanes : 1;       // rows a CTA walks side by side
  const int group = LANES ? threadIdx.x / lanes : 0;
  const float inv = 1.0f / (float)p.width;
  using V = typename Lanes<VEC>::V;
  constexpr int NP = Lanes<VEC>::N;
  V dw[NV][NP], db[NV][NP];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < NP; ++i) dw[k][i] = db[k][i] = vset(V{}, 0.f);
  Weights<TW, VEC> held[HELD ? NV : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (p.w && (t + k * lanes) * VEC < p.width) held[k].load(p.w, (t + k * lanes) * VEC);
  }
  auto weights = [&](int k, int col, V (&w)[NP]) {
    if (p.w) {
      if constexpr (!HELD) held[0].load(p.w, col);
      held[HELD ? k : 0].get(w);
    } else {
#pragma unroll
      for (int i = 0; i < NP; ++i) w[i] = vset(V{}, 1.f);
    }
  };

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
    const V minus = vset(V{}, -m), scale = vset(V{}, r);
    V a1 = vset(V{}, 0.f), a2 = vset(V{}, 0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (t + k * lanes) * VEC;
      if (col >= p.width) continue;
      V x[NP], d[NP], w[NP];
      unpack_lanes<T, VEC>(cx[k], x);
      unpack_lanes<T, VEC>(cd[k], d);
      weights(k, col, w);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const V xh = vmul(vadd(x[i], minus), scale), td = vmul(w[i], d[i]);
        a1 = vadd(a1, td);
        a2 = vfma(td, xh, a2);
        dw[k][i] = vfma(d[i], xh, dw[k][i]);
        db[k][i] = vadd(db[k][i], d[i]);
      }
    }
    float s[2] = {hsum(a1), hsum(a2)};
    row_sums<LANES>(s, scratch[half]);
    if (row >= p.rows) continue;
    const V c1 = vset(V{}, -s[0] * inv * r), c2 = vset(V{}, -s[1] * inv * r);
    T* dx = static_cast<T*>(p.dx) + row * p.dx_ld;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (t + k * lanes) * VEC;
      if (col >= p.width) continue;
      V x[NP], d[NP], w[NP];
      unpack_lanes<T, VEC>(cx[k], x);
      unpack_lanes<T, VEC>(cd[k], d);
      weights(k, col, w);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const V xh = vmul(vadd(x[i], minus), scale);
        x[i] = vfma(xh, c2, vfma(vmul(w[i], d[i]), scale, c1));
      }
      store_once(dx + col, pack_lanes<T, VEC>(x));
    }
  }

  float* part = p.part + (int64_t)blockIdx.x * 2 * p.width;
  if constexpr (LANES == 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (t + k * lanes) * VEC;
      if (col >= p.width) continue;
      float ew[VEC], eb[VEC];
      from_lanes(dw[k], ew);
      from_lanes(db[k], eb);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        part[col + i] = ew[i];
        part[p.width + col + i] = eb[i];
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
        float e[VEC];
        from_lanes(which ? db[k] : dw[k], e);
#pragma unroll
        for (int i = 0; i < VEC; ++i) lines[group * p.width + col + i] = e[i];
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

// Long rows whose start and length are multiples of 16 bytes: bulk copies stream x and dy rows
// into a ring of shared memory (no addresses, predicates or registers per thread), ROWS rows
// a stage.  Both passes read the stage; one barrier per stage joins the rows' sums, and
// behind it the stage before is free: thread 0 refills it there.
template <int N>
__device__ __forceinline__ void warp_scatter_sum(float (&v)[N], int lane) {   // N = 2 or 4: lane holds sum lane / (32 / N)
#pragma unroll
  for (int n = N, o = 16; n > 1; n >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < n / 2; ++j) {
      const float send = up ? v[j] : v[j + n / 2], keep = up ? v[j + n / 2] : v[j];
      v[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
#pragma unroll
  for (int o = 16 / N; o; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
}

constexpr int kMaxStages = 4;

template <typename T, typename TW, int VEC, int NV, int ROWS, int MAXT, int PER_SM, bool HELD>
__global__ void __launch_bounds__(MAXT, PER_SM) backward_ring_kernel(const Bwd p, const int stages) {
  using namespace sm100;
  using R = Raw<T, VEC>;
  using V = typename Lanes<VEC>::V;
  constexpr int NP = Lanes<VEC>::N, SUMS = 2 * ROWS, SHARE = 32 / SUMS;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kMaxStages];
  __shared__ float scratch[2][SUMS][33];
  __shared__ int given_up;
  const int lanes = blockDim.x, warps = lanes >> 5;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const uint32_t row_bytes = p.width * sizeof(T), stage_bytes = 2 * ROWS * row_bytes;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  auto fill = [&](int stage, int64_t row) {                  // one thread
    if (row >= p.rows) return;
    const int n = row + ROWS <= p.rows ? ROWS : (int)(p.rows - row);
    mbar_arrive_expect_tx(&full[stage], 2 * n * row_bytes);
    uint8_t* to = ring + (size_t)stage * stage_bytes;
    for (int r = 0; r < n; ++r) {
      bulk_load(to + 2 * r * row_bytes, static_cast<const T*>(p.x) + (row + r) * p.x_ld, row_bytes, &full[stage]);
      bulk_load(to + (2 * r + 1) * row_bytes, static_cast<const T*>(p.dy) + (row + r) * p.dy_ld, row_bytes, &full[stage]);
    }
  };
  int64_t row = (int64_t)blockIdx.x * ROWS;
  if (t == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    given_up = 0;
    fence_barrier_init();
    for (int s = 0; s < stages; ++s) fill(s, row + s * step);
  }
  for (int i = t; i < 2 * SUMS * 33; i += lanes) (&scratch[0][0][0])[i] = 0.f;   // warps that are not there count zero
  __syncthreads();

  const float inv = 1.0f / (float)p.width;
  V dw[NV][NP], db[NV][NP];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < NP; ++i) dw[k][i] = db[k][i] = vset(V{}, 0.f);
  Weights<TW, VEC> held[HELD ? NV : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (p.w && (t + k * lanes) * VEC < p.width) held[k].load(p.w, (t + k * lanes) * VEC);
  }
  auto weights = [&](int k, int col, V (&w)[NP]) {
    if (p.w) {
      if constexpr (!HELD) held[0].load(p.w, col);
      held[HELD ? k : 0].get(w);
    } else {
#pragma unroll
      for (int i = 0; i < NP; ++i) w[i] = vset(V{}, 1.f);
    }
  };
  float mean[ROWS], rstd[ROWS];
  auto stats = [&](int64_t row) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      mean[r] = row + r < p.rows ? __ldg(p.mean + row + r) : 0.f;
      rstd[r] = row + r < p.rows ? __ldg(p.rstd + row + r) : 0.f;
    }
  };
  stats(row);
  int stage = 0, half = 0;
  uint32_t phase = 0;
  for (; row < p.rows; row += step, half ^= 1) {
    int ok = mbar_wait(&full[stage], phase, &given_up);
    const uint8_t* from = ring + (size_t)stage * stage_bytes;
    const int n = row + ROWS <= p.rows ? ROWS : (int)(p.rows - row);
    float sums[SUMS], m[ROWS], q[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      m[r] = mean[r];
      q[r] = rstd[r];
      V a1 = vset(V{}, 0.f), a2 = vset(V{}, 0.f);
      if (r < n) {
        const V minus = vset(V{}, -m[r]), scale = vset(V{}, q[r]);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int col = (t + k * lanes) * VEC;
          if (col >= p.width) break;
          V x[NP], d[NP], w[NP];
          unpack_lanes<T, VEC>(*reinterpret_cast<const R*>(from + 2 * r * row_bytes + col * sizeof(T)), x);
          unpack_lanes<T, VEC>(*reinterpret_cast<const R*>(from + (2 * r + 1) * row_bytes + col * sizeof(T)), d);
          weights(k, col, w);
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const V xh = vmul(vadd(x[i], minus), scale), td = vmul(w[i], d[i]);
            a1 = vadd(a1, td);
            a2 = vfma(td, xh, a2);
            dw[k][i] = vfma(d[i], xh, dw[k][i]);
            db[k][i] = vadd(db[k][i], d[i]);
          }
        }
      }
      sums[2 * r] = hsum(a1);
      sums[2 * r + 1] = hsum(a2);
    }
    stats(row + step);                                       // of the next stage, while this one is joined
    warp_scatter_sum(sums, lane);
    if (lane % SHARE == 0) scratch[half][lane / SHARE][warp] = sums[0];
    ok = __syncthreads_and(ok);                              // every warp has data, or all stop together
    if (!ok) {
      if (t == 0) {                                          // copies already issued land before the CTA exits
        const uint64_t t0 = globaltimer();
        for (int i = 0; i < stages && row < p.rows; ++i, row += step) {
          while (!mbar_try_wait(&full[stage], phase) && globaltimer() - t0 < kWaitLimitNs) {
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      break;
    }
    if (t == 0 && row != (int64_t)blockIdx.x * ROWS) fill(stage ? stage - 1 : stages - 1, row + (stages - 1) * step);
    float s = 0.f;                                           // sum lane / SHARE over the warps
#pragma unroll
    for (int w = 0; w < 32; w += SHARE)
      if (w < warps) s += scratch[half][lane / SHARE][w + lane % SHARE];
#pragma unroll
    for (int o = SHARE / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float s1 = __shfl_sync(0xffffffffu, s, 2 * r * SHARE), s2 = __shfl_sync(0xffffffffu, s, (2 * r + 1) * SHARE);
      if (r >= n) continue;
      // dx = q t - q s1 - q xh s2 with xh = (x - m) q.  x is centred first: the mean folded into the
      // offset saves an addition a value but leaves x slope and m slope to cancel, an error of u |m| / std
      const V minus = vset(V{}, -m[r]), scale = vset(V{}, q[r]), c2 = vset(V{}, -s2 * inv * q[r] * q[r]),
              c1 = vset(V{}, -s1 * inv * q[r]);
      T* dx = static_cast<T*>(p.dx) + (row + r) * p.dx_ld;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (t + k * lanes) * VEC;
        if (col >= p.width) break;
        V x[NP], d[NP], w[NP];
        unpack_lanes<T, VEC>(*reinterpret_cast<const R*>(from + 2 * r * row_bytes + col * sizeof(T)), x);
        unpack_lanes<T, VEC>(*reinterpret_cast<const R*>(from + (2 * r + 1) * row_bytes + col * sizeof(T)), d);
        weights(k, col, w);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          x[i] = vfma(vadd(x[i], minus), c2, vfma(vmul(w[i], d[i]), scale, c1));
        }
        store_once(dx + col, pack_lanes<T, VEC>(x));
      }
    }
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
  float* part = p.part + (int64_t)blockIdx.x * 2 * p.width;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int col = (t + k * lanes) * VEC;
    if (col >= p.width) break;
    float ew[VEC], eb[VEC];
    from_lanes(dw[k], ew);
    from_lanes(db[k], eb);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      part[col + i] = ew[i];
      part[p.width + col + i] = eb[i];
    }
  }
  if (given_up && t == 0 && p.status) atomicExch(p.status, VDN_ERR_TIMEOUT);
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
  s1 = row_sum<0>(s1, scratch) * inv;
  s2 = row_sum<0>(s2, scratch + 1) * inv;
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

constexpr int kSMs = 148;

template <typename T, typename TW, int VEC, int LANES>
static int launch_forward(const Fwd& p, cudaStream_t stream) {
  constexpr int64_t per = 256 / LANES, most = kSMs * 5;
  const int64_t ctas = (p.rows + per - 1) / per;
  forward_kernel<T, TW, VEC, LANES><<<(unsigned)(ctas < most ? ctas : most), 256, 0, stream>>>(p);
  VDN_LAUNCH_CHECK("layer norm");
  return VDN_OK;
}

template <typename T, typename TW, int VEC, int NV, int ROWS, int LANES, int MAXT, int PER_SM>
static int launch_row(const Fwd& p, int block, cudaStream_t stream) {
  const int64_t per = (LANES ? block / (LANES ? LANES : 1) : 1) * ROWS;
  forward_row_kernel<T, TW, VEC, NV, ROWS, LANES, MAXT, PER_SM><<<(unsigned)((p.rows + per - 1) / per), block, 0, stream>>>(p);
  VDN_LAUNCH_CHECK("layer norm (rows)");
  return VDN_OK;
}

// Elements per access that the width, the strides and the addresses allow: 16 bytes, 4, or one.
template <typename T>
static int vector_of(int width, std::initializer_list<int64_t> strides, std::initializer_list<const void*> rows,
                     std::initializer_list<const void*> params, size_t param_size) {
  for (int v : {16 / (int)sizeof(T), 2}) {
    bool ok = width % v == 0;
    for (int64_t s : strides) ok = ok && s % v == 0;
    for (const void* q : rows) ok = ok && aligned_to(q, v * sizeof(T));
    for (const void* q : params) ok = ok && (!q || aligned_to(q, v * param_size > 16 ? 16 : v * param_size));
    if (ok) return v;
  }
  return 1;
}

template <typename T, typename TW>
static int forward(const Fwd& p, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int vec = vector_of<T>(p.width, {p.x_ld, p.y_ld}, {p.x, p.y}, {p.w, p.b}, sizeof(TW));
  const int n = p.width / vec;
  if (vec == V) {
    if (n <= 8) return launch_forward<T, TW, V, 8>(p, stream);
    if (n <= 16) return launch_forward<T, TW, V, 16>(p, stream);
    if (n <= 32) return launch_forward<T, TW, V, 32>(p, stream);
    // 16-bit rows under fp32 weights are bound by the weights' loads: two rows share them.
    if constexpr (sizeof(T) == 2) {
      if (n <= 2 * 32) return launch_row<T, TW, V, 2, 2, 32, 128, 8>(p, 128, stream);
      if (n <= 4 * 32) return launch_row<T, TW, V, 4, 2, 32, 128, 6>(p, 128, stream);
      if (n <= 5 * 256) return launch_row<T, TW, V, 5, 2, 0, 256, 2>(p, (n + 159) / 160 * 32, stream);
      if (n <= 8 * 256) return launch_row<T, TW, V, 8, 1, 0, 256, 3>(p, (n + 255) / 256 * 32, stream);
      if (n <= 8 * 1024) return launch_row<T, TW, V, 8, 1, 0, 1024, 1>(p, (n + 255) / 256 * 32, stream);
    } else {
      if (n <= 4 * 32) return launch_row<T, TW, V, 4, 1, 32, 256, 4>(p, 256, stream);
      if (n <= 8 * 32) return launch_row<T, TW, V, 8, 1, 32, 256, 3>(p, 256, stream);
      if (n <= 12 * 128) return launch_row<T, TW, V, 12, 1, 0, 512, 1>(p, (n + 383) / 384 * 32, stream);
      if (n <= 4 * 1024) return launch_row<T, TW, V, 4, 1, 0, 1024, 1>(p, (n + 127) / 128 * 32, stream);
      if (n <= 12 * 512) return launch_row<T, TW, V, 12, 1, 0, 512, 1>(p, (n + 383) / 384 * 32, stream);
    }
  } else if (vec == 2) {
    if (n <= 8 * 32) return launch_row<T, TW, 2, 8, 4, 32, 128, 4>(p, 128, stream);
    if (n <= 16 * 32) return launch_row<T, TW, 2, 16, 2, 32, 128, 4>(p, 128, stream);
    if (n <= 8 * 512) return launch_row<T, TW, 2, 8, 2, 0, 512, 2>(p, (n + 255) / 256 * 32, stream);
    if (n <= 16 * 1024) return launch_row<T, TW, 2, 16, 1, 0, 1024, 1>(p, (n + 511) / 512 * 32, stream);
  } else {
    if (n <= 8 * 32) return launch_row<T, TW, 1, 8, 4, 32, 128, 4>(p, 128, stream);
    if (n <= 16 * 32) return launch_row<T, TW, 1, 16, 2, 32, 128, 4>(p, 128, stream);
    if (n <= 8 * 1024) return launch_row<T, TW, 1, 8, 2, 0, 1024, 1>(p, (n + 255) / 256 * 32, stream);
    if (n <= 16 * 1024) return launch_row<T, TW, 1, 16, 1, 0, 1024, 1>(p, (n + 511) / 512 * 32, stream);
  }
  forward_wide_kernel<T, TW><<<(unsigned)p.rows, 1024, 0, stream>>>(p);
  VDN_LAUNCH_CHECK("layer norm (wide)");
  return VDN_OK;
}

// CTAs of the backward, one line of partial sums each.  A CTA per row has about width / 16
// threads, so narrower rows take more CTAs to fill 148 SMs (the 16-bit ring kernel: a warp
// per 1280 columns, eight warps an SM).  The count depends on the shape and type alone, so
// results do not vary.
static int64_t plain_lines(int64_t width) { return 2 * kSMs * (width >= 5120 ? 1 : width <= 512 ? 10 : 5120 / width); }
static int64_t ring_lines(int64_t width) {
  const int64_t warps = (width + 1279) / 1280;
  return kSMs * (warps >= 4 ? 2 : warps == 3 ? 3 : 8 / warps);
}
static int64_t line_count(int64_t rows, int64_t width) {   // the most that any kernel takes
  const int64_t a = plain_lines(width), b = ring_lines(width), lines = a > b ? a : b;
  return rows < lines ? rows : lines;
}
constexpr int kGroupLines = 4 * kSMs;        // where a lane group takes a row: CTAs of several rows

template <typename T, typename TW, int VEC, int NV, int LANES, int MAXT, int PER_SM, bool HELD>
static int launch_backward(const Bwd& p, int block, int lines, cudaStream_t stream) {
  const size_t smem = LANES ? sizeof(float) * (block / (LANES ? LANES : 1)) * (size_t)p.width : 0;
  backward_kernel<T, TW, VEC, NV, LANES, MAXT, PER_SM, HELD><<<lines, block, smem, stream>>>(p);
  VDN_LAUNCH_CHECK("layer norm backward");
  return VDN_OK;
}

// The ring kernel, where two stages fit beside the CTAs that share an SM (0: they do not).
constexpr int kSmemPerSM = 227 * 1024;
template <typename T, typename TW, int VEC, int NV, int ROWS, int MAXT, int PER_SM, bool HELD>
static int launch_ring(const Bwd& p, int block, int lines, cudaStream_t stream, bool& done) {
  const int64_t stage = 2ll * ROWS * p.width * sizeof(T);
  int stages = 0;                                    // as many CTAs an SM as its threads allow, or fewer for two stages
  for (int share = PER_SM * (MAXT / block < 1 ? 1 : MAXT / block); share >= 1 && stages < 2; --share) {
    const int64_t n = (kSmemPerSM / share - 2048) / stage;
    stages = (int)(n < kMaxStages ? n : kMaxStages);
  }
  if (stages < 2) return VDN_OK;
  auto* kernel = backward_ring_kernel<T, TW, VEC, NV, ROWS, MAXT, PER_SM, HELD>;
  static bool set[64] = {};
  int dev = 0;
  VDN_CUDA_TRY(cudaGetDevice(&dev));
  VDN_CHECK_ARG(dev >= 0 && dev < 64, "device index out of range");
  if (!set[dev]) {
    VDN_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerSM - 2048));
    set[dev] = true;
  }
  kernel<<<lines, block, stages * stage, stream>>>(p, stages);
  VDN_LAUNCH_CHECK("layer norm backward (ring)");
  done = true;
  return VDN_OK;
}

template <typename T, typename TW>
static int backward(const Bwd& p, void* dw, void* db, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T), M = sizeof(T) / 2;   // M: fp32 holds half the values per vector
  const int vec = vector_of<T>(p.width, {p.x_ld, p.dy_ld, p.dx_ld}, {p.x, p.dy, p.dx}, {p.w}, sizeof(TW));
  auto few_of = [&](int64_t most) { return (int)(p.rows < most ? p.rows : most); };
  const int n = p.width / vec, few = few_of(kGroupLines);
  int lines = few_of(plain_lines(p.width)), rc = -1;
  if (vec == V) {
    bool done = false;
    if (n <= 8) rc = launch_backward<T, TW, V, 1, 8, 128, 4, true>(p, 128, lines = few, stream);
    else if (n <= 16) rc = launch_backward<T, TW, V, 1, 16, 128, 4, true>(p, 128, lines = few, stream);
    else if (n <= 32) rc = launch_backward<T, TW, V, 1, 32, 128, 4, true>(p, 128, lines = few, stream);
    else if (n <= 64) rc = launch_backward<T, TW, V, 2, 32, 128, 4, true>(p, 128, lines = few, stream);
    // 16 bits: few fat threads (40 columns, up to 255 registers) cost the fewest instructions a
    // value (5120 columns: 183 us against 227 for 16 columns a thread); 32 bits: bound by HBM
    else if (M == 1 && n <= 640) {
      if constexpr (M == 1)
        rc = launch_ring<T, TW, V, 5, 2, 128, 2, true>(p, (n + 159) / 160 * 32, lines = few_of(ring_lines(p.width)), stream, done);
    } else if (M == 2 && n <= 4 * 320) {
      if constexpr (M == 2) rc = launch_ring<T, TW, V, 4, 1, 320, 2, true>(p, (n + 127) / 128 * 32, lines, stream, done);
    } else if (n <= 4 * M * 512) {
      rc = launch_ring<T, TW, V, 4 * M, 1, 512, 1, false>(p, (n + 128 * M - 1) / (128 * M) * 32, lines, stream, done);
      if constexpr (M == 2)                          // 32-bit rows too long for two stages (16-bit ones never are)
        if (rc == VDN_OK && !done) rc = launch_backward<T, TW, V, 4 * M, 0, 512, 1, false>(p, (n + 128 * M - 1) / (128 * M) * 32, lines, stream);
    }
  } else if (vec == 2) {
    if (n <= 128) rc = launch_backward<T, TW, 2, 4, 32, 128, 4, true>(p, 128, lines = few, stream);
    else if (n <= 8 * 512) rc = launch_backward<T, TW, 2, 8, 0, 512, 1, true>(p, (n + 255) / 256 * 32, lines, stream);
  } else {
    if (n <= 256) rc = launch_backward<T, TW, 1, 8, 32, 128, 4, true>(p, 128, lines = few, stream);
    else if (n <= 16 * 512) rc = launch_backward<T, TW, 1, 16, 0, 512, 1, true>(p, (n + 511) / 512 * 32, lines, stream);
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
  return sizeof(float) * 2 * (size_t)vdn::lnorm::line_count(rows, width) * (size_t)width;
}

extern "C" int vdn_layer_norm_backward(const void* dy, int dtype, int64_t rows, int64_t width, int64_t dy_stride,
                                       const void* x, int64_t x_stride, const void* weight, int w_dtype,
                                       const float* mean, const float* rstd, void* dx, int64_t dx_stride,
                                       void* d_weight, void* d_bias, void* workspace, size_t workspace_bytes,
                                       int* status, cudaStream_t stream) {
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
  VDN_CHECK_ARG(aligned_to(workspace, sizeof(float)), "the workspace must be aligned to fp32 values");
  const Bwd p = {dy, x, weight, mean, rstd, dx, static_cast<float*>(workspace), rows, dy_stride, x_stride, dx_stride,
                 (int)width, status};
  VDN_LN_DISPATCH(backward, p, d_weight, d_bias, stream)
}
