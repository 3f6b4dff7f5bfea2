// Gated linear recurrence per channel, forward and backward, sm_100a.
//
//   forward   h_t = a_t h_{t-1} + x_t,  a_t = exp(g_t),  y_t = h_t
//   backward  u_t = dy_t + c_t,  dx_t = u_t,  c_{t-1} = a_t u_t,  dg_t = c_{t-1} h_{t-1}
//             (c_T = gradient of the last state, c_0 = gradient of the first; h_{t-1} is
//             the saved y_{t-1}, or the first state)
//
// Both are a chain of maps c -> A c + H, so a run of tokens folds into one (A, H) pair
// per channel and runs join in any grouping.  HBM is the bound: the forward moves three
// elements per token and channel, the backward five, for a dozen instructions each.  So
// the inputs are read ONCE and kept in registers while the runs are joined:
//   * a warp owns L tokens of 32 * VEC channels (lane = VEC neighbouring channels) and folds
//     them into (A, H), keeping for each token its state from zero and its reach, the
//     product of the decays so far; after the join its true states are state + reach * carry;
//   * a CTA of up to four warps owns neighbouring runs, joined through shared memory;
//   * a cluster of up to eight CTAs owns neighbouring CTA runs and walks the sequence in
//     rounds.  Each CTA sends its pair into the others' shared memory with asynchronous
//     stores that count on their mbarriers: unlike a cluster barrier (whose release waits
//     for the round's output stores: 480 against 355 us below) this orders nothing else.
//     No flags in global memory, no workspace, and the order of every sum is fixed: the
//     same bits on every run.
//
// Numerics: states, folds and sums in fp32.  A decay close to 1 loses its distance from
// 1 when it is rounded to fp32 (a memory of n tokens then errs by n * 2^-25, and a constant decay errs
// the same way at every token), so exp(g) is kept as a pair hi + lo with 2^n as a common
// factor: hi = fp32(1 + e), lo = e - (hi - 1), e = expm1(r) with r = g - n ln 2 in [-0.35,
// 0.35] from a polynomial fitted at Chebyshev nodes (2.5e-8 relative).  It runs on packed
// fp32 pairs with no branch and no MUFU operation.  A run's A comes from the sum of its g, not
// from the product of its rounded decays.  exp(g) is 0 below g = -87.7.
#include <initializer_list>
#include <type_traits>

#include "train_common.cuh"
#include "sm100.cuh"

namespace vdn {
namespace gscan {

using namespace sm100;

constexpr int MAX_WARPS = 4, MAX_CLUSTER = 8;

struct Params {
  const void* x;        // forward: x; backward: dy
  const void* g;        // log decay
  const void* y_in;     // backward: saved y
  void* out;            // forward: y; backward: dx
  void* dg;             // backward
  const float* first;   // first state [S, C] or null
  const float* dlast;   // backward: gradient of the last state [S, C] or null
  float* last;          // forward: last state; backward: gradient of the first state; or null
  const int32_t* cu;    // [S + 1] row offsets of packed sequences, or null (dense: S batches of T rows)
  int64_t x_row, g_row, y_row, out_row, dg_row;            // strides in elements
  int64_t x_batch, g_batch, y_batch, out_batch, dg_batch;  // dense only
  int rows;             // dense: T; packed: rows of the tensors
  int64_t seqs, channels;
  int tiles;
  bool reverse, zero_tail;
  int* status;
};

// 2^n from the low bits of t = fp32(n + 127 + 1.5 * 2^23); 0 for n = -127, inf for n = 128.
__device__ __forceinline__ float two_to(float t) { return __uint_as_float(__float_as_uint(t) << 23); }
__device__ __forceinline__ f2 two_to(f2 t) {
  float a, b;
  f2_unpack(t, a, b);
  return f2_pack(two_to(a), two_to(b));
}
__device__ __forceinline__ float clamp_decay(float g) {       // NaN stays NaN
  float r;
  asm("max.NaN.f32 %0, %1, 0fC2AFCCCD;\n\tmin.NaN.f32 %0, %0, 0f42B18000;" : "=f"(r) : "f"(g));   // [-87.9, 88.75]
  return r;
}
__device__ __forceinline__ f2 clamp_decay(f2 g) {
  float a, b;
  f2_unpack(g, a, b);
  return f2_pack(clamp_decay(a), clamp_decay(b));
}

// exp(g) as hi + lo (see above): n = round(g / ln 2), r = g - n ln 2, e = expm1(r).
template <typename V>
__device__ __forceinline__ void decay_pair(V g, V& hi, V& lo) {
  auto c = [](float v) { return vset(V{}, v); };
  g = clamp_decay(g);
  const V t = vfma(g, c(1.4426950408889634f), c(12582912.0f + 127.0f));
  const V n = vadd(t, c(-12582912.0f - 127.0f));
  V r = vfma(n, c(-0.693359375f), g);                // exact: n has 8 bits, the constant 12
  r = vfma(n, c(2.12194440e-4f), r);
  V e = vfma(r, c(1.3942162e-3f), c(8.369872e-3f));
  e = vfma(e, r, c(4.166634e-2f));
  e = vfma(e, r, c(1.6666499e-1f));
  e = vfma(e, r, c(0.5f));
  e = vmul(vfma(e, r, c(1.0f)), r);
  const V one = vadd(e, c(1.0f)), scale = two_to(t);
  hi = vmul(one, scale);
  lo = vmul(vadd(e, vfma(one, c(-1.0f), c(1.0f))), scale);
}
template <typename V>
__device__ __forceinline__ V decay_of(V g) {
  V hi, lo;
  decay_pair(g, hi, lo);
  return vadd(hi, lo);
}

// A run's map c -> a c + h.
template <typename V> struct Fold;
template <> struct __align__(8) Fold<float> { float a, h; };
template <> struct __align__(16) Fold<f2> { f2 a, h; };
// Stores to a CTA of the cluster that count on its mbarrier when they arrive.
__device__ __forceinline__ void send(uint32_t addr, const Fold<float>& f, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(addr),
               "f"(f.a), "f"(f.h), "r"(bar) : "memory");
}
__device__ __forceinline__ void send(uint32_t addr, const Fold<f2>& f, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(addr),
               "l"(f.a), "l"(f.h), "r"(bar) : "memory");
}

template <typename T, typename TG, int VEC, int L, bool BWD, bool SHARED>
__global__ void __launch_bounds__(MAX_WARPS * 32, 5) scan_kernel(const Params p, const int cluster) {
  constexpr int GV = SHARED ? 1 : VEC;               // decays per lane and token
  constexpr int TILE = 32 * VEC;
  using RX = Raw<T, VEC>;
  using RG = Raw<TG, GV>;
  using V = typename Lanes<VEC>::V;                  // values
  using G = typename Lanes<GV>::V;                   // decays
  constexpr int NV = Lanes<VEC>::N, NG = Lanes<GV>::N;
  __shared__ Fold<V> folds[2][MAX_WARPS][NV][32];
  __shared__ G sums[2][MAX_WARPS][NG][32];
  __shared__ Fold<V> runs[2][MAX_CLUSTER][NV][32];   // one line from every CTA of the cluster
  __shared__ uint64_t arrived[2];
  __shared__ int given_up;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int rank = (int)cluster_ctarank();
  const int64_t id = blockIdx.x / cluster;           // sequence-major, channel tiles fastest
  const int64_t seq = id / p.tiles;
  const int tile = (int)(id - seq * p.tiles);
  const int64_t c = (int64_t)tile * TILE + lane * VEC;
  const bool live = c < p.channels;
  const bool full = (int64_t)(tile + 1) * TILE <= p.channels;
  const int64_t gc = SHARED ? tile : c;              // shared: one head is one tile

  int begin = 0, len = p.rows;
  if (p.cu) {
    const int lo = seq < p.seqs ? p.cu[seq] : p.cu[p.seqs];
    const int hi = seq < p.seqs ? p.cu[seq + 1] : p.rows;
    begin = min(max(lo, 0), p.rows);                 // offsets out of range stay inside the tensors
    len = max(min(hi, p.rows) - begin, 0);
  }
  if (seq >= p.seqs) {                               // rows behind the last sequence
    for (int64_t t = rank * warps + warp; t < len; t += warps * cluster) {
      if (live) *reinterpret_cast<RX*>(static_cast<T*>(p.out) + (begin + t) * p.out_row + c) = raw_zero<RX>();
      if (BWD && (SHARED ? lane == 0 : live))
        *reinterpret_cast<RG*>(static_cast<TG*>(p.dg) + (begin + t) * p.dg_row + gc) = raw_zero<RG>();
    }
    return;                                          // the whole cluster is here
  }

  if (threadIdx.x == 0) {
    mbar_init(&arrived[0], 1);
    mbar_init(&arrived[1], 1);
    given_up = 0;
    fence_barrier_init();
  }
  cluster_sync();                                    // the barriers stand before anyone sends

  // Walk order: the forward follows the recurrence, the backward its reverse.
  const bool down = p.reverse != BWD;                // token rows descend along the walk
  const int64_t row0 = down ? (int64_t)begin + len - 1 : begin;
  const int sgn = down ? -1 : 1;
  const int64_t b = p.cu ? 0 : seq;
  const T* px = static_cast<const T*>(p.x) + b * p.x_batch + row0 * p.x_row + c;
  const TG* pg = static_cast<const TG*>(p.g) + b * p.g_batch + row0 * p.g_row + gc;
  const T* py = BWD ? static_cast<const T*>(p.y_in) + b * p.y_batch + row0 * p.y_row + c : nullptr;
  T* po = static_cast<T*>(p.out) + b * p.out_batch + row0 * p.out_row + c;
  TG* pdg = BWD ? static_cast<TG*>(p.dg) + b * p.dg_batch + row0 * p.dg_row + gc : nullptr;
  const int sx = sgn * (int)p.x_row, sg = sgn * (int)p.g_row, sy = sgn * (int)p.y_row, so = sgn * (int)p.out_row,
            sdg = sgn * (int)p.dg_row;

  V carry[NV];                                       // the state in front of the round
  {
    const float* from = BWD ? p.dlast : p.first;
    float e[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) e[v] = from && live ? from[seq * p.channels + c + v] : 0.f;
    to_lanes(e, carry);
  }

  RX rx[L], ry[BWD ? L : 1];
  RG rg[L];
  auto load = [&](int64_t i0) {
    const T* qx = px + i0 * sx;
    const TG* qg = pg + i0 * sg;
    if (full && i0 + L + (BWD ? 1 : 0) <= len) {      // the common case, without predicates
      const T* qy = BWD ? py + (i0 + 1) * sy : nullptr;
#pragma unroll
      for (int l = 0; l < L; ++l) {
        rx[l] = load_once<RX>(qx + l * sx);
        rg[l] = load_once<RG>(qg + l * sg);
        if constexpr (BWD) ry[l] = load_once<RX>(qy + l * sy);
      }
      return;
    }
    const int n = live ? (int)min((int64_t)len - i0, (int64_t)L) : 0;
    const int ng = SHARED ? (int)min((int64_t)len - i0, (int64_t)L) : n;
#pragma unroll
    for (int l = 0; l < L; ++l) {
      rx[l] = l < n ? load_once<RX>(qx + l * sx) : raw_zero<RX>();
      rg[l] = l < ng ? load_once<RG>(qg + l * sg) : raw_zero<RG>();
    }
    if constexpr (BWD) {
      const T* qy = py + (i0 + 1) * sy;
      const int ny = i0 + n == len ? n - 1 : n;      // the oldest token's h_{t-1} is the first state
#pragma unroll
      for (int l = 0; l < L; ++l) ry[l] = l < ny ? load_once<RX>(qy + l * sy) : raw_zero<RX>();
    }
  };

  const int round_tokens = cluster * warps * L;
  int64_t i0 = (rank * warps + warp) * L;
  int buf = 0;
  uint32_t phase = 0;
  for (int64_t done = 0; done < len; done += round_tokens, i0 += round_tokens, buf ^= 1) {
    load(i0);
    // First walk, from zero: part[l] the state after token l, reach[l] the product of the
    // decays up to it, so that the true state is part + reach * (the carry).
    V part[L][NV], fold[NV];
    G reach[L][NG], sum[NG], far[NG];
#pragma unroll
    for (int v = 0; v < NV; ++v) fold[v] = vset(V{}, 0.f);
#pragma unroll
    for (int v = 0; v < NG; ++v) {
      sum[v] = vset(G{}, 0.f);
      far[v] = vset(G{}, 1.f);
    }
#pragma unroll
    for (int l = 0; l < L; ++l) {
      V x[NV];
      G g[NG], hi[NG], lo[NG];
      unpack_lanes<T, VEC>(rx[l], x);
      unpack_lanes<TG, GV>(rg[l], g);
#pragma unroll
      for (int v = 0; v < NG; ++v) {
        decay_pair(g[v], hi[v], lo[v]);
        sum[v] = vadd(sum[v], g[v]);
        far[v] = vmul(far[v], hi[v]);
        reach[l][v] = far[v];
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        V h, e;
        spread(hi[SHARED ? 0 : v], h);
        spread(lo[SHARED ? 0 : v], e);
        if (BWD) {
          const V u = vadd(x[v], fold[v]);
          fold[v] = vfma(h, u, vmul(e, u));
        } else {
          fold[v] = vfma(h, fold[v], vfma(e, fold[v], x[v]));
        }
        part[l][v] = fold[v];
      }
    }

    // Join the warps of the CTA: `before` is the fold of the warps in front of this one.
    Fold<V> own[NV], before[NV];
    {
      G a[NG];
#pragma unroll
      for (int v = 0; v < NG; ++v) {
        a[v] = decay_of(sum[v]);
        sums[buf][warp][v][lane] = sum[v];
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        spread(a[SHARED ? 0 : v], own[v].a);
        own[v].h = fold[v];
        folds[buf][warp][v][lane] = own[v];
        before[v].a = vset(V{}, 1.f);
        before[v].h = vset(V{}, 0.f);
      }
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < MAX_WARPS - 1; ++w) {
      if (w < warp) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const Fold<V> f = folds[buf][w][v][lane];
          before[v].a = vmul(before[v].a, f.a);
          before[v].h = vfma(f.a, before[v].h, f.h);
        }
      }
    }
    if (warp == warps - 1) {                         // the CTA's own fold, to every CTA
      G s[NG];
#pragma unroll
      for (int v = 0; v < NG; ++v) s[v] = sum[v];
      for (int w = 0; w < warp; ++w) {
#pragma unroll
        for (int v = 0; v < NG; ++v) s[v] = vadd(s[v], sums[buf][w][v][lane]);
      }
#pragma unroll
      for (int v = 0; v < NG; ++v) s[v] = decay_of(s[v]);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        Fold<V> f;
        spread(s[SHARED ? 0 : v], f.a);
        f.h = vfma(own[v].a, before[v].h, own[v].h);
        for (int r = 0; r < cluster; ++r)
          send(mapa_shared(&runs[buf][rank][v][lane], r), f, mapa_shared(&arrived[buf], r));
      }
      if (lane == 0) mbar_arrive_expect_tx(&arrived[buf], cluster * (uint32_t)sizeof(runs[0][0]));
    }
    // A line's buffer is written again two rounds later, by CTAs that have this one's next
    // line, which it sends after all its warps have read this round's.
    if (!mbar_wait(&arrived[buf], phase, &given_up)) break;
    phase ^= buf;
    V in[NV];                                        // the true carry in front of this warp
#pragma unroll
    for (int v = 0; v < NV; ++v) in[v] = carry[v];
#pragma unroll
    for (int r = 0; r < MAX_CLUSTER; ++r) {
      if (r < cluster) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          if (r == rank) in[v] = carry[v];
          const Fold<V> f = runs[buf][r][v][lane];
          carry[v] = vfma(f.a, carry[v], f.h);
        }
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) in[v] = vfma(before[v].a, in[v], before[v].h);

    // Second walk, with the true carry.
    const int left = (int)min((int64_t)len - i0, (int64_t)L + 1);   // L + 1: more tokens follow
    T* qo = po + i0 * so;
    if constexpr (!BWD) {
      auto walk = [&](auto all) {
#pragma unroll
        for (int l = 0; l < L; ++l) {
          V y[NV];
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            V r;
            spread(reach[l][SHARED ? 0 : v], r);
            y[v] = vfma(r, in[v], part[l][v]);
          }
          if (all.value || (live && l < left)) store_once(qo + l * so, pack_lanes<T, VEC>(y));
        }
      };
      if (full && left >= L) walk(std::true_type{}); else walk(std::false_type{});
    } else {
      TG* qdg = pdg + i0 * sdg;
      float dgs[L];
      auto walk = [&](auto all) {
        V c0[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) c0[v] = in[v];
#pragma unroll
        for (int l = 0; l < L; ++l) {
          V u[NV], d[NV], y[NV];
          unpack_lanes<T, VEC>(ry[l], y);
          if (!all.value && l + 1 == left) {         // the oldest token
            float e[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) e[v] = p.first && live ? p.first[seq * p.channels + c + v] : 0.f;
            to_lanes(e, y);
          }
          unpack_lanes<T, VEC>(rx[l], u);
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            V r;
            spread(reach[l][SHARED ? 0 : v], r);
            u[v] = vadd(u[v], c0[v]);
            c0[v] = vfma(r, in[v], part[l][v]);
            d[v] = vmul(c0[v], y[v]);
          }
          if (all.value || (live && l < left)) store_once(qo + l * so, pack_lanes<T, VEC>(u));
          if constexpr (SHARED) {
            float e[VEC];
            from_lanes(d, e);
            dgs[l] = 0.f;
#pragma unroll
            for (int v = 0; v < VEC; ++v) dgs[l] += e[v];
          } else {
            if (all.value || (live && l < left)) store_once(qdg + l * sdg, pack_lanes<TG, VEC>(d));
          }
        }
      };
      if (full && left > L) walk(std::true_type{}); else walk(std::false_type{});
      if constexpr (SHARED) {
        // Sum each token's terms over the head: the first rounds halve the tokens a lane
        // holds while they halve the lanes, so L sums cost about L + 5 shuffles.
        int off = 16;
#pragma unroll
        for (int n = L; n > 1; n >>= 1, off >>= 1) {
          const bool up = lane & off;
#pragma unroll
          for (int j = 0; j < n / 2; ++j) {
            const float send = up ? dgs[j] : dgs[j + n / 2], keep = up ? dgs[j + n / 2] : dgs[j];
            dgs[j] = keep + __shfl_xor_sync(0xffffffffu, send, off);
          }
        }
        float total = dgs[0];
        const int per = 2 * off;                     // lanes that hold parts of one token
        for (; off; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
        if (lane % per == 0 && lane / per < left) qdg[lane / per * sdg] = from_f32<TG>(total);
      }
    }
  }
  if (given_up && threadIdx.x == 0 && p.status) atomicExch(p.status, VDN_ERR_TIMEOUT);
  if (p.last && rank == 0 && warp == 0 && live) {
    float e[VEC];
    from_lanes(carry, e);
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.last[seq * p.channels + c + v] = e[v];
  }
}

// One token per sequence (serving): h = a h + x, one thread per VEC channels.
template <typename T, typename TG, int VEC, bool SHARED>
__global__ void __launch_bounds__(256) step_kernel(const Params p, const int head_dim) {
  constexpr int GV = SHARED ? 1 : VEC;
  const int64_t per = p.channels / VEC;
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= per * p.seqs) return;
  const int64_t seq = n / per, c = (n - seq * per) * VEC;
  float x[VEC], g[GV], h[VEC];
  unpack<T, VEC>(*reinterpret_cast<const Raw<T, VEC>*>(static_cast<const T*>(p.x) + seq * p.x_batch + c), x);
  unpack<TG, GV>(*reinterpret_cast<const Raw<TG, GV>*>(static_cast<const TG*>(p.g) + seq * p.g_batch +
                                                       (SHARED ? c / head_dim : c)), g);
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float hi, lo;
    decay_pair(g[SHARED ? 0 : v], hi, lo);
    h[v] = p.first ? p.first[seq * p.channels + c + v] : 0.f;
    h[v] = fmaf(hi, h[v], fmaf(lo, h[v], x[v]));
  }
  *reinterpret_cast<Raw<T, VEC>*>(static_cast<T*>(p.out) + seq * p.out_batch + c) = pack<T, VEC>(h);
  if (p.last) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.last[seq * p.channels + c + v] = h[v];
  }
}

static int pow2_at_least(int64_t n, int most) {
  int v = 1;
  while (v < n && v < most) v *= 2;
  return v;
}

template <typename T, typename TG, int VEC, int L, bool BWD, bool SHARED>
static int launch(const Params& p, cudaStream_t stream) {
  // The typical length decides how many warps and CTAs share a sequence (a packed batch's
  // lengths live on the device: their mean stands for them).
  const int64_t len = p.cu ? (p.rows + p.seqs - 1) / p.seqs : (int64_t)p.rows;
  const int warps = pow2_at_least((len + L - 1) / L, MAX_WARPS);
  const int cluster = pow2_at_least((len + warps * L - 1) / (warps * L), MAX_CLUSTER);
  const int64_t ids = (p.seqs + (p.zero_tail ? 1 : 0)) * p.tiles;
  VDN_CHECK_ARG(ids * cluster < (1ll << 31), "too many sequences times channels for one launch");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ids * cluster));
  cfg.blockDim = dim3(warps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VDN_CUDA_TRY(cudaLaunchKernelEx(&cfg, scan_kernel<T, TG, VEC, L, BWD, SHARED>, p, cluster));
  return VDN_OK;
}

template <typename T, typename TG, bool BWD>
static int dispatch(Params& p, int shared_dim, cudaStream_t stream) {
  const bool step = !BWD && !p.cu && p.rows == 1;
  // Two channels per lane move whole 128-byte lines of 16-bit rows; a channel count,
  // stride or address that does not allow it takes one channel per lane.
  auto fits = [&](int vec) {
    const size_t ex = sizeof(T) * vec, eg = shared_dim ? sizeof(TG) : sizeof(TG) * vec;
    auto ok = [&](const void* q, int64_t row, int64_t batch, size_t e, size_t size) {
      return !q || (aligned_to(q, e) && row * size % e == 0 && batch * size % e == 0);
    };
    return p.channels % vec == 0 && ok(p.x, p.x_row, p.x_batch, ex, sizeof(T)) &&
           ok(p.g, p.g_row, p.g_batch, eg, sizeof(TG)) && ok(p.y_in, p.y_row, p.y_batch, ex, sizeof(T)) &&
           ok(p.out, p.out_row, p.out_batch, ex, sizeof(T)) && ok(p.dg, p.dg_row, p.dg_batch, eg, sizeof(TG));
  };
  if (step) {
    const bool two = fits(2) && (!shared_dim || shared_dim % 2 == 0);
    const int64_t n = p.seqs * p.channels / (two ? 2 : 1), blocks = (n + 255) / 256;
    VDN_CHECK_ARG(blocks < (1ll << 31), "too many sequences times channels for one launch");
    const unsigned grid = (unsigned)blocks;
    if (shared_dim) {
      if (two) step_kernel<T, TG, 2, true><<<grid, 256, 0, stream>>>(p, shared_dim);
      else step_kernel<T, TG, 1, true><<<grid, 256, 0, stream>>>(p, shared_dim);
    } else {
      if (two) step_kernel<T, TG, 2, false><<<grid, 256, 0, stream>>>(p, 1);
      else step_kernel<T, TG, 1, false><<<grid, 256, 0, stream>>>(p, 1);
    }
    VDN_LAUNCH_CHECK("gated scan step");
    return VDN_OK;
  }
  // Tokens a warp: as many as its registers hold (the backward keeps twice the arrays),
  // the same whatever the alignment, so that strides do not change the order of the sums.
  constexpr int L = BWD ? 8 : 16;
  if (shared_dim) {                                  // one head per tile
    const int vec = shared_dim / 32;
    VDN_CHECK_ARG(fits(vec), "a shared decay needs rows aligned to %d elements", vec);
    p.tiles = (int)(p.channels / shared_dim);
    if (vec == 4) return launch<T, TG, 4, L / 2, BWD, true>(p, stream);
    if (vec == 2) return launch<T, TG, 2, L, BWD, true>(p, stream);
    return launch<T, TG, 1, L, BWD, true>(p, stream);
  }
  const int vec = fits(2) ? 2 : 1;
  p.tiles = (int)((p.channels + 32 * vec - 1) / (32 * vec));
  if (vec == 2) return launch<T, TG, 2, L, BWD, false>(p, stream);
  return launch<T, TG, 1, L, BWD, false>(p, stream);
}

template <bool BWD>
static int run_typed(Params& p, int dtype, int g_dtype, int shared_dim, cudaStream_t stream) {
  if (dtype == VDN_DTYPE_F32) return dispatch<float, float, BWD>(p, shared_dim, stream);
  if (dtype == VDN_DTYPE_BF16) {
    if (g_dtype == VDN_DTYPE_F32) return dispatch<__nv_bfloat16, float, BWD>(p, shared_dim, stream);
    return dispatch<__nv_bfloat16, __nv_bfloat16, BWD>(p, shared_dim, stream);
  }
  if (g_dtype == VDN_DTYPE_F32) return dispatch<__half, float, BWD>(p, shared_dim, stream);
  return dispatch<__half, __half, BWD>(p, shared_dim, stream);
}

static int check(int dtype, int g_dtype, int64_t seqs, int64_t rows, int64_t heads, int64_t d, int shared,
                 std::initializer_list<int64_t> strides) {
  if (!dtype_known(dtype) || !dtype_known(g_dtype)) return set_error(VDN_ERR_TYPE, "unknown dtype code");
  if (g_dtype != dtype && g_dtype != VDN_DTYPE_F32)
    return set_error(VDN_ERR_TYPE, "log_decay must have x's dtype or be fp32");
  VDN_CHECK_ARG(seqs >= 0 && rows >= 0 && heads >= 1 && d >= 1, "bad scan extents");
  VDN_CHECK_ARG(rows < (1ll << 30) && heads < (1ll << 30) && d < (1ll << 30) && heads * d < (1ll << 30), "extents too large");
  for (int64_t s : strides)   // 32-bit offsets inside a warp's run of tokens
    VDN_CHECK_ARG(s > -(1ll << 26) && s < (1ll << 26), "row strides must lie below 2^26 elements");
  VDN_CHECK_ARG(!shared || d == 32 || d == 64 || d == 128,
                "a decay per head needs a head dim of 32, 64 or 128 (expand it per channel for others)");
  return VDN_OK;
}

}  // namespace gscan
}  // namespace vdn

using namespace vdn;

extern "C" int vdn_gated_scan(const void* x, int dtype, int64_t x_batch, int64_t x_row, const void* log_decay,
                              int g_dtype, int64_t g_batch, int64_t g_row, int shared, const float* state,
                              const int32_t* cu_seqlens, int64_t seqs, int64_t rows, int64_t heads, int64_t d,
                              int reverse, void* y, int64_t y_batch, int64_t y_row, int zero_tail,
                              float* out_state, int* status, cudaStream_t stream) {
  using namespace vdn::gscan;
  if (int rc = check(dtype, g_dtype, seqs, rows, heads, d, shared, {x_row, g_row, y_row})) return rc;
  if (seqs == 0 || (rows == 0 && !out_state)) return VDN_OK;
  VDN_CHECK_ARG((x && log_decay && y) || rows == 0, "null pointer");
  Params p = {};
  p.x = x;
  p.g = log_decay;
  p.out = y;
  p.first = state;
  p.last = out_state;
  p.cu = cu_seqlens;
  p.x_row = x_row;
  p.g_row = g_row;
  p.out_row = y_row;
  p.x_batch = x_batch;
  p.g_batch = g_batch;
  p.out_batch = y_batch;
  p.rows = (int)rows;
  p.seqs = seqs;
  p.channels = heads * d;
  p.reverse = reverse != 0;
  p.zero_tail = zero_tail && cu_seqlens;
  p.status = status;
  return run_typed<false>(p, dtype, g_dtype, shared ? (int)d : 0, stream);
}

extern "C" int vdn_gated_scan_backward(const void* dy, int dtype, int64_t dy_batch, int64_t dy_row,
                                       const void* log_decay, int g_dtype, int64_t g_batch, int64_t g_row,
                                       int shared, const void* y, int64_t y_batch, int64_t y_row,
                                       const float* state, const float* d_out_state, const int32_t* cu_seqlens,
                                       int64_t seqs, int64_t rows, int64_t heads, int64_t d, int reverse, void* dx,
                                       int64_t dx_batch, int64_t dx_row, void* dg, int64_t dg_batch, int64_t dg_row,
                                       int zero_tail, float* d_state, int* status, cudaStream_t stream) {
  using namespace vdn::gscan;
  if (int rc = check(dtype, g_dtype, seqs, rows, heads, d, shared, {dy_row, g_row, y_row, dx_row, dg_row})) return rc;
  if (seqs == 0 || (rows == 0 && !d_state)) return VDN_OK;
  VDN_CHECK_ARG((dy && log_decay && y && dx && dg) || rows == 0, "null pointer");
  Params p = {};
  p.x = dy;
  p.g = log_decay;
  p.y_in = y;
  p.out = dx;
  p.dg = dg;
  p.first = state;
  p.dlast = d_out_state;
  p.last = d_state;
  p.cu = cu_seqlens;
  p.x_row = dy_row;
  p.g_row = g_row;
  p.y_row = y_row;
  p.out_row = dx_row;
  p.dg_row = dg_row;
  p.x_batch = dy_batch;
  p.g_batch = g_batch;
  p.y_batch = y_batch;
  p.out_batch = dx_batch;
  p.dg_batch = dg_batch;
  p.rows = (int)rows;
  p.seqs = seqs;
  p.channels = heads * d;
  p.reverse = reverse != 0;
  p.zero_tail = zero_tail && cu_seqlens;
  p.status = status;
  return run_typed<true>(p, dtype, g_dtype, shared ? (int)d : 0, stream);
}
