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
//   * rows travel as tiles (L tokens of a warp's channels) by tensor-map copies, a round ahead,
//     and results leave the same way from the tile they replace: no addresses or predicates
//     per element (with plain loads the scan was bound by issue, half of it such overhead);
//   * a warp owns L tokens of 32 * VEC channels (lane = VEC neighbouring channels) and folds
//     them into (A, H), keeping for each token its state from zero and its reach, the
//     product of the decays so far; after the join its true states are state + reach * carry;
//   * a CTA of up to eight warps owns neighbouring runs, joined through shared memory;
//   * a cluster of up to eight CTAs owns neighbouring CTA runs and walks the sequence in
//     rounds.  Each CTA sends its pair into the others' shared memory with asynchronous
//     stores that count on their mbarriers: unlike a cluster barrier (whose release waits
//     for the round's output stores: 480 against 355 us on an early form of the forward
//     below) this orders nothing else.  No flags in global memory, no workspace, and the
//     order of every sum is fixed: the same bits on every run.
// Measured, 16 bits: 1 x 32760 x 5120 forward 270 us (3.7 TB/s), backward 330 (5.1 TB/s); seven
// packed sequences of 16389 x 5120 backward, an fp32 decay per head, 133 us (3.8 TB/s).  DRAM
// and issue slots are half idle: what bounds it is the latency of a round (two walks and the
// exchange) at the warps that registers and tiles allow.
//
// Numerics: states, folds and sums in fp32.  A decay close to 1 loses its distance from
// 1 when it is rounded to fp32 (a memory of n tokens then errs by n * 2^-25, and a constant decay errs
// the same way at every token), so exp(g) is kept as a pair hi + lo with 2^n as a common
// factor: hi = fp32(1 + e), lo = e - (hi - 1), e = expm1(r) with r = g - n ln 2 in [-0.35,
// 0.35] from a polynomial fitted at Chebyshev nodes (2.5e-8 relative).  It runs on packed
// fp32 pairs with no branch and no MUFU operation.  A run's A comes from the sum of its g where
// that lies in [-2, 2], else from the product of its decays (run_factor).  exp(g) is 0 below g = -87.7 and inf
// above 88.37.
#include <initializer_list>
#include <type_traits>

#include "train_common.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace vdn {
namespace gscan {

using namespace sm100;

constexpr int MAX_CLUSTER = 8;

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
// log decays as loaded, held in [-87.9, 88.75] (where two_to works); NaN stays NaN.  16-bit pairs
// are clamped in one instruction before they are widened.
__device__ __forceinline__ float clamp_decay(float g) {
  float r;
  asm("max.NaN.f32 %0, %1, 0fC2AFCCCD;\n\tmin.NaN.f32 %0, %0, 0f42B18000;" : "=f"(r) : "f"(g));
  return r;
}
__device__ __forceinline__ f2 clamp_decay(f2 g) {
  float a, b;
  f2_unpack(g, a, b);
  return f2_pack(clamp_decay(a), clamp_decay(b));
}
template <typename T> __device__ __forceinline__ uint32_t clamp_word(uint32_t w);
template <> __device__ __forceinline__ uint32_t clamp_word<float>(uint32_t w) {
  return __float_as_uint(clamp_decay(__uint_as_float(w)));
}
template <> __device__ __forceinline__ uint32_t clamp_word<__nv_bfloat16>(uint32_t w) {   // -88, 88.5
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\tmax.NaN.bf16x2 t, %1, %2;\n\tmin.NaN.bf16x2 %0, t, %3;\n\t}" : "=r"(r) : "r"(w), "r"(0xC2B0C2B0u), "r"(0x42B142B1u));
  return r;
}
template <> __device__ __forceinline__ uint32_t clamp_word<__half>(uint32_t w) {          // -87.875, 88.5
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\tmax.NaN.f16x2 t, %1, %2;\n\tmin.NaN.f16x2 %0, t, %3;\n\t}" : "=r"(r) : "r"(w), "r"(0xD57ED57Eu), "r"(0x55885588u));
  return r;
}
template <typename TG, int GV, typename V, int N>
__device__ __forceinline__ void unpack_decays(const Raw<TG, GV>& raw, V (&g)[N]) {
  if constexpr (GV * sizeof(TG) < 4) {
    float e[1];
    unpack<TG, 1>(raw, e);
    e[0] = clamp_decay(e[0]);
    to_lanes(e, g);
  } else {
    uint32_t w[GV * sizeof(TG) / 4];
    words(raw, w);
#pragma unroll
    for (auto& x : w) x = clamp_word<TG>(x);
    const auto held = join(w);
    unpack_lanes<TG, GV>(held, g);
  }
}

// exp(g) as hi + lo (see above), g clamped: n = round(g / ln 2) (by adding 1.5 * 2^23, whose neighbours lie 1
// apart), r = g - n ln 2 with ln 2 in two parts, 355 / 512 and the rest (W. J. Cody and W. Waite, Software Manual
// for the Elementary Functions, 1980, chapter 6), e = expm1(r).
template <typename V>
__device__ __forceinline__ void decay_pair(V g, V& hi, V& lo) {
  auto c = [](float v) { return vset(V{}, v); };
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
__device__ __forceinline__ V decay_of(V g) {         // of any g
  V hi, lo;
  decay_pair(clamp_decay(g), hi, lo);
  return vadd(hi, lo);
}

// The factor of a CTA's run from the sum s of its log decays or the product p of their hi parts.  The product
// errs by u a token (u = 2^-24), all in one direction where the decays are alike, and slow decays remember that over
// many runs; the sum's exponential errs by half a unit of s an addition, 32 u at s = -62, which tells where little
// of the carry is left.  At |s| = 2 the product's errors leave at most 256 u / (e^2 - 1) = 40 u in a stationary state.
// A product of 0 stands: some decay was 0 (the sum holds it as -87.9, and growth beside it would cancel that).
__device__ __forceinline__ float run_factor(float s, float p, float e) { return fabsf(s) <= 2.f && p != 0.f ? e : p; }
__device__ __forceinline__ float run_factor(float s, float p) { return run_factor(s, p, decay_of(s)); }
__device__ __forceinline__ f2 run_factor(f2 s, f2 p) {
  float s0, s1, p0, p1, e0, e1;
  f2_unpack(s, s0, s1);
  f2_unpack(p, p0, p1);
  f2_unpack(decay_of(s), e0, e1);
  return f2_pack(run_factor(s0, p0, e0), run_factor(s1, p1, e1));
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

// Where a warp's rows come from: ROWS_LOAD plain loads into registers (any stride and alignment);
// ROWS_UP / ROWS_DOWN tensor-map copies into a ring of tiles in shared memory, token rows
// ascending or descending along the walk.
enum { ROWS_LOAD = 0, ROWS_UP = 1, ROWS_DOWN = 2 };
constexpr int kStages = 2;

struct Maps {
  CUtensorMap x, g, y, out, dg;
};

template <typename T, typename TG, int VEC, int L, bool BWD, bool SHARED>
constexpr int tile_bytes() {   // of one warp and stage: x (dy), the saved y, the decays
  return 32 * VEC * L * ((BWD ? 2 : 1) * (int)sizeof(T) + (SHARED ? 0 : (int)sizeof(TG)));
}

// Tokens a warp.  Runs of 32 keep all their arrays in up to 255 registers and halve the rounds,
// each of which costs a warp some 250 instructions beside its tokens'; runs of 16 leave room
// for more warps.  The same for both ways to load rows, so that strides do not change the order of
// the sums as long as a lane keeps its two channels.
constexpr int kRun = 16, kLongRun = 32;      // half of that where a lane has four channels
template <int VEC, int L> constexpr bool long_run() { return L * (VEC == 4 ? 2 : 1) >= kLongRun; }

// Warps a CTA, at most.  Runs of 16: the backward per channel keeps the most tiles, so that
// eight warps would leave one CTA an SM (480 us against 327 on a 1 x 32760 x 5120 backward).
// Runs of 32: as many as fit the shared memory beside the kernel's fixed arrays.
template <typename T, typename TG, int VEC, int L, bool BWD, bool SHARED>
constexpr int max_warps() {
  if (!long_run<VEC, L>()) return BWD && !SHARED ? 4 : 8;
  constexpr int line = Lanes<VEC>::N * 32 * (int)sizeof(Fold<typename Lanes<VEC>::V>);
  int w = 8;   // folds of two rounds, of the cluster's CTAs, and sums
  while (w > 1 && w * kStages * tile_bytes<T, TG, VEC, L, BWD, SHARED>() + (3 * w + 2 * MAX_CLUSTER) * line + 1024 > 227 * 1024)
    w /= 2;
  return w;
}

// Packed sequences start longest first, so that more CTAs a sequence pay although they do not all
// fit the GPU at once (7 random cuts of 16389 x 5120 backward, shared decays: 205 us as one wave
// of clusters of two, 150 as three waves of clusters of three).  The turn-th longest; each
// lane ranks one, hence at most 32.
constexpr int kSorted = 32;
__device__ __forceinline__ int longest_first(const Params& p, int turn, int lane) {
  const int seqs = (int)p.seqs;
  int len = -1, place = 0;
  if (lane < seqs) len = max(min(p.cu[lane + 1], p.rows) - min(max(p.cu[lane], 0), p.rows), 0);
  for (int j = 0; j < seqs; ++j) {
    const int other = __shfl_sync(0xffffffffu, len, j);
    place += other > len || (other == len && j < lane);
  }
  return __ffs(__ballot_sync(0xffffffffu, lane < seqs && place == turn)) - 1;
}

template <typename T, typename TG, int VEC, int L, bool BWD, bool SHARED, int FROM>
__global__ void __launch_bounds__(max_warps<T, TG, VEC, L, BWD, SHARED>() * 32, long_run<VEC, L>() ? 1 : BWD && !SHARED ? 3 : 2)
    scan_kernel(const Params p, const int cluster, const __grid_constant__ Maps maps) {
  constexpr int GV = SHARED ? 1 : VEC;               // decays per lane and token
  constexpr int TILE = 32 * VEC, MAX_WARPS = max_warps<T, TG, VEC, L, BWD, SHARED>();
  constexpr bool RING = FROM != ROWS_LOAD;
  using RX = Raw<T, VEC>;
  using RG = Raw<TG, GV>;
  using V = typename Lanes<VEC>::V;                  // values
  using G = typename Lanes<GV>::V;                   // decays
  constexpr int NV = Lanes<VEC>::N, NG = Lanes<GV>::N;
  extern __shared__ __align__(128) uint8_t tiles[];  // RING: [warps][kStages][tile_bytes]
  __shared__ Fold<V> folds[2][MAX_WARPS][NV][32];
  __shared__ G sums[2][MAX_WARPS][NG][32];
  __shared__ Fold<V> runs[2][MAX_CLUSTER][NV][32];   // one line from every CTA of the cluster
  __shared__ uint64_t arrived[2], full[MAX_WARPS][kStages];
  __shared__ int given_up;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int rank = (int)cluster_ctarank();
  const int64_t id = blockIdx.x / cluster;           // sequence-major, channel tiles fastest
  const int64_t turn = id / p.tiles;
  const int tile = (int)(id - turn * p.tiles);
  const int64_t seq = p.cu && p.seqs <= kSorted && turn < p.seqs ? longest_first(p, (int)turn, lane) : turn;
  const int64_t c = (int64_t)tile * TILE + lane * VEC;
  const bool live = c < p.channels;
  const bool whole = (int64_t)(tile + 1) * TILE <= p.channels;
  const int64_t gc = SHARED ? tile : c;              // shared: one head is one tile

  int begin = 0, len = p.rows;
  if (p.cu) {
    const int lo = seq < p.seqs ? p.cu[seq] : p.cu[p.seqs];
    const int hi = seq < p.seqs ? p.cu[seq + 1] : p.rows;
    begin = min(max(lo, 0), p.rows);                 // offsets out of range stay inside the tensors
    len = max(min(hi, p.rows) - begin, 0);
  }
  if (seq >= p.seqs) {                               // rows in front of the first sequence and behind the last
    const int head = min(min(max(p.cu[0], 0), p.rows), begin);
    for (int64_t i = rank * warps + warp; i < head + len; i += warps * cluster) {
      const int64_t t = i < head ? i - begin : i - head;
      if (live) *reinterpret_cast<RX*>(static_cast<T*>(p.out) + (begin + t) * p.out_row + c) = raw_zero<RX>();
      if (BWD && (SHARED ? lane == 0 : live))
        *reinterpret_cast<RG*>(static_cast<TG*>(p.dg) + (begin + t) * p.dg_row + gc) = raw_zero<RG>();
    }
    return;                                          // the whole cluster is here
  }

  // Walk order: the forward follows the recurrence, the backward its reverse.
  const bool down = RING ? FROM == ROWS_DOWN : p.reverse != BWD;   // token rows descend along the walk
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

  const int round_tokens = cluster * warps * L;
  int64_t i0 = (rank * warps + warp) * L;

  // Tiles: x, then the saved y, then the decays; a lane's VEC values of token row r at r * pitch.
  constexpr int PX = TILE * sizeof(T), PG = TILE * sizeof(TG), BYTES = tile_bytes<T, TG, VEC, L, BWD, SHARED>();
  uint8_t* ring = tiles + warp * kStages * BYTES;
  auto copy = [&](int stage, int64_t i) {            // one lane: the rows of walk tokens i .. i + L - 1
    if (i >= len) return;
    const int r = (int)(down ? row0 - i - (L - 1) : row0 + i), x0 = tile * TILE;
    uint8_t* to = ring + stage * BYTES;
    uint64_t* bar = &full[warp][stage];
    mbar_arrive_expect_tx(bar, BYTES);
    tma_load_3d(to, &maps.x, bar, x0, r, (int)b);
    if (BWD) tma_load_3d(to + L * PX, &maps.y, bar, x0, r + sgn, (int)b);   // the tokens before them
    if (!SHARED) tma_load_3d(to + (BWD ? 2 : 1) * L * PX, &maps.g, bar, x0, r, (int)b);
  };

  if (threadIdx.x == 0) {
    mbar_init(&arrived[0], 1);
    mbar_init(&arrived[1], 1);
    if (RING)
      for (int w = 0; w < warps; ++w)
        for (int s = 0; s < kStages; ++s) mbar_init(&full[w][s], 1);
    given_up = 0;
    fence_barrier_init();
  }
  cluster_sync();                                    // the barriers stand before anyone sends
  if (RING && lane == 0)
    for (int s = 0; s < kStages - 1; ++s) copy(s, i0 + (int64_t)s * round_tokens);

  RX rx[RING ? 1 : L], ry[!RING && BWD ? L : 1];
  RG rg[RING || SHARED ? 1 : L];
  auto load = [&](int64_t i) {                       // ROWS_LOAD: a round's rows into registers
    const T* qx = px + i * sx;
    const TG* qg = pg + i * sg;
    const int n = live ? (int)min((int64_t)len - i, (int64_t)L) : 0;
#pragma unroll
    for (int l = 0; l < L; ++l) {
      rx[RING ? 0 : l] = l < n ? load_once<RX>(qx + l * sx) : raw_zero<RX>();
      if (!SHARED) rg[RING || SHARED ? 0 : l] = l < n ? load_once<RG>(qg + l * sg) : raw_zero<RG>();
    }
    if constexpr (BWD) {
      const T* qy = py + (i + 1) * sy;
      const int ny = i + n == len ? n - 1 : n;       // the oldest token's h_{t-1} is the first state
#pragma unroll
      for (int l = 0; l < L; ++l) ry[RING ? 0 : l] = l < ny ? load_once<RX>(qy + l * sy) : raw_zero<RX>();
    }
  };
  // Shared decays: lane l has token l's, one round ahead.
  auto load_shared = [&](int64_t i) {
    const bool in = lane < L && i + lane < len;
    float e[1] = {0.f};
    if (in) unpack<TG, 1>(*reinterpret_cast<const Raw<TG, 1>*>(pg + (i + lane) * sg), e);
    return e[0];
  };
  float g_next = SHARED ? load_shared(i0) : 0.f;

  int buf = 0, stage = 0;
  uint32_t phase = 0, full_phase = 0;
  for (int64_t done = 0; done < len; done += round_tokens, i0 += round_tokens, buf ^= 1) {
    const int n = (int)min((int64_t)len - i0, (int64_t)L);   // this warp's tokens; none or fewer at the end
    const bool last_run = (int64_t)len - i0 <= L;    // the oldest token is among them (or none is)
    int ok = 1;
    uint8_t* at = ring + stage * BYTES + lane * (VEC * (int)sizeof(T));
    uint8_t* at_g = ring + stage * BYTES + (BWD ? 2 : 1) * L * PX + lane * (GV * (int)sizeof(TG));
    auto row = [](int l) { return FROM == ROWS_DOWN ? L - 1 - l : l; };
    auto x_at = [&](int l) { return reinterpret_cast<RX*>(at + row(l) * PX); };
    auto y_at = [&](int l) { return reinterpret_cast<RX*>(at + (L + row(l)) * PX); };
    auto g_at = [&](int l) { return reinterpret_cast<RG*>(at_g + row(l) * PG); };
    if constexpr (RING) {
      if (n > 0) {
        ok = mbar_wait(&full[warp][stage], full_phase, &given_up);
        if (n < L) {                                 // rows of other sequences, or of none
#pragma unroll
          for (int l = 0; l < L; ++l)
            if (l >= n) {
              *x_at(l) = raw_zero<RX>();
              if (!SHARED) *g_at(l) = raw_zero<RG>();
            }
        }
      }
    } else {
      load(i0);
    }

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
    float hi_lane = 1.f, lo_lane = 0.f;
    if constexpr (SHARED) {
      float s = clamp_decay(g_next);                 // not at the load: nothing waits for it there
      decay_pair(s, hi_lane, lo_lane);
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      sum[0] = vset(G{}, s);
      g_next = load_shared(i0 + round_tokens);
    }
    if (!RING || n > 0) {
#pragma unroll
      for (int l = 0; l < L; ++l) {
        V x[NV];
        G g[NG], hi[NG], lo[NG];
        unpack_lanes<T, VEC>(RING ? *x_at(l) : rx[RING ? 0 : l], x);
        if constexpr (SHARED) {
          hi[0] = vset(G{}, __shfl_sync(0xffffffffu, hi_lane, l));
          lo[0] = vset(G{}, __shfl_sync(0xffffffffu, lo_lane, l));
        } else {
          unpack_decays<TG, GV>(RING ? *g_at(l) : rg[RING || SHARED ? 0 : l], g);
        }
#pragma unroll
        for (int v = 0; v < NG; ++v) {
          if constexpr (!SHARED) {
            decay_pair(g[v], hi[v], lo[v]);
            sum[v] = vadd(sum[v], g[v]);
          }
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
    }
    if (RING && lane == 0) {                         // refill the stage before, once its results have left it
      bulk_wait_group_read<0>();
      copy(stage ? stage - 1 : kStages - 1, i0 + (int64_t)(kStages - 1) * round_tokens);
    }

    // Join the warps of the CTA: `before` is the fold of the warps in front of this one.
    // (Inside a round the product of the run's decays will do; run_factor chooses for the long chain.)
    Fold<V> own[NV], before[NV];
#pragma unroll
    for (int v = 0; v < NG; ++v) sums[buf][warp][v][lane] = sum[v];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      spread(far[SHARED ? 0 : v], own[v].a);
      own[v].h = fold[v];
      folds[buf][warp][v][lane] = own[v];
      before[v].a = vset(V{}, 1.f);
      before[v].h = vset(V{}, 0.f);
    }
    if (!__syncthreads_and(ok && !given_up)) break;  // a wait that gave up ends the whole CTA
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
      for (int v = 0; v < NV; ++v) {
        Fold<V> f;
        if constexpr (SHARED) {
          float p;                                   // one decay for the whole head
          if constexpr (std::is_same<V, float>::value) {
            p = before[v].a * own[v].a;
          } else {
            float unused;
            f2_unpack(vmul(before[v].a, own[v].a), p, unused);
          }
          spread(run_factor(s[0], p), f.a);
        } else {
          f.a = run_factor(s[v], vmul(before[v].a, own[v].a));
        }
        f.h = vfma(own[v].a, before[v].h, own[v].h);
        for (int r = 0; r < cluster; ++r)
          send(mapa_shared(&runs[buf][rank][v][lane], r), f, mapa_shared(&arrived[buf], r));
      }
      if (lane == 0) mbar_arrive_expect_tx(&arrived[buf], cluster * (uint32_t)sizeof(runs[0][0]));
    }
    // A line's buffer is written again two rounds later, by CTAs that have this one's next
    // line, which it sends after all its warps have read this round's.
    mbar_wait(&arrived[buf], phase, &given_up);      // a failure ends the loop at the next round's barrier
    phase ^= buf;
    V in[NV];                                        // the true carry in front of this warp
    const Fold<V>(*line)[NV][32] = &runs[buf][0];
    auto pass = [&](int from, int to) {
      for (int r = from; r < to; ++r)
#pragma unroll
        for (int v = 0; v < NV; ++v) carry[v] = vfma(line[r][v][lane].a, carry[v], line[r][v][lane].h);
    };
    pass(0, rank);
#pragma unroll
    for (int v = 0; v < NV; ++v) in[v] = vfma(before[v].a, carry[v], before[v].h);
    pass(rank, cluster);

    // Second walk, with the true carry.  A whole run of a ring takes the place of its inputs
    // and leaves as it came; others are stored row by row.
    T* qo = po + i0 * so;
    TG* qdg = BWD ? pdg + i0 * sdg : nullptr;
    float dgs[BWD && SHARED ? L : 1];
    auto walk = [&](auto all, auto tile_out) {
      V c0[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v) c0[v] = in[v];
#pragma unroll
      for (int l = 0; l < L; ++l) {
        V y[NV];
        const bool store = all.value || (live && l < n);
        if constexpr (!BWD) {
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            V r;
            spread(reach[l][SHARED ? 0 : v], r);
            y[v] = vfma(r, in[v], part[l][v]);
          }
          if constexpr (tile_out.value) *x_at(l) = pack_lanes<T, VEC>(y);
          else if (store) store_once(qo + l * so, pack_lanes<T, VEC>(y));
        } else {
          V u[NV], d[NV];
          unpack_lanes<T, VEC>(RING ? *y_at(l) : ry[RING ? 0 : l], y);
          if (!all.value && last_run && l + 1 == n) {        // the oldest token
            float e[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) e[v] = p.first && live ? p.first[seq * p.channels + c + v] : 0.f;
            to_lanes(e, y);
          }
          unpack_lanes<T, VEC>(RING ? *x_at(l) : rx[RING ? 0 : l], u);
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            V r;
            spread(reach[l][SHARED ? 0 : v], r);
            u[v] = vadd(u[v], c0[v]);
            c0[v] = vfma(r, in[v], part[l][v]);
            d[v] = vmul(c0[v], y[v]);
          }
          if constexpr (tile_out.value) *x_at(l) = pack_lanes<T, VEC>(u);
          else if (store) store_once(qo + l * so, pack_lanes<T, VEC>(u));
          if constexpr (SHARED) {
            float e[VEC];
            from_lanes(d, e);
            float t = e[0];
#pragma unroll
            for (int v = 1; v < VEC; ++v) t += e[v];
            dgs[SHARED ? l : 0] = t;
          } else {
            if constexpr (tile_out.value) *g_at(l) = pack_lanes<TG, VEC>(d);
            else if (store) store_once(qdg + l * sdg, pack_lanes<TG, VEC>(d));
          }
        }
      }
    };
    if constexpr (RING) {
      if (n == L && !(BWD && last_run)) {
        walk(std::true_type{}, std::true_type{});
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          const int r = (int)(down ? row0 - i0 - (L - 1) : row0 + i0), x0 = tile * TILE;
          uint8_t* from = ring + stage * BYTES;
          tma_store_3d(&maps.out, from, x0, r, (int)b);
          if (BWD && !SHARED) tma_store_3d(&maps.dg, from + 2 * L * PX, x0, r, (int)b);
          bulk_commit_group();
        }
      } else if (n > 0) {
        walk(std::false_type{}, std::false_type{});
      }
    } else {
      if (whole && n == L && !(BWD && last_run)) walk(std::true_type{}, std::false_type{});
      else walk(std::false_type{}, std::false_type{});
    }
    if constexpr (BWD && SHARED) {
      // Sum each token's terms over the head: the first rounds halve the tokens a lane
      // holds while they halve the lanes, so L sums cost about L + 5 shuffles.
      if (n > 0) {
        constexpr int per = 32 / L;                  // lanes that end with parts of one token
        int off = 16;
#pragma unroll
        for (int m = L; m > 1; m >>= 1, off >>= 1) {
          const bool up = lane & off;
#pragma unroll
          for (int j = 0; j < m / 2; ++j) {
            const float give = up ? dgs[j] : dgs[j + m / 2], keep = up ? dgs[j + m / 2] : dgs[j];
            dgs[j] = keep + __shfl_xor_sync(0xffffffffu, give, off);
          }
        }
        float total = dgs[0];
        for (; off; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
        if (lane % per == 0 && lane / per < n) qdg[lane / per * sdg] = from_f32<TG>(total);
      }
    }
    if (++stage == kStages) {
      stage = 0;
      full_phase ^= 1;
    }
  }
  if (RING && lane == 0) {
    if (given_up) {                                  // copies that were issued land before the CTA exits
      const uint64_t t0 = globaltimer();
      for (int s = 0; s < kStages && i0 < len; ++s, i0 += round_tokens) {
        while (!mbar_try_wait(&full[warp][stage], full_phase) && globaltimer() - t0 < kWaitLimitNs) {
        }
        if (++stage == kStages) {
          stage = 0;
          full_phase ^= 1;
        }
      }
    }
    bulk_wait_group<0>();                            // results are written before the CTA exits
  }
  if (given_up && threadIdx.x == 0 && p.status) atomicExch(p.status, VDN_ERR_TIMEOUT);
  if (p.last && rank == 0 && warp == 0 && live) {
    float e[VEC];
    from_lanes(carry, e);
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.last[seq * p.channels + c + v] = e[v];
  }
  __syncwarp();
  cluster_sync();                                    // nobody leaves while lines may still be sent to it
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
    decay_pair(clamp_decay(g[SHARED ? 0 : v]), hi, lo);
    h[v] = p.first ? p.first[seq * p.channels + c + v] : 0.f;
    h[v] = fmaf(hi, h[v], fmaf(lo, h[v], x[v]));
  }
  *reinterpret_cast<Raw<T, VEC>*>(static_cast<T*>(p.out) + seq * p.out_batch + c) = pack<T, VEC>(h);
  if (p.last) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.last[seq * p.channels + c + v] = h[v];
  }
}

template <int MOST>
static int pow2_at_least(int64_t n) {                // the least power of two >= n, at most MOST
  static_assert(MOST > 0 && (MOST & (MOST - 1)) == 0, "a power of two bounds a power of two");
  int v = 1;
  while (v < n && v < MOST) v *= 2;
  return v;
}

template <typename T>
static CUtensorMapDataType map_type() {
  return sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
         : std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}
// Boxes of `tokens` rows x `tile` channels over [batches, rows, channels].
template <typename T>
static int rows_map(CUtensorMap* map, const void* base, int64_t channels, int64_t rows, int64_t batches, int64_t row,
                    int64_t batch, int tile, int tokens) {
  const int64_t one = (channels * (int64_t)sizeof(T) + 15) / 16 * 16;   // a stride that no index multiplies
  cuuint64_t dims[3] = {(cuuint64_t)channels, (cuuint64_t)rows, (cuuint64_t)batches};
  cuuint64_t strides[2] = {(cuuint64_t)(row ? row * (int64_t)sizeof(T) : one),
                           (cuuint64_t)(batch ? batch * (int64_t)sizeof(T) : one)};
  cuuint32_t box[3] = {(cuuint32_t)tile, (cuuint32_t)tokens, 1};
  return encode_map_swizzle(map, map_type<T>(), 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}
template <typename T>
static bool map_takes(const void* base, int64_t rows, int64_t batches, int64_t row, int64_t batch) {
  return aligned16(base) && row * (int64_t)sizeof(T) % 16 == 0 && batch * (int64_t)sizeof(T) % 16 == 0 &&
         (rows == 1 || row > 0) && (batches == 1 || batch > 0);
}

constexpr int kDevices = 64;

// Raises the kernel's shared-memory limit, once per device.
template <typename T, typename TG, int VEC, int L, bool BWD, bool SHARED, int FROM>
static int prepare(int& dev) {
  constexpr int bytes = FROM == ROWS_LOAD ? 0 : kStages * tile_bytes<T, TG, VEC, L, BWD, SHARED>();
  static bool set[kDevices] = {};
  VDN_CUDA_TRY(cudaGetDevice(&dev));
  VDN_CHECK_ARG(dev >= 0 && dev < kDevices, "device index out of range");
  if (bytes && !set[dev]) {
    VDN_CUDA_TRY(cudaFuncSetAttribute(scan_kernel<T, TG, VEC, L, BWD, SHARED, FROM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      max_warps<T, TG, VEC, L, BWD, SHARED>() * bytes));
    set[dev] = true;
  }
  return VDN_OK;
}

template <typename T, typename TG, int VEC, int L, bool BWD, bool SHARED, int FROM>
static void configure(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, int64_t blocks, int warps, int cluster) {
  constexpr int bytes = FROM == ROWS_LOAD ? 0 : kStages * tile_bytes<T, TG, VEC, L, BWD, SHARED>();
  cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(warps * 32);
  cfg.dynamicSmemBytes = warps * bytes;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
}

// Warps a CTA and CTAs a cluster.  More CTAs on a sequence shorten its walk, but a grid that does
// not fit the GPU at once runs in waves, the last perhaps nearly empty (80 tiles of 32760 tokens,
// four warps a CTA and 16 tokens a warp: 305 us with clusters of 8, which need 640 places where
// there are 592, and 282 us with 5), and every CTA starts up anew.  Measured over clusters of one
// to eight, CTAs of two, four and eight warps and nine shapes, a round takes about as long as
// 1 + (the warps on the fullest SM) / 4, and starting up as two rounds; choosing by that was
// within a tenth of the best of them.  Shared decays cost one evaluation per token instead of
// one per element: 2 + .. / 4.  Runs of 32 take (2 + the warps) / 4, each scheduler's warps
// counting as its fullest one's, and no less than 6 / 4: a CTA of six warps on four schedulers
// takes eight warps' time.  The ring kernel's places decide for both kernels, so that rows which tensor
// maps cannot take are summed in the same order; rows that start at an odd element take one channel a
// lane, and with it a shape of their own.
template <typename T, typename TG, int VEC, int L, bool BWD, bool SHARED>
static int choose_shape(int64_t mean, int64_t longest, int64_t seqs, bool sorted, int64_t tiles, int& warps, int& cluster) {
  constexpr int FROM = VEC > 1 || SHARED ? ROWS_UP : ROWS_LOAD;
  static int places[kDevices][4][MAX_CLUSTER + 1] = {};
  int dev = 0;
  if (int rc = prepare<T, TG, VEC, L, BWD, SHARED, FROM>(dev)) return rc;
  warps = pow2_at_least<max_warps<T, TG, VEC, L, BWD, SHARED>()>((longest + L - 1) / L);
  cluster = 1;
  const int64_t ids = seqs * tiles;
  int64_t best = -1;
  const int most = warps;
  for (int w = most; w == most || w >= (long_run<VEC, L>() ? 2 : 4); w /= 2) {
    const int64_t runs = (mean + w * L - 1) / (w * L), most_runs = (longest + w * L - 1) / (w * L);
    for (int c = 1; c <= MAX_CLUSTER && c <= (most_runs > 1 ? most_runs : 1); ++c) {
      int& fit = places[dev][w == 8 ? 3 : w >> 1][c];   // clusters resident at once
      if (!fit) {
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr[1];
        configure<T, TG, VEC, L, BWD, SHARED, FROM>(cfg, attr, 148 * 64 / c * c, w, c);
        int n = 0;
        VDN_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, scan_kernel<T, TG, VEC, L, BWD, SHARED, FROM>, &cfg));
        fit = n > 0 ? n : 1;
      }
      const int64_t waves = (ids + fit - 1) / fit, tail = ids - (waves - 1) * fit;
      auto load = [&](int64_t clusters) {
        const int64_t on_sm = w * ((clusters * c + 147) / 148);
        if (!long_run<VEC, L>()) return (SHARED ? 8 : 4) + on_sm;
        const int64_t t = 2 + (on_sm + 3) / 4 * 4;
        return t > 6 ? t : 6;
      };
      const int64_t walk = (runs + c - 1) / c, longest_walk = (most_runs + c - 1) / c;
      int64_t t = (walk + 2) * ((waves - 1) * load(fit) + load(tail));
      if (sorted && waves > 1) {                     // the longest start first, the others fill the places behind
        const int64_t first = (longest_walk + 2) * load(fit);
        t = (walk + 2) * load(fit) * ids / fit;
        if (t < first) t = first;
      } else {
        t += (longest_walk - walk) * load(tiles);    // the longest sequences' tiles go on alone
      }
      if (best < 0 || t < best) {
        best = t;
        warps = w;
        cluster = c;
      }
    }
  }
  return VDN_OK;
}

template <typename T, typename TG, int VEC, int L, bool BWD, bool SHARED, int FROM>
static int launch_from(const Params& p, int warps, int cluster, const Maps& maps, cudaStream_t stream) {
  const int64_t ids = (p.seqs + (p.zero_tail ? 1 : 0)) * p.tiles;
  VDN_CHECK_ARG(ids * cluster < (1ll << 31), "too many sequences times channels for one launch");
  int dev = 0;
  if (int rc = prepare<T, TG, VEC, L, BWD, SHARED, FROM>(dev)) return rc;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[1];
  configure<T, TG, VEC, L, BWD, SHARED, FROM>(cfg, attr, ids * cluster, warps, cluster);
  cfg.stream = stream;
  VDN_CUDA_TRY(cudaLaunchKernelEx(&cfg, scan_kernel<T, TG, VEC, L, BWD, SHARED, FROM>, p, cluster, maps));
  return VDN_OK;
}

static int64_t mean_length(const Params& p) {
  return p.cu ? (p.rows + p.seqs - 1) / p.seqs : (int64_t)p.rows;
}

template <typename T, typename TG, int VEC, int L, bool BWD, bool SHARED>
static int launch(const Params& p, cudaStream_t stream) {
  // A packed batch's lengths live on the device.  Their mean stands for most of them, and random
  // cuts make the longest somewhat above 1 + ln(sequences) times as long.
  const int64_t len = mean_length(p);
  int64_t longest = len;
  if (p.cu) {
    for (int64_t s = p.seqs; s > 1; s /= 2) longest += len * 17 / 20;
    if (longest > p.rows) longest = p.rows;
  }
  int warps = 1, cluster = 1;
  if (int rc = choose_shape<T, TG, VEC, L, BWD, SHARED>(len, longest, p.seqs, p.cu && p.seqs <= kSorted, p.tiles, warps, cluster)) return rc;
  Maps maps = {};
  // Tiles of whole runs pay from two runs a sequence on; shorter ones would mostly copy others' rows.
  if constexpr (VEC > 1 || SHARED) {
    const int64_t batches = p.cu ? 1 : p.seqs, rows = p.rows;
    const bool ring = len >= 2 * L && map_takes<T>(p.x, rows, batches, p.x_row, p.x_batch) &&
                      (SHARED || map_takes<TG>(p.g, rows, batches, p.g_row, p.g_batch)) &&
                      map_takes<T>(p.out, rows, batches, p.out_row, p.out_batch) &&
                      (!BWD || map_takes<T>(p.y_in, rows, batches, p.y_row, p.y_batch)) &&
                      (!BWD || SHARED || map_takes<TG>(p.dg, rows, batches, p.dg_row, p.dg_batch));
    if (ring) {
      const int64_t c = p.channels;
      if (int rc = rows_map<T>(&maps.x, p.x, c, rows, batches, p.x_row, p.x_batch, 32 * VEC, L)) return rc;
      if (int rc = rows_map<T>(&maps.out, p.out, c, rows, batches, p.out_row, p.out_batch, 32 * VEC, L)) return rc;
      if (!SHARED)
        if (int rc = rows_map<TG>(&maps.g, p.g, c, rows, batches, p.g_row, p.g_batch, 32 * VEC, L)) return rc;
      if (BWD)
        if (int rc = rows_map<T>(&maps.y, p.y_in, c, rows, batches, p.y_row, p.y_batch, 32 * VEC, L)) return rc;
      if (BWD && !SHARED)
        if (int rc = rows_map<TG>(&maps.dg, p.dg, c, rows, batches, p.dg_row, p.dg_batch, 32 * VEC, L)) return rc;
      if (p.reverse != BWD) return launch_from<T, TG, VEC, L, BWD, SHARED, ROWS_DOWN>(p, warps, cluster, maps, stream);
      return launch_from<T, TG, VEC, L, BWD, SHARED, ROWS_UP>(p, warps, cluster, maps, stream);
    }
  }
  return launch_from<T, TG, VEC, L, BWD, SHARED, ROWS_LOAD>(p, warps, cluster, maps, stream);
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
  if (shared_dim) {                                  // one head per tile
    const int vec = shared_dim / 32;
    VDN_CHECK_ARG(fits(vec), "a shared decay needs rows aligned to %d elements", vec);
    p.tiles = (int)(p.channels / shared_dim);
    // Long runs as below, us without and with: 4 tiles of 16384 x 128 81 and 48 (backward 95 and 58),
    // 16 tiles 97 and 87 (117 and 101), 80 tiles of 16384 x 64 123 and 155 (153 and 183).
    const bool few = p.seqs * p.tiles <= 37 && mean_length(p) >= 1024;
    if (vec == 4 && few) return launch<T, TG, 4, kLongRun / 2, BWD, true>(p, stream);
    if (vec == 4) return launch<T, TG, 4, kRun / 2, BWD, true>(p, stream);
    if (vec == 2 && few) return launch<T, TG, 2, kLongRun, BWD, true>(p, stream);
    if (vec == 2) return launch<T, TG, 2, kRun, BWD, true>(p, stream);
    if (few) return launch<T, TG, 1, kLongRun, BWD, true>(p, stream);
    return launch<T, TG, 1, kRun, BWD, true>(p, stream);
  }
  const int vec = fits(2) ? 2 : 1;
  p.tiles = (int)((p.channels + 32 * vec - 1) / (32 * vec));
  // Long runs where tiles are few and sequences long, so that a round's latency counts and not
  // the number of warps: us with 16 and 32 tokens a warp, 16-bit rows of 1 x 16384 x 512 (8 tiles)
  // 46 and 34 (backward 71 and 41), 1 x 32760 x 5120 (80) 288 and 272 (327 and 348), 64 x 512 x
  // 5120 (5120) 223 and 233 (317 and 390), 2 x 500 x 512 (16) 8 and 8 (8 and 10).  Widths that
  // tensor maps cannot take keep to 16 (3 x 1001 x 515 in fp32: 13 and 21, 19 and 29).
  const bool few = p.seqs * ((p.channels + 63) / 64) <= (BWD ? 37 : 148) && mean_length(p) >= 1024 && p.channels % 8 == 0;
  if (vec == 2 && few) return launch<T, TG, 2, kLongRun, BWD, false>(p, stream);
  if (vec == 2) return launch<T, TG, 2, kRun, BWD, false>(p, stream);
  if (few) return launch<T, TG, 1, kLongRun, BWD, false>(p, stream);
  return launch<T, TG, 1, kRun, BWD, false>(p, stream);
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
