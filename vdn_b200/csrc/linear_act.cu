// Linear layer with bias, activation and residual in its epilogue, and its gradients, on
// tcgen05 (16-bit operands, fp32 accumulation), sm_100a.
//
//   forward   z = x w^T + b,  pre = z (optional output),  y = act(z) + residual
//   backward  dz = dy act'(pre),  db = sum_rows dz,  dx = dz w,  dw = dz^T x
//
// All three products are D[i, j] = sum_r P[i, r] Q[j, r] with each operand either r-contiguous
// (K-major) or i/j-contiguous (MN-major, read by the tensor cores as it lies): forward
// K/K, dx K/MN, dw MN/MN.  No operand is transposed in memory.
//
//   * pair kernel: 256 x 256 tiles on a cluster of two CTAs (cta_group::2).  Each CTA stages
//     its 128 rows of P and its 128-row half of Q per 64-deep block (six stages of 32 KB);
//     the even CTA's MMA warp issues 256 x 256 x 16 products into one of two TMEM
//     accumulators, so that eight epilogue warps work on a tile while the next one runs.
//     Bound by the tensor pipe for deep products (32760 x 5120 x 5120: 1123 to 1265 us with
//     the clocks under load, 1.36 to 1.53 PFLOP/s, as torch's own), by its epilogue for
//     shallow ones.
//   * narrow kernel: 128 features x up to 128 tokens per CTA with the features on the MMA's M
//     side, for outputs too small to fill the GPU with pair tiles (few tokens: the weight's
//     bytes are the bound).  A cluster of up to eight CTAs splits the sum; the parts meet
//     through distributed shared memory in rank order.  Lanes are features, so any output
//     stride is stored coalesced.  16 x 13824 x 5120: 31 us, 4.6 TB/s of weight.
//
// Rounding: z is rounded once for `pre` and once, after activation and residual in fp32,
// for y.  dz is rounded to the operand type because the tensor cores take 16 bits; db sums
// the unrounded dz.  Every wait is bounded (VDN_ERR_TIMEOUT).  No TMA multicast.
#include <initializer_list>

#include "train_common.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace vdn {
namespace lact {

using namespace sm100;

constexpr int BK = 64;                    // 64 values of 16 bits = one 128-byte swizzle row
enum { NONE = VDN_ACT_NONE, TANH = VDN_ACT_GELU_TANH, ERF = VDN_ACT_GELU_ERF, SILU = VDN_ACT_SILU };

// ------------------------------------------------------------------ activations
// gelu(tanh form) = z sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3); silu = z sigmoid(z).
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == NONE) return z;
  if constexpr (ACT == ERF) return 0.5f * z * erfcf(z * -0.7071067811865476f);   // 1 + erf cancels below z = -3
  const float v = ACT == TANH ? 1.5957691216057308f * fmaf(0.044715f * z * z, z, z) : z;
  return __fdividef(z, 1.0f + __expf(-v));   // exp overflow: z / inf = 0
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == NONE) return 1.0f;
  float c;                                   // past 30 the slope is 0 or 1; NaN stays NaN
  asm("max.NaN.f32 %0, %1, 0fC1F00000;\n\tmin.NaN.f32 %0, %0, 0f41F00000;" : "=f"(c) : "f"(z));
  if constexpr (ACT == ERF)
    return 0.5f * erfcf(c * -0.7071067811865476f) + c * 0.3989422804014327f * __expf(-0.5f * c * c);
  const float k = 1.5957691216057308f;
  const float v = ACT == TANH ? k * fmaf(0.044715f * c * c, c, c) : c;
  const float dv = ACT == TANH ? k * fmaf(0.134145f * c, c, 1.0f) : 1.0f;
  const float e = __expf(-fabsf(v)), r = __fdividef(1.0f, 1.0f + e);
  return (v >= 0.f ? r : e * r) + c * dv * (e * r * r);
}

// Two slopes at a time on packed pairs (gelu's tanh form and silu): the same formula with one
// reciprocal for both, r0 = q (1 + e1), r1 = q (1 + e0), q = 1 / ((1 + e0) (1 + e1)).
template <int ACT>
__device__ __forceinline__ f2 act_slope2(f2 z) {
  auto c2 = [](float v) { return f2_pack(v, v); };
  float z0, z1;
  f2_unpack(z, z0, z1);
  if constexpr (ACT == NONE || ACT == ERF) return f2_pack(act_slope<ACT>(z0), act_slope<ACT>(z1));
  asm("max.NaN.f32 %0, %0, 0fC1F00000;\n\tmin.NaN.f32 %0, %0, 0f41F00000;" : "+f"(z0));
  asm("max.NaN.f32 %0, %0, 0fC1F00000;\n\tmin.NaN.f32 %0, %0, 0f41F00000;" : "+f"(z1));
  const f2 c = f2_pack(z0, z1);
  f2 v = c, cdv = c;                         // the sigmoid's argument, and c dv/dc
  if constexpr (ACT == TANH) {
    const float k = 1.5957691216057308f;
    const f2 s = f2_mul(c, c);
    v = f2_mul(c, f2_fma(s, c2(0.044715f * k), c2(k)));
    cdv = f2_mul(c, f2_fma(s, c2(0.134145f * k), c2(k)));
  }
  float v0, v1, a, b, q0, q1, p0, p1;
  f2_unpack(v, v0, v1);
  f2_unpack(f2_mul(f2_pack(fabsf(v0), fabsf(v1)), c2(-1.4426950408889634f)), a, b);
  // fmaxf: a NaN's exponential becomes 0, so that the shared reciprocal stays its neighbour's; its own
  // slope is NaN through cdv
  const f2 e = f2_pack(ex2_approx(fmaxf(a, -150.f)), ex2_approx(fmaxf(b, -150.f)));
  f2_unpack(f2_add(e, c2(1.0f)), a, b);
  const float q = rcp_approx(a * b);
  const f2 r = f2_mul(f2_pack(b, a), c2(q)), er = f2_mul(e, r);
  f2_unpack(r, q0, q1);
  f2_unpack(er, p0, p1);
  return f2_fma(cdv, f2_mul(er, r), f2_pack(v0 >= 0.f ? q0 : p0, v1 >= 0.f ? q1 : p1));
}

// ------------------------------------------------------------------ shared pieces
__device__ __forceinline__ void mma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
template <typename T>
constexpr uint32_t idesc_f16(int m, int n, int a_mn, int b_mn) {
  constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;   // both operands alike
  return (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Operand tile of 64-deep block `s` at step ks (16 deep).  K-major: rows of 128 bytes, a
// step is 32 bytes along the row.  MN-major: regions of 64 rows x 64 deep (8 KB), a step
// is 16 of the 128-byte depth rows.
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t base, int ks) {
  return MN ? desc_mn_sw128(base + ks * 2048, 8192) : desc_k_sw128(base + ks * 32);
}

struct Params {
  const void* bias;      // [cols] or null
  const void* resid;     // [rows, cols], row stride ldr, or null
  void* y;               // [rows, cols], row stride ldy
  void* pre;             // or null
  int64_t rows, cols, ldr, ldy, ldp;
  int m_tiles, n_tiles, k_blocks;
  bool tma_y, tma_p, tma_r;   // alignment allows bulk stores / loads of that matrix
  bool bias_vec;
  int* status;
};

// ------------------------------------------------------------------ pair kernel
constexpr int STAGES = 6, P_A = 128 * BK * 2, P_B = 128 * BK * 2;
constexpr int PAIR_THREADS = 320, PIECE = 32 * 128, GROUP_M = 16;
constexpr size_t PAIR_SMEM = 1024 + STAGES * (P_A + P_B) + 8 * PIECE + 256;
static_assert(PAIR_SMEM <= 232448, "shared memory per CTA");

// Tiles in groups of GROUP_M rows of tiles, row fastest: a group's P stays in L2 while Q passes.
__device__ __forceinline__ void tile_at(int t, int m_tiles, int n_tiles, int& mb, int& nb) {
  const int per = GROUP_M * n_tiles, g = t / per, first = g * GROUP_M;
  const int rows = min(GROUP_M, m_tiles - first), r = t - g * per;
  mb = first + r % rows;
  nb = r / rows;
}

// A 32 x 64 piece (lane = row, 128-byte swizzled rows) from or to a matrix whose alignment
// allows no bulk copy: lane pairs of columns, row by row.
template <typename T>
__device__ __forceinline__ uint16_t* piece_at(uint8_t* piece, int row, int col) {
  return reinterpret_cast<uint16_t*>(piece + row * 128 + (((col >> 3) ^ (row & 7)) << 4) + (col & 7) * 2);
}
template <typename T>
__device__ __forceinline__ void piece_out(uint8_t* piece, void* dst, int64_t ld, int64_t row0, int64_t col0,
                                          const Params& p, int lane) {
  for (int r = 0; r < 32 && row0 + r < p.rows; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (col0 + h * 32 + lane < p.cols)
        static_cast<uint16_t*>(dst)[(row0 + r) * ld + col0 + h * 32 + lane] = *piece_at<T>(piece, r, h * 32 + lane);
}
template <typename T>
__device__ __forceinline__ void piece_in(uint8_t* piece, const void* src, int64_t ld, int64_t row0, int64_t col0,
                                         const Params& p, int lane) {
  for (int r = 0; r < 32; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t c = col0 + h * 32 + lane;
      *piece_at<T>(piece, r, h * 32 + lane) =
          row0 + r < p.rows && c < p.cols ? static_cast<const uint16_t*>(src)[(row0 + r) * ld + c] : (uint16_t)0;
    }
}

template <typename T, bool A_MN, bool B_MN, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                const __grid_constant__ CUtensorMap ty, const __grid_constant__ CUtensorMap tp,
                const __grid_constant__ CUtensorMap tr, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * P_A;
  uint8_t* pieces = sB + STAGES * P_B;
  uint64_t* full = reinterpret_cast<uint64_t*>(pieces + 8 * PIECE);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;       // 2
  uint64_t* acc_empty = acc_full + 2;        // 2
  uint64_t* mma_done = acc_empty + 2;
  uint64_t* resid_bar = mma_done + 1;        // 8, one per epilogue warp
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(resid_bar + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((2 * STAGES + 13) * 8 + 8 <= 256, "barrier region");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair_id = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 16);          // the epilogue warps of both CTAs
    }
    mbar_init(mma_done, 1);
    for (int w = 0; w < 8; ++w) mbar_init(&resid_bar[w], 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&ta);
    prefetch_tensormap(&tb);
  }
  if (warp == 1) tmem_alloc_pair(tmem_holder, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();                            // barriers stand before any remote arrive or copy
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const int num_tiles = p.m_tiles * p.n_tiles;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ producer
      const uint32_t full_leader = mapa_shared(full, 0);
      int stage = 0;
      uint32_t phase = 0, pending = 0, pending_phase = 0;
      for (int t = pair_id; t < num_tiles && !*abort_flag; t += npairs) {
        int mb, nb;
        tile_at(t, p.m_tiles, p.n_tiles, mb, nb);
        const int arow = (mb * 2 + (int)rank) * 128, brow = (nb * 2 + (int)rank) * 128;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) break;
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * (P_A + P_B));
          const uint32_t fb = full_leader + stage * 8;
          uint8_t* a = sA + stage * P_A;
          uint8_t* b = sB + stage * P_B;
          if constexpr (A_MN) {
            tma_load_2d_pair(a, &ta, fb, arow, kb * BK);
            tma_load_2d_pair(a + 8192, &ta, fb, arow + 64, kb * BK);
          } else {
            tma_load_2d_pair(a, &ta, fb, kb * BK, arow);
          }
          if constexpr (B_MN) {
            tma_load_2d_pair(b, &tb, fb, brow, kb * BK);
            tma_load_2d_pair(b + 8192, &tb, fb, brow + 64, kb * BK);
          } else {
            tma_load_2d_pair(b, &tb, fb, kb * BK, brow);
          }
          pending |= 1u << stage;
          pending_phase = (pending_phase & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (*abort_flag && pending) {          // copies already issued land before the CTA may exit
        const uint64_t t0 = globaltimer();
        if (leader) {
          for (int s = 0; s < STAGES; ++s)
            while ((pending >> s & 1) && !mbar_try_wait(&full[s], (pending_phase >> s) & 1) &&
                   globaltimer() - t0 < kWaitLimitNs) {
            }
        } else {                             // these signal the leader's barriers: a fixed time
          while (globaltimer() - t0 < 200000) {
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ----------------------------------------------------------------- MMA
      constexpr uint32_t kIdesc = idesc_f16<T>(256, 256, A_MN, B_MN);
      int stage = 0, k = 0;
      uint32_t phase = 0;
      bool issued = false;
      for (int t = pair_id; t < num_tiles; t += npairs, ++k) {
        const int b = k & 1;
        if (!mbar_wait(&acc_empty[b], ((k >> 1) & 1) ^ 1, abort_flag)) break;
        tc_fence_after();
        bool ok = true;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + stage * P_A), b0 = smem_u32(sB + stage * P_B);
#pragma unroll
          for (int ks = 0; ks < BK / 16; ++ks)
            mma_f16_pair(tmem + b * 256, operand_desc<A_MN>(a0, ks), operand_desc<B_MN>(b0, ks), kIdesc, (kb | ks) != 0);
          issued = true;
          tc_commit_pair(&empty[stage], 0x3);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        tc_commit_pair(&acc_full[b], 0x3);
      }
      if (*abort_flag && issued) {
        tc_commit_pair(mma_done, 0x1);
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(mma_done, 0) && globaltimer() - t0 < kWaitLimitNs) {
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3, half = (warp - 2) >> 2;   // TMEM lane quadrant, 128-column half
    uint8_t* piece = pieces + (warp - 2) * PIECE;
    uint8_t* line = piece + lane * 128;
    uint64_t* rbar = &resid_bar[warp - 2];
    uint32_t rphase = 0;
    const bool has_p = p.pre != nullptr, has_r = p.resid != nullptr;
    int k = 0;
    for (int t = pair_id; t < num_tiles; t += npairs, ++k) {
      int mb, nb;
      tile_at(t, p.m_tiles, p.n_tiles, mb, nb);
      const int b = k & 1;
      const int64_t row0 = (int64_t)(mb * 2 + (int)rank) * 128 + quad * 32;
      bool waited = false;
      for (int part = 0; part < 2; ++part) {             // 64 columns at a time
        const int64_t col0 = (int64_t)nb * 256 + half * 128 + part * 64;
        const bool live = row0 < p.rows && col0 < p.cols;   // warp-uniform
        if (live) {
          if (lane == 0) bulk_wait_group_read<0>();      // the piece's last store has left it
          __syncwarp();
          if (has_r && !has_p && p.tma_r && lane == 0) {
            mbar_arrive_expect_tx(rbar, PIECE);
            tma_load_2d(piece, &tr, rbar, (int)col0, (int)row0);
          }
        }
        if (!waited && !__all_sync(0xffffffffu, mbar_wait(&acc_full[b], (k >> 1) & 1, abort_flag))) break;
        waited = true;
        tc_fence_after();
        uint32_t r[64];
        const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + b * 256 + half * 128 + part * 64;
        tmem_ld_32x32b_x32(taddr, r);
        tmem_ld_32x32b_x32(taddr + 32, r + 32);
        tmem_ld_wait();
        if (part == 1) {                                 // the accumulator is free for the tile after next
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (leader) mbar_arrive(&acc_empty[b]);
            else mbar_arrive_cluster(mapa_shared(&acc_empty[b], 0));
          }
        }
        if (!live) continue;
        if (p.bias) {                                    // the same address in every lane: one broadcast each
          const T* bias = static_cast<const T*>(p.bias) + col0;
          if (p.bias_vec && col0 + 64 <= p.cols) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              float e[8];
              unpack<T, 8>(__ldg(reinterpret_cast<const uint4*>(bias) + c), e);
#pragma unroll
              for (int i = 0; i < 8; ++i) r[8 * c + i] = __float_as_uint(__uint_as_float(r[8 * c + i]) + e[i]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 64; ++c)
              if (col0 + c < p.cols) r[c] = __float_as_uint(__uint_as_float(r[c]) + to_f32(bias[c]));
          }
        }
        auto put = [&](auto value) {                     // 64 results of this row, rounded, to the piece
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint4 w;
            w.x = pack2<T>(value(8 * c), value(8 * c + 1));
            w.y = pack2<T>(value(8 * c + 2), value(8 * c + 3));
            w.z = pack2<T>(value(8 * c + 4), value(8 * c + 5));
            w.w = pack2<T>(value(8 * c + 6), value(8 * c + 7));
            *reinterpret_cast<uint4*>(line + ((c ^ (lane & 7)) << 4)) = w;
          }
        };
        auto send = [&](const CUtensorMap& map, bool bulk, void* dst, int64_t ld) {
          if (bulk) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&map, piece, (int)col0, (int)row0);
              bulk_commit_group();
            }
          } else {
            __syncwarp();
            piece_out<T>(piece, dst, ld, row0, col0, p, lane);
            fence_proxy_async_smem();        // a residual copy may follow these reads
            __syncwarp();
          }
        };
        if (has_p) {
          put([&](int c) { return __uint_as_float(r[c]); });
          send(tp, p.tma_p, p.pre, p.ldp);
          if (lane == 0) bulk_wait_group_read<0>();
          __syncwarp();
          if (has_r && p.tma_r && lane == 0) {
            mbar_arrive_expect_tx(rbar, PIECE);
            tma_load_2d(piece, &tr, rbar, (int)col0, (int)row0);
          }
        }
        if constexpr (ACT != NONE) {
#pragma unroll
          for (int c = 0; c < 64; ++c) r[c] = __float_as_uint(act_value<ACT>(__uint_as_float(r[c])));
        }
        if (has_r) {
          if (p.tma_r) {
            if (!__all_sync(0xffffffffu, mbar_wait(rbar, rphase, abort_flag))) break;
            rphase ^= 1;
          } else {
            piece_in<T>(piece, p.resid, p.ldr, row0, col0, p, lane);
            __syncwarp();
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float e[8];
            unpack<T, 8>(*reinterpret_cast<const uint4*>(line + ((c ^ (lane & 7)) << 4)), e);
#pragma unroll
            for (int i = 0; i < 8; ++i) r[8 * c + i] = __float_as_uint(__uint_as_float(r[8 * c + i]) + e[i]);
          }
        }
        put([&](int c) { return __uint_as_float(r[c]); });
        send(ty, p.tma_y, p.y, p.ldy);
      }
      if (*abort_flag) break;
    }
    if (lane == 0) bulk_wait_group<0>();     // every store is written before the CTA exits
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();                            // the pair's MMAs and remote arrives are done
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc_pair(tmem, 512);
  }
  cluster_sync();                            // neither CTA leaves while the pair's TMEM is in use
  if (threadIdx.x == 0 && *abort_flag && p.status) atomicExch(p.status, VDN_ERR_TIMEOUT);
}

// ---------------------------------------------------------------- narrow kernel
constexpr int NARROW_THREADS = 320;          // producer, issuer, eight epilogue warps
template <int BN> constexpr int narrow_stages() { return BN >= 128 ? 3 : BN >= 64 ? 4 : BN >= 32 ? 5 : 6; }   // two CTAs an SM
template <int BN> constexpr size_t narrow_ring() { return narrow_stages<BN>() * (size_t)(16384 + BN * 128); }
template <int BN> constexpr size_t narrow_smem() { return 1024 + narrow_ring<BN>() + 256; }
static_assert(narrow_smem<16>() <= 115712 && narrow_smem<32>() <= 115712 && narrow_smem<64>() <= 115712 &&
              narrow_smem<128>() <= 115712, "two CTAs an SM");

// Each thread of the warp reads N columns of its TMEM lane.
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld_32x32b_x32(taddr, r); }

__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// D^T: features (the output's columns) on M, tokens (its rows) on N.  m_tiles counts
// 128-feature tiles, n_tiles BN-token tiles; the cluster's CTAs share one tile's depth, and
// CTA r finishes the r-th part of its tokens from the parts that all CTAs push to it.
template <typename T, bool F_MN, bool X_MN, int ACT, int BN>
__global__ void __launch_bounds__(NARROW_THREADS, 2)
    narrow_kernel(const __grid_constant__ CUtensorMap tf, const __grid_constant__ CUtensorMap tx, const Params p,
                  const int split) {
  constexpr int ST = narrow_stages<BN>(), A_BYTES = 16384, B_BYTES = BN * 128;
  constexpr int COLS = BN < 32 ? 32 : BN;    // TMEM columns
  constexpr int CH = BN / 2 < 32 ? BN / 2 : 32;   // tokens an epilogue warp holds at a time
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + ST * A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + narrow_ring<BN>());
  uint64_t* empty = full + ST;
  uint64_t* acc_full = empty + ST;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  float* parts = reinterpret_cast<float*>(smem);   // [source rank][token of this CTA][128], in the idle ring
  static_assert(BN * 128 * 4 <= narrow_ring<BN>(), "parts fit the ring");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  const int tile = blockIdx.x / split;
  const int ft = tile % p.m_tiles, xt = tile / p.m_tiles;
  const int kb0 = (int)((int64_t)p.k_blocks * rank / split), kb1 = (int)((int64_t)p.k_blocks * (rank + 1) / split);
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_holder, COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t pending = 0;
      int stage = 0;
      uint32_t phase = 0, pending_phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) break;
        mbar_arrive_expect_tx(&full[stage], A_BYTES + B_BYTES);
        uint8_t* a = sA + stage * A_BYTES;
        uint8_t* b = sB + stage * B_BYTES;
        if constexpr (F_MN) {
          tma_load_2d(a, &tf, &full[stage], ft * 128, kb * BK);
          tma_load_2d(a + 8192, &tf, &full[stage], ft * 128 + 64, kb * BK);
        } else {
          tma_load_2d(a, &tf, &full[stage], kb * BK, ft * 128);
        }
        if constexpr (X_MN) {
#pragma unroll
          for (int c = 0; c < BN; c += 64) tma_load_2d(b + c * 128, &tx, &full[stage], xt * BN + c, kb * BK);
        } else {
          tma_load_2d(b, &tx, &full[stage], kb * BK, xt * BN);
        }
        pending |= 1u << stage;
        pending_phase = (pending_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == ST) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (*abort_flag) {                     // copies already issued land before the ring is reused
        const uint64_t t0 = globaltimer();
        for (int s = 0; s < ST; ++s)
          while ((pending >> s & 1) && !mbar_try_wait(&full[s], (pending_phase >> s) & 1) &&
                 globaltimer() - t0 < kWaitLimitNs) {
          }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t kIdesc = idesc_f16<T>(128, BN, F_MN, X_MN);   // kind::f16, the type in the descriptor
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag)) break;
        tc_fence_after();
        const uint32_t a0 = smem_u32(sA + stage * A_BYTES), b0 = smem_u32(sB + stage * B_BYTES);
#pragma unroll
        for (int ks = 0; ks < BK / 16; ++ks)
          mma_bf16(tmem, operand_desc<F_MN>(a0, ks), operand_desc<X_MN>(b0, ks), kIdesc, kb > kb0 || ks > 0);
        tc_commit(&empty[stage]);
        if (++stage == ST) {
          stage = 0;
          phase ^= 1;
        }
      }
      tc_commit(acc_full);                   // also after a give-up: the issued products drain
    }
  }
  __syncwarp();                              // no lane spins beside its warp's producer or issuer
  const bool epi = warp >= 2;
  const int quad = warp & 3, group = (warp - 2) >> 2;   // TMEM lane quadrant, half of the tokens
  const int f = quad * 32 + lane;            // feature within the tile
  const int64_t col = (int64_t)ft * 128 + f;
  const bool in = epi && col < p.cols;
  const float bias = in && p.bias ? to_f32(static_cast<const T*>(p.bias)[col]) : 0.f;
  const int64_t row0 = (int64_t)xt * BN;
  const int rows = (int)min((int64_t)BN, p.rows - row0);
  // N results of this feature, `step` tokens apart from row0 + c0; residuals in flight together.
  auto finish = [&](auto n, const float (&z)[decltype(n)::value], int c0, int step) {
    constexpr int N = decltype(n)::value;
    if (!in) return;
    float r[N];
    if (p.resid) {
      const T* q = static_cast<const T*>(p.resid) + (row0 + c0) * p.ldr + col;
      const int64_t d = p.ldr * step;
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = c0 + i * step < rows ? to_f32(q[i * d]) : 0.f;
    }
    T* q = static_cast<T*>(p.y) + (row0 + c0) * p.ldy + col;
    T* qp = static_cast<T*>(p.pre) + (row0 + c0) * p.ldp + col;
    const int64_t d = p.ldy * step, dp = p.ldp * step;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (c0 + i * step >= rows) break;
      const float v = z[i] + bias;
      if (p.pre) qp[i * dp] = from_f32<T>(v);
      float o = act_value<ACT>(v);
      if (p.resid) o += r[i];
      q[i * d] = from_f32<T>(o);
    }
  };
  mbar_wait(acc_full, 0, abort_flag);        // the ring is idle after it
  __syncwarp();
  tc_fence_after();
  if (split > 1) {
    __syncthreads();
    cluster_sync();                          // every ring of the cluster is
  }
  const int per = BN / split;
  if (epi && !*abort_flag) {
#pragma unroll 1
    for (int c0 = group * CH; c0 < BN; c0 += 2 * CH) {
      if (c0 >= rows) break;
      uint32_t r[CH];
      tmem_ld(tmem + ((uint32_t)(quad * 32) << 16) + c0, r);
      tmem_ld_wait();
      if (split == 1) {
        float z[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) z[c] = __uint_as_float(r[c]);
        finish(std::integral_constant<int, CH>{}, z, c0, 1);
      } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int t = c0 + c, owner = t / per;
          st_cluster(mapa_shared(&parts[((rank * per) + t - owner * per) * 128 + f], owner), __uint_as_float(r[c]));
        }
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (split > 1) {
    cluster_sync();                          // all parts are here; nothing remote happens after it
    if (epi && !*abort_flag) {               // this CTA's tokens, ranks in order, two at a time
      for (int t = group * 2; t < per; t += 4) {
        float z[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          z[i] = 0.f;
          for (int k = 0; k < split; ++k)
            if (t + i < per) z[i] += parts[(k * per + t + i) * 128 + f];
        }
        if (t + 1 < per) finish(std::integral_constant<int, 2>{}, z, rank * per + t, 1);
        else finish(std::integral_constant<int, 1>{}, reinterpret_cast<const float(&)[1]>(z), rank * per + t, 1);
      }
    }
  }
  if (warp == 1) {
    tc_fence_after();
    __syncwarp();
    tmem_dealloc(tmem, COLS);
  }
  if (threadIdx.x == 0 && *abort_flag && p.status) atomicExch(p.status, VDN_ERR_TIMEOUT);
}

// -------------------------------------------------------- dz and the bias gradient
// dz = dy act'(pre) (skipped for no activation), and per-chunk column sums of the unrounded
// dz.  grid (column strips of 32 * VEC, row chunks); 32 column lanes x 8 row groups a block.
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(256) dz_kernel(const T* dy, int64_t ldy, const T* pre, int64_t ldp, T* dz, int64_t ldz,
                                                 int64_t rows, int64_t cols, int64_t chunk, float* part) {
  __shared__ float sums[8][32 * VEC + 1];
  using R = Raw<T, VEC>;
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 * VEC + lane * VEC;
  const int64_t r0 = (int64_t)blockIdx.y * chunk, r1 = min(r0 + chunk, rows);
  using V = typename Lanes<VEC>::V;
  constexpr int NP = Lanes<VEC>::N;
  V total[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) total[i] = vset(V{}, 0.f);
  if (c < cols) {
    constexpr int U = 4;                     // rows in flight
    for (int64_t r = r0 + g; r < r1; r += 8 * U) {
      R a[U], b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool in = r + 8 * u < r1;
        a[u] = in ? load_once<R>(dy + (r + 8 * u) * ldy + c) : raw_zero<R>();
        if constexpr (ACT != NONE) b[u] = in ? load_once<R>(pre + (r + 8 * u) * ldp + c) : raw_zero<R>();
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        V d[NP];
        unpack_lanes<T, VEC>(a[u], d);
        if constexpr (ACT != NONE) {
          V z[NP];
          unpack_lanes<T, VEC>(b[u], z);
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            if constexpr (VEC == 1) d[i] = vmul(d[i], act_slope<ACT>(z[i]));
            else d[i] = vmul(d[i], act_slope2<ACT>(z[i]));
          }
          if (r + 8 * u < r1) *reinterpret_cast<R*>(dz + (r + 8 * u) * ldz + c) = pack_lanes<T, VEC>(d);
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) total[i] = vadd(total[i], d[i]);
      }
    }
  }
  float acc[VEC];
  from_lanes(total, acc);
  if (!part) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i) sums[g][lane * VEC + i] = acc[i];
  __syncthreads();
  for (int j = threadIdx.x; j < 32 * VEC; j += 256) {
    const int64_t col = (int64_t)blockIdx.x * 32 * VEC + j;
    if (col >= cols) break;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k][j];
    part[blockIdx.y * cols + col] = s;
  }
}

// ------------------------------------------------------------------------ host
constexpr int kDevices = 64;
struct Dev {
  int index = 0, sms = 0;
};
static int device(Dev& d) {
  static int sms[kDevices] = {};
  VDN_CUDA_TRY(cudaGetDevice(&d.index));
  VDN_CHECK_ARG(d.index >= 0 && d.index < kDevices, "device index out of range");
  if (!sms[d.index]) VDN_CUDA_TRY(cudaDeviceGetAttribute(&sms[d.index], cudaDevAttrMultiProcessorCount, d.index));
  d.sms = sms[d.index];
  return VDN_OK;
}

// An operand [outer, inner] (inner contiguous): K-major loads boxes of 64 inner (depth) x
// `span` outer rows, MN-major boxes of 64 inner (rows) x 64 outer (depth).
template <typename T>
static int operand_map(CUtensorMap* map, const void* base, int64_t inner, int64_t outer, int64_t ld, bool mn, int span) {
  const auto type = std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)(mn ? BK : span)};
  return encode_map(map, type, 2, base, dims, strides, box);
}
template <typename T>
static int piece_map(CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t ld) {
  const auto type = std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64, 32};
  return encode_map(map, type, 2, base, dims, strides, box);
}

struct Operand {
  const void* base;
  int64_t ld;
  bool mn;                                   // MN-major: stored [depth, rows]
};

// Raises a kernel's shared-memory limit, once per device.
#define VDN_ALLOW_SMEM(kernel, bytes, dev)                                                                    \
  do {                                                                                                        \
    static bool set[kDevices] = {};                                                                           \
    if (!set[dev]) {                                                                                          \
      VDN_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(bytes))); \
      set[dev] = true;                                                                                        \
    }                                                                                                         \
  } while (0)

template <typename T, bool A_MN, bool B_MN, int ACT>
static int run_pair(const Operand& x, const Operand& f, int64_t depth, Params p, const Dev& d, cudaStream_t stream) {
  CUtensorMap ma, mb, my, mp, mr;
  auto map = [&](CUtensorMap* m, const Operand& o, int64_t rows) {
    return o.mn ? operand_map<T>(m, o.base, rows, depth, o.ld, true, 0) : operand_map<T>(m, o.base, depth, rows, o.ld, false, 128);
  };
  if (int rc = map(&ma, x, p.rows)) return rc;
  if (int rc = map(&mb, f, p.cols)) return rc;
  auto bulk = [&](CUtensorMap* m, const void* base, int64_t ld, bool& on) -> int {
    on = base && aligned16(base) && ld % 8 == 0 && ld >= p.cols;
    if (!on) {
      *m = ma;
      return VDN_OK;
    }
    return piece_map<T>(m, base, p.cols, p.rows, ld);
  };
  if (int rc = bulk(&my, p.y, p.ldy, p.tma_y)) return rc;
  if (int rc = bulk(&mp, p.pre, p.ldp, p.tma_p)) return rc;
  if (int rc = bulk(&mr, p.resid, p.ldr, p.tma_r)) return rc;
  p.m_tiles = (int)((p.rows + 255) / 256);
  p.n_tiles = (int)((p.cols + 255) / 256);
  auto* kernel = pair_kernel<T, A_MN, B_MN, ACT>;
  p.bias_vec = aligned16(p.bias);
  VDN_ALLOW_SMEM(kernel, PAIR_SMEM, d.index);
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles, pairs = d.sms / 2;
  kernel<<<(unsigned)(2 * (tiles < pairs ? tiles : pairs)), PAIR_THREADS, PAIR_SMEM, stream>>>(ma, mb, my, mp, mr, p);
  VDN_LAUNCH_CHECK("linear (pair)");
  return VDN_OK;
}

template <typename T, bool F_MN, bool X_MN, int ACT, int BN>
static int run_narrow(const Operand& x, const Operand& f, int64_t depth, Params p, const Dev& d, int split,
                      cudaStream_t stream) {
  CUtensorMap mf, mx;
  if (int rc = F_MN ? operand_map<T>(&mf, f.base, p.cols, depth, f.ld, true, 0)
                    : operand_map<T>(&mf, f.base, depth, p.cols, f.ld, false, 128)) return rc;
  if (int rc = X_MN ? operand_map<T>(&mx, x.base, p.rows, depth, x.ld, true, 0)
                    : operand_map<T>(&mx, x.base, depth, p.rows, x.ld, false, BN)) return rc;
  p.m_tiles = (int)((p.cols + 127) / 128);
  p.n_tiles = (int)((p.rows + BN - 1) / BN);
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  auto* kernel = narrow_kernel<T, F_MN, X_MN, ACT, BN>;
  VDN_ALLOW_SMEM(kernel, narrow_smem<BN>(), d.index);
  VDN_CHECK_ARG(tiles * split < (1ll << 31), "too many tiles for one launch");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split));
  cfg.blockDim = dim3(NARROW_THREADS);
  cfg.dynamicSmemBytes = narrow_smem<BN>();
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VDN_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, mf, mx, p, split));
  return VDN_OK;
}

// Tokens a tile and CTAs that split the depth.  In units of 10 ns, measured: a CTA costs 300 to
// start, 10 + BN / 8 a depth block (its bytes through L2), 6 a token of epilogue; a split
// shares the epilogue but adds 250 for its two cluster barriers.  Two CTAs fit an SM; clusters
// take four fifths of the places at most (those of eight do not pack into every GPC: a second
// wave cost 6 us of 11).
static void narrow_shape(int64_t rows, int64_t cols, int k_blocks, int least, int sms, int& bn, int& split) {
  int64_t best = -1;
  for (int b = least; b <= 128; b *= 2) {
    const int64_t tiles = ((cols + 127) / 128) * ((rows + b - 1) / b);
    for (int s = 1; s <= 8; s *= 2) {
      if (s > 1 && (tiles * s * 5 > 2 * sms * 4 || k_blocks < 2 * s)) break;
      const int64_t waves = (tiles * s + 2 * sms - 1) / (2 * sms), share = tiles * s > sms ? 2 : 1;
      const int64_t t = waves * (300 + share * ((int64_t)(k_blocks + s - 1) / s * (10 + b / 8) + 6 * b / s) + (s > 1 ? 250 + b : 0));
      if (best < 0 || t < best) {
        best = t;
        bn = b;
        split = s;
      }
    }
  }
}

// y [rows, cols] = sum over depth of x[rows] f[cols].
template <typename T, bool X_MN, bool F_MN, int ACT>
static int product(const Operand& x, const Operand& f, int64_t depth, Params p, cudaStream_t stream) {
  Dev d;
  if (int rc = device(d)) return rc;
  p.k_blocks = (int)((depth + BK - 1) / BK);
  const int64_t pair_tiles = ((p.rows + 255) / 256) * ((p.cols + 255) / 256);
  // Up to 128 rows would leave half of every pair tile empty, and fewer than 28 pair tiles most
  // SMs without work; narrow tiles with a split depth fill them.
  VDN_CHECK_ARG(pair_tiles < (1ll << 29), "too many tiles for one launch");
  if (pair_tiles >= 28 && p.rows > 128) return run_pair<T, X_MN, F_MN, ACT>(x, f, depth, p, d, stream);
  int bn = 128, split = 1;
  narrow_shape(p.rows, p.cols, p.k_blocks, X_MN ? 64 : 16, d.sms, bn, split);
  if constexpr (!X_MN) {
    if (bn == 16) return run_narrow<T, F_MN, X_MN, ACT, 16>(x, f, depth, p, d, split, stream);
    if (bn == 32) return run_narrow<T, F_MN, X_MN, ACT, 32>(x, f, depth, p, d, split, stream);
  }
  if (bn == 64) return run_narrow<T, F_MN, X_MN, ACT, 64>(x, f, depth, p, d, split, stream);
  return run_narrow<T, F_MN, X_MN, ACT, 128>(x, f, depth, p, d, split, stream);
}

// Copies up to two matrices into rows whose stride the tensor maps take (odd depths, unaligned
// views): a thread per 16 bytes written, read in the widest pieces the source's alignment allows.
struct Pad {
  const uint16_t* src[2];
  uint16_t* dst[2];
  int64_t rows[2], cols[2], ld[2], to[2];
  int piece[2];          // values a load takes: 4, 2 or 1
};
__global__ void __launch_bounds__(256) pad_kernel(const Pad p) {
  const int m = blockIdx.y;
  const int64_t per = p.to[m] / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.rows[m] * per) return;
  const int64_t row = i / per, c = (i - row * per) * 8;
  const uint16_t* s = p.src[m] + row * p.ld[m] + c;
  const int n = (int)min((int64_t)8, p.cols[m] - c);
  alignas(16) uint16_t v[8] = {};
  if (n == 8 && p.piece[m] == 4) {
    reinterpret_cast<uint2*>(v)[0] = reinterpret_cast<const uint2*>(s)[0];
    reinterpret_cast<uint2*>(v)[1] = reinterpret_cast<const uint2*>(s)[1];
  } else if (n == 8 && p.piece[m] == 2) {
#pragma unroll
    for (int k = 0; k < 4; ++k) reinterpret_cast<uint32_t*>(v)[k] = reinterpret_cast<const uint32_t*>(s)[k];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) v[k] = s[k];
  }
  *reinterpret_cast<uint4*>(p.dst[m] + row * p.to[m] + c) = *reinterpret_cast<const uint4*>(v);
}

static int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
static bool fits_map(const void* base, int64_t ld, int64_t cols) { return aligned16(base) && ld >= cols && ld % 8 == 0; }
static size_t padded_bytes(const void* base, int64_t ld, int64_t rows, int64_t cols) {
  return fits_map(base, ld, cols) ? 0 : ((size_t)rows * pad8(cols) * 2 + 255) / 256 * 256;
}

// The operands as the tensor maps take them: as they lie, or copied into the workspace (which
// advances past what was used).
struct Matrix {
  const void*& base;
  int64_t& ld;
  int64_t rows, cols;
};
static int settle(std::initializer_list<Matrix> operands, uint8_t*& ws, size_t& left, cudaStream_t stream) {
  Pad p = {};
  int n = 0;
  int64_t most = 0;
  for (const Matrix& o : operands) {
    const size_t bytes = padded_bytes(o.base, o.ld, o.rows, o.cols);
    if (!bytes) continue;
    VDN_CHECK_ARG(ws && bytes <= left, "workspace smaller than the padded operands need");
    VDN_CHECK_ARG(aligned16(ws), "the workspace must be 16-byte aligned");
    p.src[n] = static_cast<const uint16_t*>(o.base);
    p.dst[n] = reinterpret_cast<uint16_t*>(ws);
    p.rows[n] = o.rows;
    p.cols[n] = o.cols;
    p.ld[n] = o.ld;
    p.to[n] = pad8(o.cols);
    p.piece[n] = o.ld % 4 == 0 && aligned_to(o.base, 8) ? 4 : o.ld % 2 == 0 && aligned_to(o.base, 4) ? 2 : 1;
    const int64_t vectors = o.rows * (pad8(o.cols) / 8);
    most = vectors > most ? vectors : most;
    o.base = ws;
    o.ld = pad8(o.cols);
    ws += bytes;
    left -= bytes;
    ++n;
  }
  if (!n) return VDN_OK;
  pad_kernel<<<dim3((unsigned)((most + 255) / 256), n), 256, 0, stream>>>(p);
  VDN_LAUNCH_CHECK("linear (padded operands)");
  return VDN_OK;
}

static int check(int dtype, int64_t rows, int64_t n, int64_t k) {
  if (dtype != VDN_DTYPE_BF16 && dtype != VDN_DTYPE_F16) return set_error(VDN_ERR_TYPE, "linear takes bf16 or fp16");
  VDN_CHECK_ARG(rows >= 0 && n >= 1 && k >= 1, "bad linear extents");
  VDN_CHECK_ARG(rows < (1ll << 30) && n < (1ll << 30) && k < (1ll << 30), "extents too large");
  return VDN_OK;
}
template <typename T, int ACT>
static int forward(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t k, const Params& p, cudaStream_t s) {
  return product<T, false, false, ACT>({x, ldx, false}, {w, ldw, false}, k, p, s);
}

// Row chunks of the bias gradient, at most: 64, or as many as give narrow outputs eight CTAs an SM.
static int64_t chunk_count(int64_t n) {
  const int64_t c = 8 * 148 / ((n + 255) / 256);
  return c > 64 ? c : 64;
}
static int64_t chunk_rows(int64_t rows, int64_t n) { return (((rows + chunk_count(n) - 1) / chunk_count(n)) + 31) / 32 * 32; }

template <typename T, int ACT>
static int dz_run(const void* dy, int64_t ldy, const void* pre, int64_t ldp, void* dz, int64_t ldz, int64_t rows,
                  int64_t n, void* db, float* part, cudaStream_t stream) {
  constexpr int V = 8;
  auto ok = [&](const void* q, int64_t ld) { return !q || (aligned16(q) && ld % V == 0); };
  const bool vec = n % V == 0 && ok(dy, ldy) && ok(pre, ldp) && ok(dz, ldz);
  const int64_t chunk = chunk_rows(rows, n), chunks = (rows + chunk - 1) / chunk;
  float* to = db ? part : nullptr;
  if (ACT != NONE || db) {
    if (vec)
      dz_kernel<T, V, ACT><<<dim3((unsigned)((n + 32 * V - 1) / (32 * V)), (unsigned)chunks), 256, 0, stream>>>(
          static_cast<const T*>(dy), ldy, static_cast<const T*>(pre), ldp, static_cast<T*>(dz), ldz, rows, n, chunk, to);
    else
      dz_kernel<T, 1, ACT><<<dim3((unsigned)((n + 31) / 32), (unsigned)chunks), 256, 0, stream>>>(
          static_cast<const T*>(dy), ldy, static_cast<const T*>(pre), ldp, static_cast<T*>(dz), ldz, rows, n, chunk, to);
    VDN_LAUNCH_CHECK("activation gradient");
  }
  if (db) return add_lines<T>(part, (int)chunks, n, static_cast<T*>(db), n, static_cast<T*>(nullptr), stream);
  return VDN_OK;
}

}  // namespace lact
}  // namespace vdn

using namespace vdn;

#define VDN_LACT_BY_ACT(T, fn, ...)                                      \
  switch (act) {                                                         \
    case VDN_ACT_NONE: return fn<T, VDN_ACT_NONE>(__VA_ARGS__);          \
    case VDN_ACT_GELU_TANH: return fn<T, VDN_ACT_GELU_TANH>(__VA_ARGS__); \
    case VDN_ACT_GELU_ERF: return fn<T, VDN_ACT_GELU_ERF>(__VA_ARGS__);  \
    case VDN_ACT_SILU: return fn<T, VDN_ACT_SILU>(__VA_ARGS__);          \
    default: return set_error(VDN_ERR_VALUE, "unknown activation %d", act); \
  }

extern "C" size_t vdn_linear_workspace_size(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows,
                                            int64_t n, int64_t k) {
  using namespace vdn::lact;
  if (rows < 1 || n < 1 || k < 1) return 0;
  return padded_bytes(x, ldx, rows, k) + padded_bytes(w, ldw, n, k);
}

extern "C" int vdn_linear_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                              const void* residual, int64_t ldr, int dtype, int act, int64_t rows, int64_t n,
                              int64_t k, void* y, int64_t ldy, void* pre, int64_t ldp, void* workspace,
                              size_t workspace_bytes, int* status, cudaStream_t stream) {
  using namespace vdn::lact;
  if (int rc = check(dtype, rows, n, k)) return rc;
  VDN_CHECK_ARG(act == NONE || act == TANH || act == ERF || act == SILU, "unknown activation %d", act);
  if (rows == 0) return VDN_OK;
  VDN_CHECK_ARG(x && w && y && ldy >= n && (!pre || ldp >= n), "null pointer or bad row stride");
  VDN_CHECK_ARG(residual != y && (!pre || (pre != y && pre != residual)), "y, pre and residual must not overlap");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (int rc = settle({{x, ldx, rows, k}, {w, ldw, n, k}}, ws, workspace_bytes, stream)) return rc;
  Params p = {};
  p.bias = bias;
  p.resid = residual;
  p.y = y;
  p.pre = pre;
  p.rows = rows;
  p.cols = n;
  p.ldr = ldr;
  p.ldy = ldy;
  p.ldp = ldp;
  p.status = status;
  if (dtype == VDN_DTYPE_BF16) {
    VDN_LACT_BY_ACT(__nv_bfloat16, forward, x, ldx, w, ldw, k, p, stream)
  } else {
    VDN_LACT_BY_ACT(__half, forward, x, ldx, w, ldw, k, p, stream)
  }
}

namespace vdn {
namespace lact {

// What the backward needs beside its outputs: dz (or dy) where the tensor maps cannot read dy
// itself, the bias gradient's partial sums, and x and w padded.
static size_t dz_bytes(const void* dy, int64_t ldy, int act, int64_t rows, int64_t n) {
  return act != NONE ? ((size_t)rows * pad8(n) * 2 + 255) / 256 * 256 : padded_bytes(dy, ldy, rows, n);
}
static size_t part_bytes(int64_t n) { return (sizeof(float) * (size_t)chunk_count(n) * (size_t)n + 255) / 256 * 256; }

template <typename T>
static int backward(const void* dy, int64_t ldy, const void* pre, int64_t ldp, const void* x, int64_t ldx,
                    const void* w, int64_t ldw, int act, int64_t rows, int64_t n, int64_t k, void* dx, int64_t lddx,
                    void* dw, int64_t lddw, void* db, uint8_t* ws, size_t left, int* status, cudaStream_t stream) {
  auto take = [&](size_t bytes) -> uint8_t* {
    if (!ws || bytes > left) return nullptr;
    uint8_t* at = ws;
    ws += bytes;
    left -= bytes;
    return at;
  };
  float* part = nullptr;
  if (db) {
    part = reinterpret_cast<float*>(take(part_bytes(n)));
    VDN_CHECK_ARG(part, "workspace smaller than vdn_linear_backward_workspace_size");
    VDN_CHECK_ARG(aligned_to(part, sizeof(float)), "the workspace must be 16-byte aligned");
  }
  const void* dz = dy;
  int64_t ldz = ldy;
  void* out = nullptr;
  if (act != NONE) {
    out = take(dz_bytes(dy, ldy, act, rows, n));
    VDN_CHECK_ARG(out, "workspace smaller than vdn_linear_backward_workspace_size");
    VDN_CHECK_ARG(aligned16(out), "the workspace must be 16-byte aligned");
    dz = out;
    ldz = pad8(n);
  }
  int rc = VDN_OK;
  switch (act) {
    case TANH: rc = dz_run<T, TANH>(dy, ldy, pre, ldp, out, ldz, rows, n, db, part, stream); break;
    case ERF: rc = dz_run<T, ERF>(dy, ldy, pre, ldp, out, ldz, rows, n, db, part, stream); break;
    case SILU: rc = dz_run<T, SILU>(dy, ldy, pre, ldp, out, ldz, rows, n, db, part, stream); break;
    default: rc = dz_run<T, NONE>(dy, ldy, pre, ldp, nullptr, ldz, rows, n, db, part, stream);
  }
  if (rc) return rc;
  if (dx) {
    if (int rc2 = settle({{dz, ldz, rows, n}, {w, ldw, n, k}}, ws, left, stream)) return rc2;
    Params p = {};
    p.y = dx;
    p.ldy = lddx;
    p.rows = rows;
    p.cols = k;
    p.status = status;
    if (int rc2 = product<T, false, true, NONE>({dz, ldz, false}, {w, ldw, true}, n, p, stream)) return rc2;
  }
  if (dw) {
    if (int rc2 = settle({{dz, ldz, rows, n}, {x, ldx, rows, k}}, ws, left, stream)) return rc2;
    Params p = {};
    p.y = dw;
    p.ldy = lddw;
    p.rows = n;
    p.cols = k;
    p.status = status;
    if (int rc2 = product<T, true, true, NONE>({dz, ldz, true}, {x, ldx, true}, rows, p, stream)) return rc2;
  }
  return VDN_OK;
}

}  // namespace lact
}  // namespace vdn

extern "C" size_t vdn_linear_backward_workspace_size(const void* dy, int64_t ldy, const void* x, int64_t ldx,
                                                     const void* w, int64_t ldw, int act, int64_t rows, int64_t n,
                                                     int64_t k) {
  using namespace vdn::lact;
  if (rows < 1 || n < 1 || k < 1) return 0;
  return part_bytes(n) + dz_bytes(dy, ldy, act, rows, n) + padded_bytes(x, ldx, rows, k) + padded_bytes(w, ldw, n, k);
}

extern "C" int vdn_linear_act_backward(const void* dy, int64_t ldy, const void* pre, int64_t ldp, const void* x,
                                       int64_t ldx, const void* w, int64_t ldw, int dtype, int act, int64_t rows,
                                       int64_t n, int64_t k, void* dx, int64_t lddx, void* dw, int64_t lddw,
                                       void* d_bias, void* workspace, size_t workspace_bytes, int* status,
                                       cudaStream_t stream) {
  using namespace vdn::lact;
  if (int rc = check(dtype, rows, n, k)) return rc;
  VDN_CHECK_ARG(act == NONE || act == TANH || act == ERF || act == SILU, "unknown activation %d", act);
  VDN_CHECK_ARG((!dx || lddx >= k) && (!dw || lddw >= k), "bad output row stride");
  if (rows == 0) {
    if (dw) VDN_CUDA_TRY(cudaMemset2DAsync(dw, (size_t)lddw * 2, 0, (size_t)k * 2, (size_t)n, stream));
    if (d_bias) VDN_CUDA_TRY(cudaMemsetAsync(d_bias, 0, (size_t)n * 2, stream));
    return VDN_OK;
  }
  VDN_CHECK_ARG(dy && (act == NONE || pre) && (!dx || w) && (!dw || x), "null pointer");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (dtype == VDN_DTYPE_BF16)
    return backward<__nv_bfloat16>(dy, ldy, pre, ldp, x, ldx, w, ldw, act, rows, n, k, dx, lddx, dw, lddw, d_bias, ws,
                                   workspace_bytes, status, stream);
  return backward<__half>(dy, ldy, pre, ldp, x, ldx, w, ldw, act, rows, n, k, dx, lddx, dw, lddw, d_bias, ws,
                          workspace_bytes, status, stream);
}
