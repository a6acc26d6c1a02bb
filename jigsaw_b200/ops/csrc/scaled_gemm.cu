// 8-bit matrix product with power-of-two block scales on the 5th-generation tensor cores.
//
//   out[m, n] = sum_k a[m, k] sa(m, k) * b[n, k] sb(n, k) + bias[n]
//
// a [M, K] and b [N, K] are e4m3 codes, K contiguous; a scale is one e8m0 byte (2^(byte - 127)) per 128 values of K
// and per row, or per 128 rows.  tcgen05.mma applies the scales itself (kind::mxf8f6f4.block_scale, one scale per 32
// values of K): every product of two codes and two scales is exact, and the sum stays in fp32 in TMEM from the first
// k-block to the last.  The 128-wide block is handed to the instruction by writing each scale byte four times.
//
// One CTA, twelve warps: warp 0 issues the TMA loads of the code tiles, warps 2 and 3 lay the scale bytes of the same
// k-block out in shared memory in the form that tcgen05.cp copies to TMEM (row r of a 128-row group at byte
// (r % 32) * 16 + (r / 32) * 4), warp 1 issues the copies and the products, warps 4..11 drain.  The drain reads a
// warp's whole share of the accumulator into registers and gives the TMEM columns back before it converts and stores,
// so that the products of the next tile run under the stores.
#include <type_traits>

#include "ptx.cuh"
#include "scaled_abi.h"
#include "tmap.cuh"

namespace jb {

// ---------------------------------------------------------------- instructions of this kernel
// Block-scaled instruction descriptor: e4m3 x e4m3, e8m0 scales (byte 0 of each TMEM word), fp32 accumulation, M = 128.
__host__ __device__ constexpr uint32_t make_idesc_mxf8(uint32_t N) {
  return ((N >> 3) << 17) | (1u << 23) | ((128u >> 7) << 27);
}
__device__ __forceinline__ void umma_mxf8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 32 rows of 16 bytes -> 32 lanes x 4 columns, repeated in all four lane quadrants.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// No swizzle: groups of eight 16-byte rows, 128 bytes apart.
__device__ __forceinline__ uint64_t make_smem_desc_scales(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) |
         (static_cast<uint64_t>(1) << 46);
}
__device__ __forceinline__ void cluster_arrive_wait() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t local_saddr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_saddr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// ---------------------------------------------------------------- arguments
enum : int { JB_T_F32 = 0, JB_T_BF16 = 1, JB_T_F16 = 2 };

__device__ __forceinline__ float load_typed(const void* p, int type, long long i) {
  if (type == JB_T_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (type == JB_T_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_typed(void* p, int type, long long i, float v) {
  if (type == JB_T_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(v);
  else if (type == JB_T_F16) static_cast<__half*>(p)[i] = __float2half(v);
  else static_cast<float*>(p)[i] = v;
}
__device__ __forceinline__ uint32_t pack_half16(float lo, float hi, int type) {
  if (type == JB_T_BF16) return pack_bf16x2(lo, hi);
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

struct ScaledOperand {       // scales of one operand: byte of (row r, k-block kb) at (r >> shift) * row + kb * k
  const uint8_t* scales;
  long long row, k;
  int shift;                 // 0: a scale per row, 7: per 128 rows
  int rows;
};
struct ScaledGemmArgs {
  ScaledOperand p, q;        // the operand along the accumulator's lanes (128 rows a tile), and along its columns
  void* out;
  long long ldo;             // elements between rows m of the output
  int out_type;
  const void* bias;          // [N] or null
  int bias_type;
  int kblocks;               // blocks of 128 along K
  int tiles_p, tiles_q;
  int vec_out;               // rows of the output start on 16-byte boundaries
};

constexpr int SG_BP = 128;
constexpr int SG_EPI_WARPS = 8;
constexpr int SG_THREADS = 32 * (4 + SG_EPI_WARPS);
constexpr int SG_PITCH = SG_BP + 1;          // floats between columns of a dumped accumulator

// BQ: columns of a tile.  JOIN: the accumulator goes through shared memory, where the CTAs of a cluster that share a
// tile (each with its own range of k-blocks) add their parts in rank order.
template <int BQ, bool JOIN>
struct SgSmem {
  static constexpr int Q_ATOMS = (BQ + 127) / 128;
  static constexpr int P_BYTES = SG_BP * 128;
  static constexpr int Q_BYTES = BQ * 128;
  static constexpr int TILE_BYTES = P_BYTES + Q_BYTES;             // multiples of 1024: swizzled operands
  static constexpr int SF_BYTES = 512 * (1 + Q_ATOMS);
  static constexpr int STAGES = BQ >= 256 ? 4 : (BQ >= 128 ? 6 : 8);
  static constexpr int ACCS = BQ >= 256 ? 1 : 2;
  static constexpr int SF_OFFSET = STAGES * TILE_BYTES;
  static constexpr int STAGE_OUT = SF_OFFSET + STAGES * SF_BYTES;  // 32 rows x 64 bytes per draining warp
  static constexpr int BAR_OFFSET = STAGE_OUT + (JOIN ? 0 : SG_EPI_WARPS * 2048);
  static constexpr int TOTAL = BAR_OFFSET + 256 + 1024;
  static_assert(TOTAL <= 227 * 1024, "shared memory of one CTA");
  static_assert(!JOIN || BQ * SG_PITCH * 4 <= SF_OFFSET, "the dumped accumulator reuses the tile buffers");
  static constexpr int SF_COL = ACCS * BQ < 32 ? 32 : ACCS * BQ;   // first TMEM column of the scales
  static_assert(SF_COL + STAGES * 4 * (1 + Q_ATOMS) <= 512, "TMEM columns");
};

// Position of tile t: groups of eight tile rows, walked down first, so that the CTAs of one wave share operand tiles.
__device__ __forceinline__ void sg_tile(int t, int tiles_p, int tiles_q, int& tp, int& tq) {
  const int group = 8 * tiles_q;
  const int g = t / group, first = g * 8;
  const int height = min(8, tiles_p - first);
  const int r = t - g * group;
  tp = first + r % height;
  tq = r / height;
}

// One warp writes the scale words of `atoms` groups of 128 rows for its share of k-blocks, four k-blocks of loads ahead
// of the stores (the loads' latency is several times a stage's time).
template <int ATOMS>
__device__ __forceinline__ void sg_load_scales(const ScaledOperand& o, int row0, int kb, int kend, uint32_t (&w)[ATOMS * 4], int lane) {
#pragma unroll
  for (int j = 0; j < ATOMS * 4; ++j) {
    const int r = row0 + 32 * j + lane;
    w[j] = 127u;
    if (r < o.rows && kb < kend) w[j] = __ldg(o.scales + static_cast<long long>(r >> o.shift) * o.row + kb * o.k);
  }
}

template <int BQ, bool SWAP, bool JOIN>
__global__ void __launch_bounds__(SG_THREADS, 1)
scaled_gemm_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ, const ScaledGemmArgs a,
                   int* status) {
  using S = SgSmem<BQ, JOIN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BAR_OFFSET);
  uint64_t* full = bars;                               // [STAGES]: TMA bytes and two scale warps
  uint64_t* empty = bars + S::STAGES;                  // [STAGES]
  uint64_t* acc_full = bars + 2 * S::STAGES;           // [ACCS]
  uint64_t* acc_empty = acc_full + S::ACCS;            // [ACCS]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + S::ACCS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * S::STAGES + 2 * S::ACCS) * 8 + 8 <= 256, "barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full[s], 3);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < S::ACCS; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], SG_EPI_WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmP);
    tma_prefetch_desc(&tmQ);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  // The CTAs of a cluster (JOIN) take one tile together and cut its k-blocks into consecutive ranges; otherwise a CTA
  // takes whole tiles in steps of the grid.
  const int tiles = a.tiles_p * a.tiles_q;
  int kb0 = 0, kb1 = a.kblocks, first_tile = blockIdx.x, step = gridDim.x;
  uint32_t split = 1, rank = 0;
  if constexpr (JOIN) {
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(split));
    rank = cluster_rank();
    first_tile = blockIdx.x / split;
    step = tiles;
    kb0 = static_cast<int>(static_cast<long long>(a.kblocks) * rank / split);
    kb1 = static_cast<int>(static_cast<long long>(a.kblocks) * (rank + 1) / split);
  }

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = first_tile; t < tiles && ok; t += step) {
        int tp, tq;
        sg_tile(t, a.tiles_p, a.tiles_q, tp, tq);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&empty[s], ph ^ 1u, abort_flag, status, 1);
          if (!ok) break;
          uint8_t* dst = smem + s * S::TILE_BYTES;
          mbar_expect_tx(&full[s], S::TILE_BYTES);
          tma_load_2d(dst, &tmP, &full[s], kb * 128, tp * SG_BP);
          tma_load_2d(dst + S::P_BYTES, &tmQ, &full[s], kb * 128, tq * BQ);
          if (++s == S::STAGES) { s = 0; ph ^= 1u; }
        }
      }
      if (!ok) {                       // a wait gave up: let the copies already issued arrive before the CTA ends
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
      }
    }
  } else if (warp == 2 || warp == 3) {
    // ------------------------------------------------------------ scale bytes
    auto run = [&](auto atoms_c, const ScaledOperand& o, int rows_per_tile, bool is_q, int offset) {
      constexpr int ATOMS = decltype(atoms_c)::value;
      constexpr int AHEAD = 4;
      int s = 0;
      uint32_t ph = 0;
      for (int t = first_tile; t < tiles; t += step) {
        int tp, tq;
        sg_tile(t, a.tiles_p, a.tiles_q, tp, tq);
        const int row0 = (is_q ? tq : tp) * rows_per_tile;
        uint32_t w[AHEAD][ATOMS * 4];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) sg_load_scales<ATOMS>(o, row0, kb0 + i, kb1, w[i], lane);
        for (int kb = kb0; kb < kb1; kb += AHEAD) {
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {
            if (kb + i < kb1) {
              mbar_wait(&empty[s], ph ^ 1u, abort_flag, status, 2);
              uint8_t* dst = smem + S::SF_OFFSET + s * S::SF_BYTES + offset;
#pragma unroll
              for (int g = 0; g < ATOMS; ++g) {
                uint4 v;
                v.x = w[i][4 * g] * 0x01010101u;
                v.y = w[i][4 * g + 1] * 0x01010101u;
                v.z = w[i][4 * g + 2] * 0x01010101u;
                v.w = w[i][4 * g + 3] * 0x01010101u;
                *reinterpret_cast<uint4*>(dst + g * 512 + lane * 16) = v;
              }
              sg_load_scales<ATOMS>(o, row0, kb + i + AHEAD, kb1, w[i], lane);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&full[s]);
              if (++s == S::STAGES) { s = 0; ph ^= 1u; }
            }
          }
        }
      }
    };
    if (warp == 2) run(std::integral_constant<int, 1>{}, a.p, SG_BP, false, 0);
    else run(std::integral_constant<int, S::Q_ATOMS>{}, a.q, BQ, true, 512);
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    constexpr uint32_t idesc = make_idesc_mxf8(BQ);
    int s = 0, it = 0;
    uint32_t ph = 0;
    const uint32_t base = smem_u32(smem);
    const uint64_t pd0 = make_smem_desc_sw128(base, 16, 1024);
    const uint64_t qd0 = make_smem_desc_sw128(base + S::P_BYTES, 16, 1024);
    const uint64_t sd0 = make_smem_desc_scales(base + S::SF_OFFSET);
    for (int t = first_tile; t < tiles; t += step, ++it) {
      const int as = it % S::ACCS;
      const uint32_t aph = static_cast<uint32_t>(it / S::ACCS) & 1u;
      mbar_wait(&acc_empty[as], aph ^ 1u, abort_flag, status, 3);
      tc_fence_after_sync();
      const uint32_t d = tmem + static_cast<uint32_t>(as * BQ);
      for (int kb = kb0; kb < kb1; ++kb) {
        mbar_wait(&full[s], ph, abort_flag, status, 4);
        tc_fence_after_sync();
        const uint64_t pd = desc_advance(pd0, static_cast<uint32_t>(s * S::TILE_BYTES));
        const uint64_t qd = desc_advance(qd0, static_cast<uint32_t>(s * S::TILE_BYTES));
        const uint64_t sd = desc_advance(sd0, static_cast<uint32_t>(s * S::SF_BYTES));
        const uint32_t sfp = tmem + S::SF_COL + static_cast<uint32_t>(s * 4 * (1 + S::Q_ATOMS));
        const uint32_t sfq = sfp + 4;
        if (elect_one()) {
          tmem_cp_scales(sfp, sd);
#pragma unroll
          for (int g = 0; g < S::Q_ATOMS; ++g) tmem_cp_scales(sfq + 4 * g, desc_advance(sd, 512 * (1 + g)));
#pragma unroll
          for (int k = 0; k < 4; ++k)          // 32 codes = 32 bytes of the swizzled row
            umma_mxf8(d, desc_advance(pd, k * 32), desc_advance(qd, k * 32), idesc, sfp, sfq, (kb > kb0 || k != 0) ? 1u : 0u);
          umma_commit(&empty[s]);
        }
        __syncwarp();
        if (++s == S::STAGES) { s = 0; ph ^= 1u; }
      }
      umma_commit_elect(&acc_full[as]);
    }
  } else {
    // ------------------------------------------------------------ drain
    const int quad = warp & 3, half = (warp - 4) >> 2;
    constexpr int COLS = BQ / 2 < 16 ? 16 : BQ / 2;       // columns per warp (the narrowest tile is drained by four warps)
    const bool drains = BQ >= 32 || half == 0;
    const int c_first = BQ >= 32 ? half * COLS : 0;
    int it = 0;
    for (int t = first_tile; t < tiles; t += step, ++it) {
      const int as = it % S::ACCS;
      const uint32_t aph = static_cast<uint32_t>(it / S::ACCS) & 1u;
      int tp, tq;
      sg_tile(t, a.tiles_p, a.tiles_q, tp, tq);
      mbar_wait(&acc_full[as], aph, abort_flag, status, 5);
      tc_fence_after_sync();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(as * BQ + c_first);
      uint32_t raw[COLS];
      if (drains) {
#pragma unroll
        for (int c = 0; c < COLS; c += 16) tmem_ld_32x16(taddr + c, *reinterpret_cast<uint32_t(*)[16]>(&raw[c]));
        tmem_ld_wait();
      }
      float acc[COLS];
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        asm volatile("" : "+r"(raw[c]));          // no use above the wait
        acc[c] = __uint_as_float(raw[c]);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[as]);
      if constexpr (JOIN) {
        // every product of this CTA is done (acc_full), so the tile buffers are free
        float* dump = reinterpret_cast<float*>(smem);
        if (drains) {
#pragma unroll
          for (int c = 0; c < COLS; ++c) dump[(c_first + c) * SG_PITCH + quad * 32 + lane] = acc[c];
        }
      } else {
        const int row0 = tp * SG_BP + quad * 32;           // rows of the output (p runs along m here)
        const int col0 = tq * BQ + c_first;
        uint8_t* stage = smem + S::STAGE_OUT + (warp - 4) * 2048;
        const int rows = a.p.rows - row0, width = a.q.rows;
        if (a.out_type == JB_T_F32) {
#pragma unroll
          for (int c = 0; c < COLS; c += 16) {
            const int col = col0 + c;
            if (col < width && rows > 0) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) =
                    make_float4(acc[c + 4 * i], acc[c + 4 * i + 1], acc[c + 4 * i + 2], acc[c + 4 * i + 3]);
              __syncwarp();
              float* dst = static_cast<float*>(a.out) + static_cast<long long>(row0) * a.ldo + col;
              if (a.vec_out && col + 16 <= width) {
                const int piece = lane & 3;
                float b[4] = {0.f, 0.f, 0.f, 0.f};
                if (a.bias != nullptr) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) b[e] = load_typed(a.bias, a.bias_type, col + piece * 4 + e);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int r = i * 8 + (lane >> 2);
                  float4 o = *reinterpret_cast<const float4*>(stage + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
                  o.x += b[0]; o.y += b[1]; o.z += b[2]; o.w += b[3];
                  if (r < rows) *reinterpret_cast<float4*>(dst + static_cast<long long>(r) * a.ldo + piece * 4) = o;
                }
              } else {
                const int e = lane & 15;
                const bool in = col + e < width;
                const float b = (a.bias != nullptr && in) ? load_typed(a.bias, a.bias_type, col + e) : 0.f;
#pragma unroll 4
                for (int r = lane >> 4; r < 32; r += 2) {
                  const float v = *reinterpret_cast<const float*>(stage + r * 64 + (((e >> 2) ^ ((r >> 1) & 3)) << 4) + (e & 3) * 4);
                  if (in && r < rows) dst[static_cast<long long>(r) * a.ldo + e] = v + b;
                }
              }
              __syncwarp();
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < COLS; c += 32) {
            const int col = col0 + c;
            if (col < width && rows > 0) {
              if (a.bias != nullptr) {          // before the rounding: every lane needs all 32 values
                const float mine = col + lane < width ? load_typed(a.bias, a.bias_type, col + lane) : 0.f;
#pragma unroll
                for (int e = 0; e < 32; ++e) acc[c + e] += __shfl_sync(0xffffffffu, mine, e);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint4 o;
                o.x = pack_half16(acc[c + 8 * i], acc[c + 8 * i + 1], a.out_type);
                o.y = pack_half16(acc[c + 8 * i + 2], acc[c + 8 * i + 3], a.out_type);
                o.z = pack_half16(acc[c + 8 * i + 4], acc[c + 8 * i + 5], a.out_type);
                o.w = pack_half16(acc[c + 8 * i + 6], acc[c + 8 * i + 7], a.out_type);
                *reinterpret_cast<uint4*>(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = o;
              }
              __syncwarp();
              uint16_t* dst = static_cast<uint16_t*>(a.out) + static_cast<long long>(row0) * a.ldo + col;
              if (a.vec_out && col + 32 <= width) {
                const int piece = lane & 3;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int r = i * 8 + (lane >> 2);
                  const uint4 o = *reinterpret_cast<const uint4*>(stage + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
                  if (r < rows) *reinterpret_cast<uint4*>(dst + static_cast<long long>(r) * a.ldo + piece * 8) = o;
                }
              } else {
#pragma unroll 4
                for (int r = 0; r < 32; ++r) {
                  const uint16_t v =
                      *reinterpret_cast<const uint16_t*>(stage + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
                  if (col + lane < width && r < rows) dst[static_cast<long long>(r) * a.ldo + lane] = v;
                }
              }
              __syncwarp();
            }
          }
        }
      }
    }
  }

  if constexpr (JOIN) {
    // The parts of a tile meet in the shared memory of the cluster; CTA `rank` finishes its share of the output's
    // columns (SWAP: of the tile's columns, which are rows of the output), always adding the parts in rank order.
    __syncthreads();
    __syncwarp();
    cluster_arrive_wait();
    const uint32_t dump = smem_u32(smem);
    int tp, tq;
    sg_tile(first_tile, a.tiles_p, a.tiles_q, tp, tq);
    if constexpr (SWAP) {          // p runs along n, q along m: lanes along n
      const int n = tp * SG_BP + (threadIdx.x & 127);
      const float b = (a.bias != nullptr && n < a.p.rows) ? load_typed(a.bias, a.bias_type, n) : 0.f;
      const int live = min(BQ, a.q.rows - tq * BQ);
      for (int c = static_cast<int>(rank) * 3 + (threadIdx.x >> 7); c < live; c += 3 * static_cast<int>(split)) {
        float v = 0.f;
        for (uint32_t r = 0; r < split; ++r) v += ld_cluster_f32(dump + (c * SG_PITCH + (threadIdx.x & 127)) * 4, r);
        if (n < a.p.rows) store_typed(a.out, a.out_type, static_cast<long long>(tq * BQ + c) * a.ldo + n, v + b);
      }
    } else {                        // lanes along the columns of the tile
      for (int c0 = 0; c0 < BQ; c0 += 32) {
        const int c = c0 + lane, n = tq * BQ + c;
        const float b = (a.bias != nullptr && n < a.q.rows) ? load_typed(a.bias, a.bias_type, n) : 0.f;
        for (int i = static_cast<int>(rank) * (SG_THREADS / 32) + warp; i < SG_BP; i += static_cast<int>(split) * (SG_THREADS / 32)) {
          float v = 0.f;
          for (uint32_t r = 0; r < split; ++r) v += ld_cluster_f32(dump + (c * SG_PITCH + i) * 4, r);
          const int m = tp * SG_BP + i;
          if (m < a.p.rows && n < a.q.rows) store_typed(a.out, a.out_type, static_cast<long long>(m) * a.ldo + n, v + b);
        }
      }
    }
    cluster_arrive_wait();          // no CTA leaves while another one reads its shared memory
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// 8-bit codes [rows, K], K contiguous, `pitch` bytes between rows; a box of 128 codes x `box_rows` rows, 128-byte swizzle.
static int make_tmap_codes(CUtensorMap* out, const void* base, long long rows, long long K, long long pitch, int box_rows) {
  EncodeTiledFn fn = get_encode_tiled();
  if (fn == nullptr) return -1;
  ensure_current_context();
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t es[2] = {1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -2;
}

template <int BQ, bool SWAP, bool JOIN>
static int launch_scaled_gemm(const void* P, long long pitch_p, const void* Q, long long pitch_q, long long K, ScaledGemmArgs a,
                              int split, int sm_count, int* status, cudaStream_t stream) {
  using S = SgSmem<BQ, JOIN>;
  CUtensorMap tmP, tmQ;
  if (make_tmap_codes(&tmP, P, a.p.rows, K, pitch_p, SG_BP) != 0) return -2;
  if (make_tmap_codes(&tmQ, Q, a.q.rows, K, pitch_q, BQ) != 0) return -2;
  a.tiles_p = (a.p.rows + SG_BP - 1) / SG_BP;
  a.tiles_q = (a.q.rows + BQ - 1) / BQ;
  auto kern = scaled_gemm_kernel<BQ, SWAP, JOIN>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL) != cudaSuccess) return -3;
  const long long tiles = static_cast<long long>(a.tiles_p) * a.tiles_q;
  if (tiles * split > 0x7fffffffLL) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(JOIN ? tiles * split : (tiles < sm_count ? tiles : sm_count)));
  cfg.blockDim = dim3(SG_THREADS);
  cfg.dynamicSmemBytes = S::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = JOIN ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, tmP, tmQ, a, status) == cudaSuccess ? 0 : -4;
}

}  // namespace jb

extern "C" int jb_scaled_gemm(const JbScaledOperand* a, const JbScaledOperand* b, long long K, void* out, long long ldo,
                              int out_type, const void* bias, int bias_type, int sm_count, int* status, void* stream) {
  using namespace jb;
  if (a == nullptr || b == nullptr || a->rows < 1 || b->rows < 1 || K < 1 || K > 0x7fffff00LL || sm_count < 1) return -1;
  if ((a->pitch & 15) || (b->pitch & 15) || (reinterpret_cast<uintptr_t>(a->codes) & 15) || (reinterpret_cast<uintptr_t>(b->codes) & 15)) return -1;
  if (out_type < 0 || out_type > 2 || bias_type < 0 || bias_type > 2) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ScaledGemmArgs g{};
  const ScaledOperand oa{static_cast<const uint8_t*>(a->scales), a->scale_row, a->scale_k, a->square ? 7 : 0, a->rows};
  const ScaledOperand ob{static_cast<const uint8_t*>(b->scales), b->scale_row, b->scale_k, b->square ? 7 : 0, b->rows};
  g.out = out; g.ldo = ldo; g.out_type = out_type; g.bias = bias; g.bias_type = bias_type;
  g.kblocks = static_cast<int>((K + 127) / 128);
  const int size = out_type == JB_T_F32 ? 4 : 2;
  g.vec_out = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (ldo * size) % 16 == 0;
  const int M = a->rows, N = b->rows;
  if (M <= 64) {
    // few rows: the weight's rows go along the 128 lanes, and several CTAs share a tile's K range until the SMs are busy
    g.p = ob; g.q = oa;
    const int tiles = (N + 127) / 128;
    int split = 1;
    while (split < 8 && tiles * split * 2 <= sm_count && g.kblocks >= split * 4) split *= 2;
    if (M <= 16) return launch_scaled_gemm<16, true, true>(b->codes, b->pitch, a->codes, a->pitch, K, g, split, sm_count, status, st);
    if (M <= 32) return launch_scaled_gemm<32, true, true>(b->codes, b->pitch, a->codes, a->pitch, K, g, split, sm_count, status, st);
    return launch_scaled_gemm<64, true, true>(b->codes, b->pitch, a->codes, a->pitch, K, g, split, sm_count, status, st);
  }
  g.p = oa; g.q = ob;
  const long long tiles256 = static_cast<long long>((M + 127) / 128) * ((N + 255) / 256);
  if (tiles256 >= sm_count) return launch_scaled_gemm<256, false, false>(a->codes, a->pitch, b->codes, b->pitch, K, g, 1, sm_count, status, st);
  const long long tiles128 = static_cast<long long>((M + 127) / 128) * ((N + 127) / 128);
  int split = 1;
  while (split < 8 && tiles128 * split * 2 <= sm_count && g.kblocks >= split * 8) split *= 2;
  if (split > 1) return launch_scaled_gemm<128, false, true>(a->codes, a->pitch, b->codes, b->pitch, K, g, split, sm_count, status, st);
  return launch_scaled_gemm<128, false, false>(a->codes, a->pitch, b->codes, b->pitch, K, g, 1, sm_count, status, st);
}
