// 8-bit matrix product with power-of-two block scales on the 5th-generation tensor cores.
//
//   out[m, n] = sum_k a[m, k] sa(m, k) * b[n, k] sb(n, k) + bias[n]
//
// a [M, K] and b [N, K] are e4m3 codes, K contiguous; a scale is one e8m0 byte (2^(byte - 127)) per 128 values of K
// and per row, or per 128 rows.  tcgen05.mma applies the scales itself (kind::mxf8f6f4.block_scale, one scale per 32
// values of K): every product of two codes and two scales is exact, and the sum stays in fp32 in TMEM.  A TMEM word holds
// the scale bytes of one row for four k-blocks; the four products of a k-block all name its byte.
//
// Twelve warps a CTA: warp 0 issues the TMA loads of the code tiles, warps 2 and 3 lay the scale words of four k-blocks
// out in shared memory in the form that tcgen05.cp copies to TMEM (row r of a 128-row group at byte
// (r % 32) * 16 + (r / 32) * 4), warp 1 issues the copies and the products, warps 4..11 drain.  The drain reads a
// warp's whole share of the accumulator into registers and gives the TMEM columns back before it converts and stores,
// so that the products of the next tile run under the stores.
//
// Three forms:
//  * PAIR: two CTAs of a cluster share a tile of 256 rows (cta_group::2); each loads its 128 rows of one operand and
//    half of the other, so that a k-block costs 32 KB of loads an SM instead of 48 KB.
//  * JOIN: a tile's k-blocks are cut over the CTAs of a cluster; the parts are pushed into the shared memory of the CTA
//    that finishes them and added in rank order.  For products with fewer tiles than SMs.
//  * SWAP (with JOIN): few rows (a token, a short batch): the weight's rows go along the 128 lanes.
#include <type_traits>

#include "ptx.cuh"
#include "scaled_abi.h"
#include "tmap.cuh"

namespace jb {

// ---------------------------------------------------------------- instructions of this kernel
// Block-scaled instruction descriptor: e4m3 x e4m3, e8m0 scales in byte `byte` of each TMEM word, fp32 accumulation, M = 128
// or 256.
__host__ __device__ constexpr uint32_t make_idesc_mxf8(uint32_t M, uint32_t N, uint32_t byte) {
  return (byte << 4) | ((N >> 3) << 17) | (1u << 23) | ((M >> 7) << 27) | (byte << 29);
}
template <bool PAIR>
__device__ __forceinline__ void umma_mxf8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// 32 rows of 16 bytes -> 32 lanes x 4 columns, repeated in all four lane quadrants (of each CTA, from its own shared memory).
template <bool PAIR>
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Arrive on the mbarrier (of both CTAs) once the tcgen05 work issued so far has finished.
template <bool PAIR>
__device__ __forceinline__ void sg_commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
  else umma_commit(bar);
}
// Arrive on the same mbarrier of the cluster's CTA 0.  What the arrival announces (tiles and scales in this CTA's own shared
// memory, or TMEM columns read) is complete by then and is not read by the other CTA's threads, only by the tensor
// cores; a release at cluster scope would wait for every store of the thread and cost 0.9 us a k-block.
__device__ __forceinline__ void mbar_arrive_leader(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %0, 0;\n\t"
      "mbarrier.arrive.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}
// No swizzle: groups of eight 16-byte rows, 128 bytes apart.
__device__ __forceinline__ uint64_t make_smem_desc_scales(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) |
         (static_cast<uint64_t>(1) << 46);
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address of the same shared-memory place in another CTA of the cluster, and a store there.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t local_saddr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_saddr), "r"(rank));
  return remote;
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_f32x4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
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
  int words;                 // k = 1, base and `row` multiples of four: four k-blocks are one aligned word
};
struct ScaledGemmArgs {
  ScaledOperand p, q;        // the operand along the accumulator's lanes (128 rows a tile), and along its columns
  void* out;
  long long ldo;             // elements between rows m of the output
  int out_type;
  const void* bias;          // [N] or null
  int bias_type;
  int kblocks;               // blocks of 128 along K
  int chunk;                 // k-blocks summed in TMEM before the drain adds them up
  int tiles_p, tiles_q;
  int vec_out;               // rows of the output start on 16-byte boundaries
};

constexpr int SG_BP = 128;                   // rows of the operand along the lanes, per CTA
constexpr int SG_EPI_WARPS = 8;
constexpr int SG_THREADS = 32 * (4 + SG_EPI_WARPS);
constexpr int SG_PITCH = SG_BP + 1;          // floats between columns of a part in shared memory (SWAP)

// BQ: columns of a tile.
template <int BQ, bool PAIR, bool JOIN>
struct SgSmem {
  static constexpr int Q_ATOMS = (BQ + 127) / 128;
  static constexpr int Q_ROWS = PAIR ? BQ / 2 : BQ;                // rows of the second operand that this CTA loads
  static constexpr int P_BYTES = SG_BP * 128;
  static constexpr int TILE_BYTES = P_BYTES + Q_ROWS * 128;        // multiples of 1024: swizzled operands
  static constexpr int SF_BYTES = 512 * (1 + Q_ATOMS);             // scale words of four k-blocks
  static constexpr int SF_SLOTS = 3;
  // Narrow tiles are bound by the hand-overs and by the latency of dependent products (16 columns: 90 cycles a product, of
  // which a k-block has four): two k-blocks a stage, and the products take turns between two accumulators.
  static constexpr int KPS = BQ <= 64 ? 2 : 1;                     // k-blocks a stage
  static constexpr bool DUAL = BQ <= 64;
  static constexpr int STAGES = TILE_BYTES >= 49152 ? 4 : TILE_BYTES >= 32768 ? (JOIN ? 4 : 6) : BQ >= 64 ? 3 : 4;
  static constexpr int ACCS = BQ >= 256 || DUAL ? 1 : 2;           // tiles in TMEM
  static constexpr int SF_OFFSET = STAGES * KPS * TILE_BYTES;
  static constexpr int OUT_OFFSET = SF_OFFSET + SF_SLOTS * SF_BYTES;
  // plain: 32 rows x 64 bytes per draining warp; JOIN: the parts of BQ / split columns from each CTA, by columns (SWAP), or by
  // rows with four floats between them (split up to 4)
  static constexpr int OUT_BYTES = !JOIN ? SG_EPI_WARPS * 2048 : BQ <= 64 ? (BQ * SG_PITCH * 4 + 15) / 16 * 16 : SG_BP * (BQ + 16) * 4;
  static constexpr int BIAS_OFFSET = OUT_OFFSET + OUT_BYTES;       // plain: the bias of a draining warp's columns
  static constexpr int BIAS_BYTES = JOIN ? 0 : SG_EPI_WARPS * (BQ / 2) * 4;
  static constexpr int BAR_OFFSET = BIAS_OFFSET + BIAS_BYTES;
  static constexpr int BARS = 2 * STAGES + 2 * SF_SLOTS + 2 * ACCS;
  static constexpr int TOTAL = BAR_OFFSET + 256 + 1024;
  static_assert(TOTAL <= 227 * 1024, "shared memory of one CTA");
  static_assert(BARS * 8 + 8 <= 256, "barriers");
  static constexpr int SF_COL = (DUAL ? 2 : ACCS) * BQ;            // first TMEM column of the scales
  static constexpr int SF_COLS = 4 * (1 + Q_ATOMS);
  static_assert(SF_COL + SF_SLOTS * SF_COLS <= 512, "TMEM columns");
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

// Scale bytes of one row for the k-blocks kb .. kb + 3 (those below kend).
__device__ __forceinline__ uint32_t sg_scale_word(const ScaledOperand& o, int r, int kb, int kend) {
  const uint8_t* p = o.scales + static_cast<long long>(r >> o.shift) * o.row + kb * o.k;
  if (o.words && kb + 4 <= kend) return __ldg(reinterpret_cast<const uint32_t*>(p));
  uint32_t w = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (kb + j < kend) w |= static_cast<uint32_t>(__ldg(p + j * o.k)) << (8 * j);
  return w;
}
// The words of `ATOMS` groups of 128 rows from row0 on, lane l: rows l, 32 + l, 64 + l, 96 + l of each.  A group whose rows
// share their scales (tiles start on multiples of their height, which divides 128 or is a multiple of it) is one word.
template <int ATOMS>
__device__ __forceinline__ void sg_scale_words(const ScaledOperand& o, int row0, int kb, int kend, uint32_t (&w)[ATOMS * 4], int lane) {
#pragma unroll
  for (int g = 0; g < ATOMS; ++g) {
    if (o.shift != 0) {
      const uint32_t v = row0 + 128 * g < o.rows && kb < kend ? sg_scale_word(o, row0 + 128 * g, kb, kend) : 0x7f7f7f7fu;
      w[4 * g] = w[4 * g + 1] = w[4 * g + 2] = w[4 * g + 3] = v;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = row0 + 128 * g + 32 * j + lane;
        w[4 * g + j] = r < o.rows && kb < kend ? sg_scale_word(o, r, kb, kend) : 0x7f7f7f7fu;
      }
    }
  }
}

template <int BQ, bool PAIR, bool SWAP, bool JOIN>
__global__ void __launch_bounds__(SG_THREADS, 1)
scaled_gemm_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ, const ScaledGemmArgs a,
                   int* status) {
  static_assert(!(PAIR && JOIN) && (JOIN || !SWAP) && SWAP == (BQ <= 64), "forms");
  using S = SgSmem<BQ, PAIR, JOIN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BAR_OFFSET);
  uint64_t* full = bars;                               // [STAGES]: TMA bytes (and the other CTA's)
  uint64_t* empty = bars + S::STAGES;                  // [STAGES]
  uint64_t* sf_full = bars + 2 * S::STAGES;            // [SF_SLOTS]: two scale warps (and the other CTA's two)
  uint64_t* sf_empty = sf_full + S::SF_SLOTS;          // [SF_SLOTS]
  uint64_t* acc_full = sf_empty + S::SF_SLOTS;         // [ACCS]
  uint64_t* acc_empty = acc_full + S::ACCS;            // [ACCS]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + S::ACCS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t split = 1, rank = 0;
  if constexpr (JOIN) asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(split));
  if constexpr (JOIN || PAIR) rank = cluster_rank();

  // The CTAs of a cluster (JOIN) take one tile together and cut its k-blocks into consecutive ranges; otherwise a CTA
  // or pair takes whole tiles in steps of the grid.
  const int tiles = a.tiles_p * a.tiles_q;
  int kb0 = 0, kb1 = a.kblocks, first_tile = blockIdx.x, step = gridDim.x;
  if constexpr (JOIN) {
    first_tile = blockIdx.x / split;
    step = tiles;
    const int quads = (a.kblocks + 3) / 4;                 // ranges start on whole scale words
    kb0 = static_cast<int>(4LL * (static_cast<long long>(quads) * rank / split));
    kb1 = min(a.kblocks, static_cast<int>(4LL * (static_cast<long long>(quads) * (rank + 1) / split)));
  }
  if constexpr (PAIR) {
    first_tile = blockIdx.x >> 1;
    step = gridDim.x >> 1;
  }
  const int p_off = PAIR ? static_cast<int>(rank) * SG_BP : 0;            // of this CTA within a tile
  const int q_off = PAIR ? static_cast<int>(rank) * S::Q_ROWS : 0;
  constexpr int P_TILE = PAIR ? 2 * SG_BP : SG_BP;

  auto load_stage = [&](int s, int kb, int tp, int tq) {          // k-blocks kb .. kb + KPS - 1 below kb1
    const int n = min(S::KPS, kb1 - kb);
    mbar_expect_tx(&full[s], n * S::TILE_BYTES);
#pragma unroll
    for (int j = 0; j < S::KPS; ++j) {
      if (j < n) {
        uint8_t* dst = smem + (s * S::KPS + j) * S::TILE_BYTES;
        tma_load_2d(dst, &tmP, &full[s], (kb + j) * 128, tp * P_TILE + p_off);
        tma_load_2d(dst + S::P_BYTES, &tmQ, &full[s], (kb + j) * 128, tq * BQ + q_off);
      }
    }
  };

  int early = 0;             // stages of the first tile whose loads are issued before the CTA has met
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full[s], PAIR && rank == 0 ? 2 : 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < S::SF_SLOTS; ++s) {
      mbar_init(&sf_full[s], PAIR ? 4 : 2);
      mbar_init(&sf_empty[s], 1);
    }
    for (int s = 0; s < S::ACCS; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], PAIR ? 2 * SG_EPI_WARPS : SG_EPI_WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
    grid_dependency_wait();
    if (first_tile < tiles) {
      int tp, tq;
      sg_tile(first_tile, a.tiles_p, a.tiles_q, tp, tq);
      for (; early < S::STAGES && kb0 + early * S::KPS < kb1; ++early) load_stage(early, kb0 + early * S::KPS, tp, tq);
    }
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (PAIR) {      // barriers of both CTAs are set up before either arrives on the other's
    cluster_arrive();
    cluster_wait();
  }
  if constexpr (JOIN)
    if (split > 1) cluster_arrive();           // waited for before the first push into another CTA
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();

  if (warp == 0) {
    if (lane == 0) {
      int s = early == S::STAGES ? 0 : early;
      uint32_t ph = early == S::STAGES ? 1u : 0u;
      bool ok = true;
      int skip = early;
      for (int t = first_tile; t < tiles && ok; t += step) {
        int tp, tq;
        sg_tile(t, a.tiles_p, a.tiles_q, tp, tq);
        for (int kb = kb0 + skip * S::KPS; kb < kb1; kb += S::KPS) {
          ok = mbar_wait(&empty[s], ph ^ 1u, abort_flag, status, 1);
          if (!ok) break;
          load_stage(s, kb, tp, tq);
          if (++s == S::STAGES) { s = 0; ph ^= 1u; }
        }
        skip = 0;
      }
      if (!ok) {                       // a wait gave up: let the copies already issued arrive before the CTA ends
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
      }
    }
  } else if (warp == 2 || warp == 3) {
    // ------------------------------------------------------------ scale words
    // The words of the next four k-blocks are loaded before the present ones are handed over: the fence in front of the
    // hand-over waits for loads in flight, and once in four k-blocks that is hidden.
    auto run = [&](auto atoms_c, const ScaledOperand& o, bool is_q, int offset) {
      constexpr int ATOMS = decltype(atoms_c)::value;
      int s = 0;
      uint32_t ph = 0;
      uint32_t w[ATOMS * 4], next[ATOMS * 4];
      auto row_of = [&](int t) {
        int tp, tq;
        sg_tile(t, a.tiles_p, a.tiles_q, tp, tq);
        return is_q ? tq * BQ : tp * P_TILE + p_off;
      };
      int row0 = 0;
      if (first_tile < tiles) {
        row0 = row_of(first_tile);
        sg_scale_words<ATOMS>(o, row0, kb0, kb1, next, lane);
      }
      for (int t = first_tile; t < tiles; t += step) {
        for (int kb = kb0; kb < kb1; kb += 4) {
#pragma unroll
          for (int j = 0; j < ATOMS * 4; ++j) w[j] = next[j];
          mbar_wait(&sf_empty[s], ph ^ 1u, abort_flag, status, 2);
          uint8_t* dst = smem + S::SF_OFFSET + s * S::SF_BYTES + offset;
#pragma unroll
          for (int g = 0; g < ATOMS; ++g)
            *reinterpret_cast<uint4*>(dst + g * 512 + lane * 16) = make_uint4(w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (PAIR && rank == 1) mbar_arrive_leader(&sf_full[s]);
            else mbar_arrive(&sf_full[s]);
          }
          if (kb + 4 < kb1) {
            sg_scale_words<ATOMS>(o, row0, kb + 4, kb1, next, lane);
          } else if (t + step < tiles) {
            row0 = row_of(t + step);
            sg_scale_words<ATOMS>(o, row0, kb0, kb1, next, lane);
          }
          if (++s == S::SF_SLOTS) { s = 0; ph ^= 1u; }
        }
      }
    };
    if (warp == 2) run(std::integral_constant<int, 1>{}, a.p, false, 0);
    else run(std::integral_constant<int, S::Q_ATOMS>{}, a.q, true, 512);
  } else if (warp == 1 && PAIR && rank == 1) {
    // ------------------------------------------------------------ this CTA's stages are ready: tell the issuing CTA
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      for (int t = first_tile; t < tiles; t += step)
        for (int kb = kb0; kb < kb1; ++kb) {
          mbar_wait(&full[s], ph, abort_flag, status, 6);
          mbar_arrive_leader(&full[s]);
          if (++s == S::STAGES) { s = 0; ph ^= 1u; }
        }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    int s = 0, it = 0, f = 0;
    uint32_t ph = 0, fph = 0;
    const uint32_t base = smem_u32(smem);
    const uint64_t pd0 = make_smem_desc_sw128(base, 16, 1024);
    const uint64_t qd0 = make_smem_desc_sw128(base + S::P_BYTES, 16, 1024);
    const uint64_t sd0 = make_smem_desc_scales(base + S::SF_OFFSET);
    for (int t = first_tile; t < tiles; t += step) {
      for (int c0 = kb0; c0 < kb1; c0 += a.chunk, ++it) {
        const int c1 = min(kb1, c0 + a.chunk);
        const int as = it % S::ACCS;
        const uint32_t aph = static_cast<uint32_t>(it / S::ACCS) & 1u;
        mbar_wait(&acc_empty[as], aph ^ 1u, abort_flag, status, 3);
        tc_fence_after_sync();
        const uint32_t d = tmem + static_cast<uint32_t>(as * BQ);
        // One scale word (four k-blocks) a turn, unrolled: the issuing warp is a single thread's chain of instructions, and for
        // narrow tiles that chain, not the products, was the time of a k-block.
        for (int kb4 = c0; kb4 < c1; kb4 += 4) {
          mbar_wait(&sf_full[f], fph, abort_flag, status, 7);
          const uint32_t sfp = tmem + S::SF_COL + static_cast<uint32_t>(f * S::SF_COLS);
          const uint32_t sfq = sfp + 4;
          const uint64_t sd = desc_advance(sd0, static_cast<uint32_t>(f * S::SF_BYTES));
          const int left = c1 - kb4;                 // k-blocks of this word
#pragma unroll
          for (int j = 0; j < 4; j += S::KPS) {
            if (j < left) {
              mbar_wait(&full[s], ph, abort_flag, status, 4);
              tc_fence_after_sync();
              const uint64_t pd = desc_advance(pd0, static_cast<uint32_t>(s * S::KPS * S::TILE_BYTES));
              const uint64_t qd = desc_advance(qd0, static_cast<uint32_t>(s * S::KPS * S::TILE_BYTES));
              if (elect_one()) {
                if (j == 0) {
                  tmem_cp_scales<PAIR>(sfp, sd);
#pragma unroll
                  for (int g = 0; g < S::Q_ATOMS; ++g) tmem_cp_scales<PAIR>(sfq + 4 * g, desc_advance(sd, 512 * (1 + g)));
                }
#pragma unroll
                for (int i = 0; i < S::KPS; ++i) {
                  if (i == 0 || j + i < left) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)          // 32 codes = 32 bytes of the swizzled row
                      umma_mxf8<PAIR>(d + (S::DUAL ? (k & 1) * BQ : 0), desc_advance(pd, i * S::TILE_BYTES + k * 32),
                                      desc_advance(qd, i * S::TILE_BYTES + k * 32), make_idesc_mxf8(P_TILE, BQ, j + i), sfp, sfq,
                                      (kb4 > c0 || j + i > 0 || k > (S::DUAL ? 1 : 0)) ? 1u : 0u);
                  }
                }
                sg_commit<PAIR>(&empty[s]);
                if (j + S::KPS >= left || j + S::KPS >= 4) sg_commit<PAIR>(&sf_empty[f]);
              }
              __syncwarp();
              if (++s == S::STAGES) { s = 0; ph ^= 1u; }
            }
          }
          if (++f == S::SF_SLOTS) { f = 0; fph ^= 1u; }
        }
        if (elect_one()) sg_commit<PAIR>(&acc_full[as]);
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------ drain
    const int quad = warp & 3, half = (warp - 4) >> 2;
    constexpr int COLS = BQ / 2 < 16 ? 16 : BQ / 2;       // columns per warp (the narrowest tile is drained by four warps)
    constexpr int GROUP = COLS < 32 ? COLS : 32;
    const bool drains = BQ >= 32 || half == 0;
    const int c_first = BQ >= 32 ? half * COLS : 0;
    int it = 0;
    for (int t = first_tile; t < tiles; t += step) {
      int tp, tq;
      sg_tile(t, a.tiles_p, a.tiles_q, tp, tq);
      float acc[COLS];
      if (!JOIN && a.bias != nullptr) {          // the sum starts from the bias (through shared memory: a lane has all columns)
        float* mine = reinterpret_cast<float*>(smem + S::BIAS_OFFSET) + (warp - 4) * COLS;
        __syncwarp();
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          const int n = tq * BQ + c_first + c + lane;
          mine[c + lane] = n < a.q.rows ? load_typed(a.bias, a.bias_type, n) : 0.f;
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < COLS; c += 4) {
          const float4 v = *reinterpret_cast<const float4*>(mine + c);
          acc[c] = v.x; acc[c + 1] = v.y; acc[c + 2] = v.z; acc[c + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[c] = 0.f;
      }
      for (int c0 = kb0; c0 < kb1; c0 += a.chunk, ++it) {
        const int as = it % S::ACCS;
        const uint32_t aph = static_cast<uint32_t>(it / S::ACCS) & 1u;
        mbar_wait(&acc_full[as], aph, abort_flag, status, 5);
        tc_fence_after_sync();
        const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(as * BQ + c_first);
        if (drains) {
#pragma unroll
          for (int c = 0; c < COLS; c += GROUP) {
            uint32_t raw[GROUP];
            if constexpr (GROUP == 32) tmem_ld_32x32(taddr + c, raw);
            else tmem_ld_32x16(taddr + c, raw);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
              asm volatile("" : "+r"(raw[j]));          // no use above the wait
              acc[c + j] += __uint_as_float(raw[j]);
            }
            if constexpr (S::DUAL) {
              if constexpr (GROUP == 32) tmem_ld_32x32(taddr + BQ + c, raw);
              else tmem_ld_32x16(taddr + BQ + c, raw);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < GROUP; ++j) {
                asm volatile("" : "+r"(raw[j]));
                acc[c + j] += __uint_as_float(raw[j]);
              }
            }
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (PAIR && rank == 1) mbar_arrive_leader(&acc_empty[as]);
          else mbar_arrive(&acc_empty[as]);
        }
      }
      if constexpr (JOIN) {
        // Column c of the tile is finished by CTA c / slots, in the row's place c % slots of what every CTA sends it (SWAP, where
        // few columns may be in use: by CTA c % split, at place c / split).
        if (SWAP && split == 1) {                        // rows of the output are columns here: lanes along n
          const int n = tp * SG_BP + quad * 32 + lane;
          if (drains && n < a.p.rows) {
            const float b = a.bias != nullptr ? load_typed(a.bias, a.bias_type, n) : 0.f;
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
              const int m = tq * BQ + c_first + c;
              if (m < a.q.rows) store_typed(a.out, a.out_type, static_cast<long long>(m) * a.ldo + n, acc[c] + b);
            }
          }
          continue;
        }
        cluster_wait();                                  // all CTAs of the cluster have started
        const uint32_t slots = BQ / split;
        if constexpr (SWAP) {
          const uint32_t out = smem_u32(smem) + S::OUT_OFFSET + (quad * 32 + lane) * 4;
          if (drains) {
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
              const uint32_t col = c_first + c;
              st_cluster_f32(cluster_addr(out + (rank * slots + col / split) * (SG_PITCH * 4), col % split), acc[c]);
            }
          }
        } else {
          const uint32_t out = smem_u32(smem) + S::OUT_OFFSET + (rank * SG_BP + quad * 32 + lane) * (slots + 4) * 4;
          const uint32_t shift = split == 4 ? 5 : 6;     // slots = 32 or 64
#pragma unroll
          for (int c = 0; c < COLS; c += 4) {
            const uint32_t col = c_first + c;
            st_cluster_f32x4(cluster_addr(out + (col & (slots - 1)) * 4, col >> shift), acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
          }
        }
      } else {
        const int row0 = tp * P_TILE + p_off + quad * 32;  // rows of the output (p runs along m here)
        const int col0 = tq * BQ + c_first;
        uint8_t* stage = smem + S::OUT_OFFSET + (warp - 4) * 2048;
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
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int r = i * 8 + (lane >> 2);
                  const float4 o = *reinterpret_cast<const float4*>(stage + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
                  if (r < rows) *reinterpret_cast<float4*>(dst + static_cast<long long>(r) * a.ldo + piece * 4) = o;
                }
              } else {
                const int e = lane & 15;
                const bool in = col + e < width;
#pragma unroll 4
                for (int r = lane >> 4; r < 32; r += 2) {
                  const float v = *reinterpret_cast<const float*>(stage + r * 64 + (((e >> 2) ^ ((r >> 1) & 3)) << 4) + (e & 3) * 4);
                  if (in && r < rows) dst[static_cast<long long>(r) * a.ldo + e] = v;
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

  if (JOIN && split > 1) {
    // CTA `rank` finishes its columns of the tile (SWAP: rows of the output), adding the parts in rank order.
    __syncwarp();
    if (warp < 4) cluster_wait();            // the draining warps waited before they pushed
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    const float* parts = reinterpret_cast<const float*>(smem + S::OUT_OFFSET);
    const int slots = BQ / static_cast<int>(split);
    int tp, tq;
    sg_tile(first_tile, a.tiles_p, a.tiles_q, tp, tq);
    if constexpr (SWAP) {          // p runs along n, q along m: lanes along n
      const int n = tp * SG_BP + (threadIdx.x & 127);
      if (n < a.p.rows) {
        const float b = a.bias != nullptr ? load_typed(a.bias, a.bias_type, n) : 0.f;
        for (int k = threadIdx.x >> 7; k < slots; k += SG_THREADS / 128) {
          const int m = tq * BQ + k * static_cast<int>(split) + static_cast<int>(rank);
          if (m >= a.q.rows) break;
          float v = 0.f;
          for (int r = 0; r < static_cast<int>(split); ++r) v += parts[(r * slots + k) * SG_PITCH + (threadIdx.x & 127)];
          store_typed(a.out, a.out_type, static_cast<long long>(m) * a.ldo + n, v + b);
        }
      }
    } else {                        // a lane takes four columns of a row
      const int per_row = slots / 4;
      for (int i = threadIdx.x / per_row; i < SG_BP; i += SG_THREADS / per_row) {
        const int m = tp * SG_BP + i;
        if (m >= a.p.rows) break;
        const int k = threadIdx.x % per_row * 4, n = tq * BQ + static_cast<int>(rank) * slots + k;
        float e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (r >= static_cast<int>(split)) break;
          const float4 x = *reinterpret_cast<const float4*>(parts + (r * SG_BP + i) * (slots + 4) + k);
          e[0] += x.x; e[1] += x.y; e[2] += x.z; e[3] += x.w;
        }
        if (a.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < a.q.rows) e[j] += load_typed(a.bias, a.bias_type, n + j);
        }
        const long long at = static_cast<long long>(m) * a.ldo + n;
        if (a.vec_out && n + 4 <= a.q.rows) {
          if (a.out_type == JB_T_F32) *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(e[0], e[1], e[2], e[3]);
          else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = make_uint2(pack_half16(e[0], e[1], a.out_type), pack_half16(e[2], e[3], a.out_type));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < a.q.rows) store_typed(a.out, a.out_type, at + j, e[j]);
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (PAIR) {             // neither CTA leaves while the other's products read its shared memory or arrive on it
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    else tmem_dealloc(tmem, 512);
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

template <int BQ, bool PAIR, bool SWAP, bool JOIN>
static int launch_scaled_gemm(const void* P, long long pitch_p, const void* Q, long long pitch_q, long long K, ScaledGemmArgs a,
                              int split, int sm_count, int* status, cudaStream_t stream) {
  using S = SgSmem<BQ, PAIR, JOIN>;
  constexpr int P_TILE = PAIR ? 2 * SG_BP : SG_BP;
  CUtensorMap tmP, tmQ;
  if (make_tmap_codes(&tmP, P, a.p.rows, K, pitch_p, SG_BP) != 0) return -2;
  if (make_tmap_codes(&tmQ, Q, a.q.rows, K, pitch_q, S::Q_ROWS) != 0) return -2;
  a.tiles_p = (a.p.rows + P_TILE - 1) / P_TILE;
  a.tiles_q = (a.q.rows + BQ - 1) / BQ;
  auto kern = scaled_gemm_kernel<BQ, PAIR, SWAP, JOIN>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL) != cudaSuccess) return -3;
  const long long tiles = static_cast<long long>(a.tiles_p) * a.tiles_q;
  if (tiles * split > 0x7fffffffLL) return -1;
  const int cluster = PAIR ? 2 : split;
  const long long teams = sm_count / (PAIR ? 2 : 1) > 0 ? sm_count / (PAIR ? 2 : 1) : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(JOIN ? tiles * split : (tiles < teams ? tiles : teams) * cluster));
  cfg.blockDim = dim3(SG_THREADS);
  cfg.dynamicSmemBytes = S::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = JOIN || PAIR ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, tmP, tmQ, a, status) == cudaSuccess ? 0 : -4;
}

}  // namespace jb

extern "C" int jb_scaled_gemm(const JbScaledOperand* a, const JbScaledOperand* b, long long K, void* out, long long ldo,
                              int out_type, const void* bias, int bias_type, int sm_count, int* status, void* stream) {
  using namespace jb;
  if (a == nullptr || b == nullptr || a->rows < 1 || b->rows < 1 || K < 1 || K > 0x7fffff00LL || sm_count < 2) return -1;
  if ((a->pitch & 15) || (b->pitch & 15) || (reinterpret_cast<uintptr_t>(a->codes) & 15) || (reinterpret_cast<uintptr_t>(b->codes) & 15)) return -1;
  if (out_type < 0 || out_type > 2 || bias_type < 0 || bias_type > 2) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ScaledGemmArgs g{};
  auto operand = [](const JbScaledOperand* o) {
    const int words = o->scale_k == 1 && (o->scale_row & 3) == 0 && (reinterpret_cast<uintptr_t>(o->scales) & 3) == 0;
    return ScaledOperand{static_cast<const uint8_t*>(o->scales), o->scale_row, o->scale_k, o->square ? 7 : 0, o->rows, words};
  };
  const ScaledOperand oa = operand(a), ob = operand(b);
  g.out = out; g.ldo = ldo; g.out_type = out_type; g.bias = bias; g.bias_type = bias_type;
  g.kblocks = static_cast<int>((K + 127) / 128);
  // The tensor cores add into TMEM by truncation: every addition (32 terms) loses up to 2^-23 of the sum so far, all towards
  // zero, so the error of a sum grows with its length and is relative to the sum of its terms' magnitudes S, not to the result
  // (8192 terms of random sign: 5e-7 of the result).  fp32 results are drained and added up in registers every 2048 terms
  // (2^-17 S at most), 16-bit ones every 16384 (2^-14 S at most: an eighth of a half step of fp16 where all terms have one
  // sign; where they cancel, more of the result, like any fp32 sum, which may lose K 2^-24 S).
  g.chunk = out_type == JB_T_F32 ? 16 : 128;
  const int size = out_type == JB_T_F32 ? 4 : 2;
  g.vec_out = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (ldo * size) % 16 == 0;
  const int M = a->rows, N = b->rows;
#define JB_SG(BQ, PAIR) return launch_scaled_gemm<BQ, PAIR, false, false>(a->codes, a->pitch, b->codes, b->pitch, K, g, 1, sm_count, status, st)
  // Up to 64 rows the weight lies along the lanes.  8192 x 4096: 10.6 us for one row, against 13.9 us in tiles of 128 rows, and
  // 13.2 us both ways for 64 rows.
  if (M <= 64) {
    g.p = ob; g.q = oa;
    // How many CTAs share a tile: the one of 1, 2, 4, 8 with the least of (k-blocks of a CTA, 0.17 us each, or reading the
    // weight at 6.5 TB/s) and the meeting of the parts (2 us).  Measured, one token: 1024 x 4096 takes 9.9 us whole, 8.5, 7.1
    // and 6.2 us in two, four and eight parts, 8192 x 4096 10.7 us whole and 12.2 us in two.
    const int tiles = (N + 127) / 128;
    const float memory = static_cast<float>(N) * static_cast<float>(K) / 6.5e6f;
    int split = 1;
    float least = 0.f;
    for (int k = 1; k <= 8 && tiles * k <= (k == 1 ? tiles : sm_count) && g.kblocks >= 4 * k; k *= 2) {
      const float own = 0.17f * g.kblocks / k;
      const float cost = (own > memory ? own : memory) + (k > 1 ? 2.f : 0.f);
      if (k == 1 || cost < least) {
        least = cost;
        split = k;
      }
    }
    if (M <= 16) return launch_scaled_gemm<16, false, true, true>(b->codes, b->pitch, a->codes, a->pitch, K, g, split, sm_count, status, st);
    if (M <= 32) return launch_scaled_gemm<32, false, true, true>(b->codes, b->pitch, a->codes, a->pitch, K, g, split, sm_count, status, st);
    return launch_scaled_gemm<64, false, true, true>(b->codes, b->pitch, a->codes, a->pitch, K, g, split, sm_count, status, st);
  }
  g.p = oa; g.q = ob;
  // Tile width.  One k-block costs a CTA about 720 cycles at 128 x 256 and 600 at 128 x 128 (shared memory, which the loads
  // fill and the products read, is the bound of both), so the wide tile wins unless it leaves a wave of SMs idle:
  // 4096 x 1024 x 4096 takes 18.5 us wide and 24.9 us narrow, 512 x 4096 x 4096 17.8 us and 15.0 us.
  const long long tiles256 = static_cast<long long>((M + 127) / 128) * ((N + 255) / 256);
  const long long tiles128 = static_cast<long long>((M + 127) / 128) * ((N + 127) / 128);
  const long long waves256 = (tiles256 + sm_count - 1) / sm_count, waves128 = (tiles128 + sm_count - 1) / sm_count;
  if (waves256 * 720 <= waves128 * 600) {
    // Pairs load a third less, which pays where rows and waves are long, and costs short products up to two microseconds of
    // hand-overs.  Pair and single CTA: 8192^3 395 and 426 us (after seconds of it, under the power limit at 1.1 to 1.2 GHz, 470
    // and 498), 8192 x 11008 x 4096 278 and 295, 4096 x 4096 x 8192 105 and 110, x 2048 33.2 and 33.6, x 1024 25.3 and 22.9;
    // a single wave: 4096 x 1024 x 4096 20.0 and 18.5, 2048 x 4096 x 4096 31.5 and 32.1.
    if (g.kblocks >= 16 && tiles256 >= 2LL * sm_count) { JB_SG(256, true); }
    JB_SG(256, false);
  }
  // A tile shared by a cluster costs 4 us (two CTAs) to 5 us (four) for the meeting of its parts, a k-block 0.26 us:
  // 256 x 1024 x 8192 takes 21.3 us whole, 17.4 in two parts and 14.0 us in four (K = 4096: 12.8, 12.8 and 11.3),
  // 1024 x 1024 x 8192 22.5 us whole and 19.3 us in two (K = 4096: 13.6 and 14.1).
  const int split = tiles128 * 4 <= sm_count && g.kblocks >= 32 ? 4 : tiles128 * 2 <= sm_count && g.kblocks >= 40 ? 2 : 1;
  if (split > 1) return launch_scaled_gemm<128, false, false, true>(a->codes, a->pitch, b->codes, b->pitch, K, g, split, sm_count, status, st);
  JB_SG(128, false);
#undef JB_SG
}
