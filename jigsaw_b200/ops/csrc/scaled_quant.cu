// Block quantisation to 8 bits (e4m3 codes, power-of-two scales) and the root-mean-square norm that feeds it.
//
// A block of 128 values with the largest finite magnitude A has the scale s = the smallest power of two with
// A <= 448 s (448 is the largest e4m3 value), at least 2^-116, and 1 for a block of zeros; the codes are v / s rounded to
// nearest even.  s is a power of two, so v / s is exact and the codes are decided by one rounding: no other program
// that follows the definition gets other codes.  Below 2^-116 nothing is lost that fp32 holds as a normal number (the
// smallest code is 2^-9 s).  Infinities and NaN become NaN codes and do not count towards A.
//
// All kernels here are bound by memory: each input byte is read once and each output byte written once.
#include <type_traits>

#include "ptx.cuh"
#include "scaled_abi.h"

namespace jb {

// ---------------------------------------------------------------- values and codes
// Magnitudes are compared as integers: the bits of a float without its sign order like the numbers, infinities and NaN above
// all of them.  A block whose largest magnitude is below INF_BITS holds finite values only, and its codes need no checks;
// otherwise the largest finite magnitude is found again, one value at a time.
constexpr uint32_t INF_BITS = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t finite_magnitude(float v) {
  const uint32_t b = magnitude(v);
  return b < INF_BITS ? b : 0u;
}
// e8m0 byte of the scale of a block whose largest finite magnitude has these bits: 1.75 * 2^(e - 127) >= A with the
// least e (adding 0x1fffff carries into the exponent exactly when the fraction is above .75), then 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_byte(uint32_t magnitude) {
  if (magnitude == 0u) return 127u;
  const int e = static_cast<int>((magnitude + 0x1fffffu) >> 23) - 8;
  return static_cast<uint32_t>(e < 11 ? 11 : e);
}
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
template <bool CHECKED>
__device__ __forceinline__ float code_input(float v, float inv) {
  const float q = v * inv;
  if constexpr (CHECKED) return magnitude(v) < INF_BITS ? q : __uint_as_float(0x7fffffffu);
  return q;
}
// Four codes in one word, a in the lowest byte; magnitudes above 448 give 448, NaN the NaN code.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  uint32_t w;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}" : "=r"(w) : "f"(a), "f"(b), "f"(c), "f"(d));
  return w;
}
template <bool CHECKED>
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float inv) {
  return make_uint2(codes4(code_input<CHECKED>(v[0], inv), code_input<CHECKED>(v[1], inv), code_input<CHECKED>(v[2], inv), code_input<CHECKED>(v[3], inv)),
                    codes4(code_input<CHECKED>(v[4], inv), code_input<CHECKED>(v[5], inv), code_input<CHECKED>(v[6], inv), code_input<CHECKED>(v[7], inv)));
}
// Four rows of four bytes -> four columns.
__device__ __forceinline__ void turn4(uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, uint32_t& c0, uint32_t& c1, uint32_t& c2, uint32_t& c3) {
  const uint32_t a = __byte_perm(r0, r1, 0x5140), b = __byte_perm(r2, r3, 0x5140);
  const uint32_t c = __byte_perm(r0, r1, 0x7362), d = __byte_perm(r2, r3, 0x7362);
  c0 = __byte_perm(a, b, 0x5410);
  c1 = __byte_perm(a, b, 0x7632);
  c2 = __byte_perm(c, d, 0x5410);
  c3 = __byte_perm(c, d, 0x7632);
}
// max(m, |a|, |b|), NaN if one of them is.
__device__ __forceinline__ float max_abs3(float m, float a, float b) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
  return r;
}

// Scale byte and codes of a block of 128 values held by 16 neighbouring lanes, eight each.
__device__ __forceinline__ uint32_t block_of_16_lanes(const float (&v)[8], uint2& codes) {
  uint32_t m = magnitude(max_abs3(max_abs3(max_abs3(max_abs3(0.f, v[0], v[1]), v[2], v[3]), v[4], v[5]), v[6], v[7]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (__any_sync(0xffffffffu, m >= INF_BITS)) {
    m = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, finite_magnitude(v[e]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t byte = scale_byte(m);
    codes = codes8<true>(v, inverse_scale(byte));
    return byte;
  }
  const uint32_t byte = scale_byte(m);
  codes = codes8<false>(v, inverse_scale(byte));
  return byte;
}

// Sum and product that keep results below 2^-126 (the library is compiled with fast math, which makes them zero).
__device__ __forceinline__ float add_full(float a, float b) {
  float r;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float mul_full(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half(v); }

// N consecutive elements from p, of which the first `live` exist; VEC: p is aligned for wide loads and live is 0 or N.
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_vec(const T* p, int live, float (&v)[N]) {
  if constexpr (VEC) {
    if (live > 0) {
      constexpr int BYTES = N * static_cast<int>(sizeof(T));
      T e[N];
      if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
      } else {
        static_assert(BYTES == 8, "vector width");
        *reinterpret_cast<uint2*>(e) = __ldg(reinterpret_cast<const uint2*>(p));
      }
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = to_f32<T>(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < live ? to_f32<T>(p[i]) : 0.f;
  }
}
template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_vec(T* p, int live, const float (&v)[N]) {
  if constexpr (VEC) {
    if (live > 0) {
      T e[N];
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = from_f32<T>(v[i]);
#pragma unroll
      for (int i = 0; i < N * static_cast<int>(sizeof(T)) / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < live) p[i] = from_f32<T>(v[i]);
  }
}

__device__ __forceinline__ float gain_at(const void* gain, int type, int c) {
  if (gain == nullptr) return 1.f;
  if (type == 1) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(gain) + c));
  if (type == 2) return __half2float(__ldg(static_cast<const __half*>(gain) + c));
  return __ldg(static_cast<const float*>(gain) + c);
}

// ---------------------------------------------------------------- rows in blocks of 1 x 128
struct QuantArgs {
  const void* x;
  long long ldx;             // elements between rows
  int rows, cols;
  uint8_t* codes;            // [rows, pitch], or null
  long long pitch;
  uint8_t* scales;           // byte of (row, block of columns) at row * scale_row + block * scale_k
  long long scale_row, scale_k;
  uint8_t* codes_t;          // transposed codes [cols, pitch_t], or null
  long long pitch_t;
  uint8_t* scales_t;         // byte of (column, block of rows) at column * scale_t_row + block * scale_t_k
  long long scale_t_row, scale_t_k;
  const float* rstd;         // per row, or null: values are x * rstd * gain
  const void* gain;          // per column
  int gain_type;
  float* colsum;             // [row tiles, cols] partial sums of the values over 128 rows, or null
  int square;                // one scale per 128 x 128
};

// A warp takes 32 rows of one block column, two rows at a time (16 lanes x 8 values); the scale bytes of the CTA's eight
// block columns meet in shared memory and leave eight to a row.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quant_rows_kernel(const QuantArgs a) {
  __shared__ __align__(8) uint8_t bytes[32][8];
  grid_dependency_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, sub = lane & 15, warp = threadIdx.x >> 5;
  const int kb0 = blockIdx.y * 8;
  const int col = (kb0 + warp) * 128 + sub * 8;
  const int live = min(8, max(0, a.cols - col));
  const long long row0 = static_cast<long long>(blockIdx.x) * 32;
  const T* x = static_cast<const T*>(a.x);
  if ((kb0 + warp) * 128 < a.cols) {
#pragma unroll
    for (int i0 = 0; i0 < 16; i0 += 4) {
      if (row0 + 2 * i0 >= a.rows) break;
      float v[4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long row = row0 + 2 * (i0 + i) + (lane >> 4);
        load_vec<T, 8, VEC>(x + row * a.ldx + col, row < a.rows ? live : 0, v[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 2 * (i0 + i) + (lane >> 4);
        uint2 q;
        const uint32_t byte = block_of_16_lanes(v[i], q);
        if (row0 + r < a.rows && col < a.pitch) *reinterpret_cast<uint2*>(a.codes + (row0 + r) * a.pitch + col) = q;
        if (sub == 0) bytes[r][warp] = static_cast<uint8_t>(byte);
      }
    }
  }
  __syncthreads();
  // scale_k = 1: a row's bytes of this CTA are neighbours
  const int n = min(8, (a.cols + 127) / 128 - kb0);
  {
    const int r = threadIdx.x >> 3, k = threadIdx.x & 7;
    if (row0 + r < a.rows && k < n) a.scales[(row0 + r) * a.scale_row + (kb0 + k) * a.scale_k] = bytes[r][k];
  }
}

// ---------------------------------------------------------------- tiles of 128 x 128
// 16 bytes from global to shared memory behind the thread's back; `bytes` < 16 leaves zeros in the rest.
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

struct TileShared {
  union {                                // the magnitudes and sums are read before the codes turn
    uint8_t turned[128 * 128];
    struct {
      uint32_t col_mag[16][128];
      float col_sum[16][128];
    };
  };
  float col_inv[128];
  uint32_t row_mag[16];
};
constexpr int QT_SHARED = (sizeof(TileShared) + 127) / 128 * 128;
// How a tile is read: element by element, with wide loads, or by copies into shared memory one tile ahead.
enum : int { QT_PLAIN = 0, QT_WIDE = 1, QT_AHEAD = 2 };
template <typename T, int MODE>
constexpr int quant_tile_smem() { return QT_SHARED + (MODE == QT_AHEAD ? 2 * 128 * 128 * static_cast<int>(sizeof(T)) : 0); }

// Tiles of 128 x 128, 32 values a thread (warp w: rows 8 w .. 8 w + 7, lane l: columns 4 l .. 4 l + 3).  Scales by row come
// from warp reductions, by column through shared memory, or from the whole tile; the transposed codes turn in shared
// memory, eight bytes of a column at a time.  A CTA takes tiles in steps of the grid; of 16-bit values it has the next tile
// copied into shared memory while it works on the present one (8192 x 11008 bf16, both layouts: that step took 134 us, half
// of it waiting for loads, to 82; 72 us now).  Two fp32 tiles ahead would leave room for one CTA an SM, which was slower than
// loads (11001 x 4100: 48 us against 42 at that time, 40 now).  16-bit rows that are not on 16-byte boundaries are read
// element by element: 8192 x 4100 in squares takes 48 us, 8192 x 4096 18.
template <typename T, int MODE, bool NORM>
__global__ void __launch_bounds__(512, 2) quant_tile_kernel(const QuantArgs a, int tiles_r, int tiles) {
  extern __shared__ __align__(128) uint8_t smem[];
  TileShared& sh = *reinterpret_cast<TileShared*>(smem);
  grid_dependency_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int E16 = 16 / static_cast<int>(sizeof(T));          // elements of a 16-byte copy
  constexpr int TILE_BYTES = 128 * 128 * static_cast<int>(sizeof(T));
  // Thread q of the copy takes 16 bytes at column (q % PER_ROW) E16 of every (512 / PER_ROW)-th row.
  constexpr int PER_ROW = 128 / E16, ROW_STEP = 512 / PER_ROW;
  const int copy_r = threadIdx.x / PER_ROW, copy_c = threadIdx.x % PER_ROW * E16;
  const long long copy_step = a.ldx * ROW_STEP;
  auto prefetch = [&](int tr, int tc, int stage) {
    const int r = tr * 128 + copy_r, c = tc * 128 + copy_c;
    const T* src = static_cast<const T*>(a.x) + r * a.ldx + c;
    const uint32_t dst = smem_u32(smem) + QT_SHARED + stage * TILE_BYTES + threadIdx.x * 16;
    const int rows = c < a.cols ? a.rows - r : 0;                // cols is a multiple of E16
#pragma unroll
    for (int k = 0; k < 128 / ROW_STEP; ++k) {
      const bool in = k * ROW_STEP < rows;
      copy16_async(dst + k * 512 * 16, in ? src : static_cast<const T*>(a.x), in ? 16 : 0);
      src += copy_step;
    }
    copies_commit();
  };
  // tiles run down the rows first; the grid's step in both directions, so that no tile costs a division
  int tile_r = blockIdx.x % tiles_r, tile_c = blockIdx.x / tiles_r;
  const int step_r = gridDim.x % tiles_r, step_c = gridDim.x / tiles_r;
  auto advance = [&](int& r, int& c) {
    r += step_r;
    c += step_c;
    if (r >= tiles_r) {
      r -= tiles_r;
      ++c;
    }
  };
  int stage = 0;
  if constexpr (MODE == QT_AHEAD) prefetch(tile_r, tile_c, 0);
  for (int t = blockIdx.x; t < tiles; t += gridDim.x, stage ^= 1, advance(tile_r, tile_c)) {
    const long long row0 = static_cast<long long>(tile_r) * 128 + warp * 8;
    const int col = tile_c * 128 + lane * 4;
    const int live = min(4, max(0, a.cols - col));
    const int live_rows = static_cast<int>(max(0LL, min(8LL, a.rows - row0)));
    float v[8][4];
    if constexpr (MODE == QT_AHEAD) {
      if (t + gridDim.x < tiles) {
        int next_r = tile_r, next_c = tile_c;
        advance(next_r, next_c);
        prefetch(next_r, next_c, stage ^ 1);
        copies_wait<1>();
      } else {
        copies_wait<0>();
      }
      __syncthreads();               // this tile is there, and the last one's turned codes have been read
      const T* in = reinterpret_cast<const T*>(smem + QT_SHARED + stage * TILE_BYTES) + (warp * 8) * 128 + lane * 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __align__(16) T e[4];
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(in + i * 128);
        else *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(in + i * 128);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = to_f32<T>(e[j]);
      }
    } else {
      __syncthreads();
      const T* x = static_cast<const T*>(a.x) + row0 * a.ldx + col;
#pragma unroll
      for (int i = 0; i < 8; ++i) load_vec<T, 4, MODE == QT_WIDE>(x + i * a.ldx, i < live_rows ? live : 0, v[i]);
    }
    if constexpr (NORM) {
      float g[4] = {1.f, 1.f, 1.f, 1.f};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live) g[j] = gain_at(a.gain, a.gain_type, col + j);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float r = i < live_rows ? __ldg(a.rstd + row0 + i) : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = mul_full(mul_full(v[i][j], r), g[j]);
      }
    }
    uint32_t cm[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i += 2) m = max_abs3(m, v[i][j], v[i + 1][j]);
      cm[j] = magnitude(m);
    }
    if (a.colsum != nullptr) {
      float s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[j] += v[i][j];
      }
      *reinterpret_cast<float4*>(&sh.col_sum[warp][lane * 4]) = make_float4(s[0], s[1], s[2], s[3]);
    }
    const uint32_t top = max(max(cm[0], cm[1]), max(cm[2], cm[3]));
    auto share = [&](uint32_t most) {
      if (a.square) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) sh.row_mag[warp] = m;
      } else if (a.codes_t != nullptr) {
        *reinterpret_cast<uint4*>(&sh.col_mag[warp][lane * 4]) = make_uint4(cm[0], cm[1], cm[2], cm[3]);
      }
    };
    share(top);
    // The rest of the tile, once for finite values and once for tiles with infinities or NaN: those leave as NaN codes, and
    // the magnitudes are found again among the finite ones.
    auto finish = [&](auto checked_c) {
      constexpr bool CHECKED = decltype(checked_c)::value;
      if constexpr (CHECKED) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          cm[j] = 0u;
#pragma unroll
          for (int i = 0; i < 8; ++i) cm[j] = max(cm[j], finite_magnitude(v[i][j]));
        }
        share(max(max(cm[0], cm[1]), max(cm[2], cm[3])));
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[i][j] = code_input<true>(v[i][j], 1.f);      // NaN for every value that is not finite
        __syncthreads();
      }
      if (a.colsum != nullptr && threadIdx.x >= 128 && threadIdx.x < 256 && tile_c * 128 + threadIdx.x - 128 < a.cols) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 16; ++w) s += sh.col_sum[w][threadIdx.x - 128];
        a.colsum[static_cast<long long>(tile_r) * a.cols + tile_c * 128 + threadIdx.x - 128] = s;
      }
      uint8_t* out = a.codes + row0 * a.pitch + col;
      const int out_rows = a.codes != nullptr && col < a.pitch ? live_rows : 0;
      uint2 turned[4];                 // columns 4 l .. 4 l + 3 of this warp's eight rows
      if (a.square) {
        uint32_t m = 0u;
#pragma unroll
        for (int w = 0; w < 16; ++w) m = max(m, sh.row_mag[w]);
        const uint32_t byte = scale_byte(m);
        if (threadIdx.x == 0) a.scales[tile_r * a.scale_row + tile_c * a.scale_k] = static_cast<uint8_t>(byte);
        const float inv = inverse_scale(byte);
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = codes4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
          if (i < out_rows) *reinterpret_cast<uint32_t*>(out) = w[i];
          out += a.pitch;
        }
        if (a.codes_t == nullptr) return;
        // one scale for both layouts: the codes of a column are bytes of the rows' words
        turn4(w[0], w[1], w[2], w[3], turned[0].x, turned[1].x, turned[2].x, turned[3].x);
        turn4(w[4], w[5], w[6], w[7], turned[0].y, turned[1].y, turned[2].y, turned[3].y);
        if (a.colsum != nullptr) __syncthreads();        // the sums have been read
      } else {
        if (a.codes_t != nullptr && threadIdx.x < 128) {
          uint32_t m = 0u;
#pragma unroll
          for (int w = 0; w < 16; ++w) m = max(m, sh.col_mag[w][threadIdx.x]);
          const uint32_t byte = scale_byte(m);
          sh.col_inv[threadIdx.x] = inverse_scale(byte);
          const int c = tile_c * 128 + threadIdx.x;
          if (c < a.cols) a.scales_t[c * a.scale_t_row + tile_r * a.scale_t_k] = static_cast<uint8_t>(byte);
        }
        if (a.codes != nullptr) {
          // lane i holds the scale of row i: one computation for eight rows
          uint32_t mine = 0u;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t m;
            if constexpr (CHECKED)
              m = max(max(finite_magnitude(v[i][0]), finite_magnitude(v[i][1])), max(finite_magnitude(v[i][2]), finite_magnitude(v[i][3])));
            else
              m = magnitude(max_abs3(max_abs3(0.f, v[i][0], v[i][1]), v[i][2], v[i][3]));
            m = __reduce_max_sync(0xffffffffu, m);
            if (lane == i) mine = m;
          }
          const uint32_t byte = scale_byte(mine);
          if (lane < live_rows) a.scales[(row0 + lane) * a.scale_row + tile_c * a.scale_k] = static_cast<uint8_t>(byte);
          const float row_inv = inverse_scale(byte);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float inv = __shfl_sync(0xffffffffu, row_inv, i);
            const uint32_t w = codes4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
            if (i < out_rows) *reinterpret_cast<uint32_t*>(out) = w;
            out += a.pitch;
          }
        }
        if (a.codes_t == nullptr) return;
        __syncthreads();
        const float4 f = *reinterpret_cast<const float4*>(&sh.col_inv[lane * 4]);
        const float inv[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float c[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i] = v[i][j];
          turned[j] = codes8<false>(c, inv[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        // piece `warp` of column 4 lane + j, at a place that differs between the sixteen lanes of a store's half warp
        *reinterpret_cast<uint2*>(sh.turned + (lane * 4 + j) * 128 + ((warp ^ (lane & 15)) << 3)) = turned[j];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = warp * 8 + i * 4 + (lane >> 3);
        const int piece = lane & 7, turn = (c >> 2) & 15;
        uint4 q = *reinterpret_cast<const uint4*>(sh.turned + c * 128 + ((((2 * piece) ^ turn) & ~1) << 3));
        if (turn & 1) q = make_uint4(q.z, q.w, q.x, q.y);
        const long long at = static_cast<long long>(tile_r) * 128 + piece * 16;
        if (tile_c * 128 + c < a.cols && at < a.pitch_t)
          *reinterpret_cast<uint4*>(a.codes_t + (static_cast<long long>(tile_c) * 128 + c) * a.pitch_t + at) = q;
      }
    };
    if (__syncthreads_or(top >= INF_BITS)) finish(std::true_type{});
    else finish(std::false_type{});
  }
}

// out[c] = sum over the rows of part [P, C], 32 columns a CTA; the order of the additions is fixed.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* part, int P, int C, void* out, int out_type) {
  __shared__ float sums[32][33];
  grid_dependency_wait();
  const int c = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (c < C)
    for (int p = threadIdx.y; p < P; p += 32) t += part[static_cast<long long>(p) * C + c];
  sums[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0 && c < C) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += sums[i][threadIdx.x];
    if (out_type == 1) static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16(t);
    else if (out_type == 2) static_cast<__half*>(out)[c] = __float2half(t);
    else static_cast<float*>(out)[c] = t;
  }
}

// ---------------------------------------------------------------- root-mean-square norm
struct RmsArgs {
  const void* x;
  const void* residual;      // or null
  long long ldx, ldr;        // elements between rows
  int rows, cols;
  float eps;
  const void* gain;          // or null
  int gain_type;
  void* sum;                 // x + residual in the type of x, contiguous; null without a residual
  float* rstd;               // per row, or null
  void* y;                   // contiguous, or null
  int y_type;
  uint8_t* codes;            // 8-bit output, or null
  long long pitch;
  uint8_t* scales;
  long long scale_row, scale_k;
};

// Eight elements of a row: VEC, consecutive ones at column c (all or none of them exist); otherwise one every `step`
// columns from c on, so that the lanes of a warp read neighbouring elements whatever the alignment (or, step = 1,
// consecutive ones one by one).
template <typename T, bool VEC>
__device__ __forceinline__ void load_raw(const T* row, int c, int step, int cols, T (&v)[8]) {
  if constexpr (VEC) {
    if (c < cols) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(row + c) + i);
      return;
    }
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4*>(v)[i] = make_uint4(0u, 0u, 0u, 0u);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e * step < cols ? row[c + e * step] : from_f32<T>(0.f);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int c, int step, int cols, float (&v)[8]) {
  __align__(16) T raw[8];
  load_raw<T, VEC>(row, c, step, cols, raw);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = to_f32<T>(raw[e]);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, int c, int step, int cols, const float (&v)[8]) {
  if constexpr (VEC) {
    if (c < cols) {
      __align__(16) T raw[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) raw[e] = from_f32<T>(v[e]);
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4*>(row + c)[i] = reinterpret_cast<const uint4*>(raw)[i];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e * step < cols) row[c + e * step] = from_f32<T>(v[e]);
  }
}
template <bool VEC>
__device__ __forceinline__ void gain8(const void* gain, int type, int c, int step, int cols, float (&g)[8]) {
  if (gain == nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = 1.f;
  } else if (type == 1) {
    load8<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16*>(gain), c, step, cols, g);
  } else if (type == 2) {
    load8<__half, VEC>(static_cast<const __half*>(gain), c, step, cols, g);
  } else {
    load8<float, VEC>(static_cast<const float*>(gain), c, step, cols, g);
  }
}

// Sum over the threads of a row: one warp, or the whole CTA (`shared` holds a value per warp).
template <bool WARP>
__device__ __forceinline__ double row_sum(double v, double* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (!WARP) {
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < warps; ++w) v += shared[w];
  }
  return v;
}

// A row belongs to one warp (WARP: eight rows a CTA) or to one CTA; a thread keeps NV vectors of eight values between the
// sum of squares and the output, so that every byte is read once.  The squares of a thread are added in fp32, the
// threads in fp64: the sum is good to the last bit of fp32 or nearly so, whatever the length of the row.
template <typename T, int NV, bool VEC, bool WARP, bool CODES, int MOST>
__global__ void __launch_bounds__(MOST) rms_fwd_kernel(const RmsArgs a) {
  __shared__ double shared[32];
  if constexpr (CODES) grid_dependency_launch();
  grid_dependency_wait();
  const int G = WARP ? 32 : blockDim.x;                          // threads of a row
  const int g = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const long long row = WARP ? static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && row >= a.rows) return;
  // consecutive values per thread where blocks of 128 columns have to meet in 16 neighbouring lanes, or loads are wide
  constexpr bool RUN = VEC || CODES;
  const int step = RUN ? 1 : G;
  auto column = [&](int i) { return RUN ? (i * G + g) * 8 : i * 8 * G + g; };
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  float t[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) load8<T, VEC>(x, column(i), step, a.cols, t[i]);
  if (a.residual != nullptr) {
    const T* res = static_cast<const T*>(a.residual) + row * a.ldr;
    __align__(16) T r[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) load_raw<T, VEC>(res, column(i), step, a.cols, r[i]);
    T* sum = static_cast<T*>(a.sum) + row * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      // the norm is of the sum as it is stored: the backward pass, which reads the stored one, differentiates this function
#pragma unroll
      for (int e = 0; e < 8; ++e) t[i][e] = to_f32<T>(from_f32<T>(add_full(t[i][e], to_f32<T>(r[i][e]))));
      store8<T, VEC>(sum, column(i), step, a.cols, t[i]);
    }
  }
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sq = fmaf(t[i][e], t[i][e], sq);
  const double mean = row_sum<WARP>(static_cast<double>(sq), shared) / a.cols;
  const float rstd = static_cast<float>(1.0 / sqrt(mean + static_cast<double>(a.eps)));
  if (a.rstd != nullptr && g == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = column(i);
    float w[8];
    gain8<VEC>(a.gain, a.gain_type, c, step, a.cols, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[i][e] = mul_full(mul_full(t[i][e], rstd), w[e]);
    if constexpr (CODES) {
      uint2 q;
      const uint32_t byte = block_of_16_lanes(t[i], q);          // 16 lanes = 128 columns
      if (c < a.pitch) *reinterpret_cast<uint2*>(a.codes + row * a.pitch + c) = q;
      if ((g & 15) == 0 && c < a.cols) a.scales[row * a.scale_row + (c >> 7) * a.scale_k] = static_cast<uint8_t>(byte);
    } else {
      if (a.y_type == 0) store8<float, VEC>(static_cast<float*>(a.y) + row * a.cols, c, step, a.cols, t[i]);
      else store8<T, VEC>(static_cast<T*>(a.y) + row * a.cols, c, step, a.cols, t[i]);
    }
  }
}

// dx = r (w g - t r^2 mean(w g t)) + gsum and the gain's gradient sum_rows g t r.  A CTA takes rows in steps of the grid
// and keeps the gain's partial sums of its columns in registers until the end; column_sum_kernel adds the CTAs' parts in
// a fixed order.  The next row is read before the present one is worked on.  For rows that the ring below does not take: off
// 16-byte boundaries, where elements are loaded one by one (16384 x 4095 bf16: 308 us, 82 of traffic; 16384 x 4100, one larger
// CTA an SM: 508), and rows too long for it (4096 x 20000 bf16, 64 registers a thread: 786 us, 100 of traffic; 8192 x 16384
// fp32: 864, 327 of traffic).
struct RmsBwdArgs {
  const void* t;             // the normalised sum, contiguous rows ldt apart
  long long ldt;
  const void* g;             // gradient of y: type of t, or fp32
  const void* gsum;          // gradient of the sum, type of t, contiguous, or null
  const float* rstd;
  const void* gain;
  int gain_type;
  int rows, cols;
  void* dx;                  // contiguous
  float* part;               // [gridDim.x * rows of a CTA, cols], or null
};

// MOST: threads of the largest CTA (registers: 128 a thread up to 512 threads, 64 beyond).
template <typename T, typename TG, int NV, bool VEC, bool WARP, int MOST>
__global__ void __launch_bounds__(MOST, MOST <= 256 ? 2 : 1) rms_bwd_kernel(const RmsBwdArgs a) {
  __shared__ double shared[2][32];
  grid_dependency_wait();
  const int G = WARP ? 32 : blockDim.x;
  const int g = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const long long first = WARP ? static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
  const long long stride = static_cast<long long>(gridDim.x) * (WARP ? 8 : 1);
  const int step = VEC ? 1 : G;
  auto column = [&](int i) { return VEC ? (i * G + g) * 8 : i * 8 * G + g; };
  const T* ts = static_cast<const T*>(a.t);
  const TG* gs = static_cast<const TG*>(a.g);
  const T* ss = static_cast<const T*>(a.gsum);
  T* dxs = static_cast<T*>(a.dx);
  float dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
  __align__(16) T nt[NV][8], ns[NV][8];
  __align__(16) TG ng[NV][8];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      load_raw<T, VEC>(ts + row * a.ldt, column(i), step, a.cols, nt[i]);
      load_raw<TG, VEC>(gs + row * a.cols, column(i), step, a.cols, ng[i]);
      if (ss != nullptr) load_raw<T, VEC>(ss + row * a.cols, column(i), step, a.cols, ns[i]);
    }
  };
  if (first < a.rows) fetch(first);
  int turn = 0;
  for (long long row = first; row < a.rows; row += stride, turn ^= 1) {     // the same trip count for all threads of a row
    float t[NV][8], y[NV][8], s[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t[i][e] = to_f32<T>(nt[i][e]);
        y[i][e] = to_f32<TG>(ng[i][e]);
        s[i][e] = ss != nullptr ? to_f32<T>(ns[i][e]) : 0.f;
      }
    const float r = __ldg(a.rstd + row);
    if (row + stride < a.rows) fetch(row + stride);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      gain8<VEC>(a.gain, a.gain_type, column(i), step, a.cols, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dw[i][e] = fmaf(y[i][e], t[i][e] * r, dw[i][e]);
        y[i][e] *= w[e];
        dot = fmaf(y[i][e], t[i][e], dot);
      }
    }
    const float inner = static_cast<float>(row_sum<WARP>(static_cast<double>(dot), shared[turn]) / a.cols);
    const float k3 = r * r * inner;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[i][e] = fmaf(r, y[i][e] - t[i][e] * k3, s[i][e]);
      store8<T, VEC>(dxs + row * a.cols, column(i), step, a.cols, s[i]);
    }
  }
  if (a.part != nullptr) {
    float* out = a.part + first * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) store8<float, VEC>(out, column(i), step, a.cols, dw[i]);
  }
}

// The same pass with the rows brought into shared memory by bulk copies several batches ahead, for rows on 16-byte
// boundaries.  A row belongs to `team` warps (8 NV values a thread), a batch is the `batch` rows that fit a CTA's eight or
// sixteen; two CTAs of eight an SM cover one another's reductions (16384 x 4096 bf16: 100 us; 119 with direct wide loads, when
// those took such rows).  The row is read from shared memory twice (for the sums, then for the gradient), so a thread keeps
// only the gain and its partial sums, which the teams of a CTA add up at the end: one row of `part` a CTA.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

template <typename T, typename TG, int NV, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS) rms_bwd_ring_kernel(const RmsBwdArgs a, int team, int batch, int stages, int* status) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[8];
  __shared__ float sums[2][WARPS];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mine = warp / team;                              // this thread's team; rows of the batch behind the last one idle
  const int G = team * 32, g = (warp % team) * 32 + lane;
  const int C = a.cols;
  const int t_bytes = C * static_cast<int>(sizeof(T)), g_bytes = C * static_cast<int>(sizeof(TG));
  const int row_bytes = t_bytes + g_bytes + (a.gsum != nullptr ? t_bytes : 0);
  const long long batches = (static_cast<long long>(a.rows) + batch - 1) / batch;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    abort_word = 0;
    fence_mbar_init();
  }
  grid_dependency_wait();
  __syncthreads();
  // one warp brings a batch: a lane per row and array
  auto fetch = [&](long long b, int s) {
    const int rows = static_cast<int>(min(static_cast<long long>(batch), a.rows - b * batch));
    if (lane == 0) mbar_expect_tx(&full[s], static_cast<uint32_t>(rows * row_bytes));
    __syncwarp();
    for (int k = lane; k < rows * 3; k += 32) {
      const long long row = b * batch + k / 3;
      const uint32_t dst = smem_u32(ring) + static_cast<uint32_t>((s * batch + k / 3) * row_bytes);
      if (k % 3 == 0) bulk_load(dst, static_cast<const T*>(a.t) + row * a.ldt, t_bytes, &full[s]);
      else if (k % 3 == 1) bulk_load(dst + t_bytes, static_cast<const TG*>(a.g) + row * C, g_bytes, &full[s]);
      else if (a.gsum != nullptr) bulk_load(dst + t_bytes + g_bytes, static_cast<const T*>(a.gsum) + row * C, t_bytes, &full[s]);
    }
  };
  if (warp == 0)
    for (int s = 0; s < stages; ++s) {
      const long long b = blockIdx.x + static_cast<long long>(s) * gridDim.x;
      if (b < batches) fetch(b, s);
    }
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    gain8<true>(a.gain, a.gain_type, (i * G + g) * 8, 1, C, w[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
  }
  auto rstd_of = [&](long long b) {
    const long long row = b * batch + mine;
    return mine < batch && row < a.rows ? __ldg(a.rstd + row) : 0.f;
  };
  auto vec = [&](auto* p, float (&v)[8]) {
    using E = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    __align__(16) E raw[8];
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(E)) / 2; ++k) reinterpret_cast<uint4*>(raw)[k] = reinterpret_cast<const uint4*>(p)[k];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f32<E>(raw[e]);
  };
  float r = rstd_of(blockIdx.x);
  int s = 0, turn = 0;
  uint32_t ph = 0;
  for (long long b = blockIdx.x; b < batches; b += gridDim.x, turn ^= 1) {
    const float r_next = rstd_of(b + gridDim.x);
    mbar_wait(&full[s], ph, abort_flag, status, 8);
    const long long row = b * batch + mine;
    if (mine < batch && row < a.rows) {
      const uint8_t* at = ring + (s * batch + mine) * row_bytes;
      const T* ts = reinterpret_cast<const T*>(at);
      const TG* gs = reinterpret_cast<const TG*>(at + t_bytes);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + g) * 8;
        if (c < C) {
          float t[8], y[8];
          vec(ts + c, t);
          vec(gs + c, y);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            dw[i][e] = fmaf(y[e], t[e] * r, dw[i][e]);
            dot = fmaf(y[e] * w[i][e], t[e], dot);
          }
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (team > 1) {
        if (lane == 0) sums[turn][warp] = dot;
        named_barrier(1 + mine, G);
        dot = 0.f;
        for (int k = 0; k < team; ++k) dot += sums[turn][mine * team + k];
      }
      const float k3 = r * r * (dot / static_cast<float>(C));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + g) * 8;
        if (c < C) {
          float t[8], y[8], d[8];
          vec(ts + c, t);
          vec(gs + c, y);
          if (a.gsum != nullptr) {
            vec(reinterpret_cast<const T*>(at + t_bytes + g_bytes) + c, d);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = 0.f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = fmaf(r, y[e] * w[i][e] - t[e] * k3, d[e]);
          store8<T, true>(static_cast<T*>(a.dx) + row * C, c, 1, C, d);
        }
      }
    }
    r = r_next;
    __syncthreads();                          // the batch has been read
    const long long later = b + static_cast<long long>(stages) * gridDim.x;
    if (warp == 0 && later < batches) fetch(later, s);
    if (++s == stages) { s = 0; ph ^= 1u; }
  }
  if (*abort_flag) {                          // a wait gave up: let the copies already issued arrive before the CTA ends
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  if (a.part != nullptr) {
    __syncthreads();
    float* sum = reinterpret_cast<float*>(ring);           // [batch][C]
    if (mine < batch) {
#pragma unroll
      for (int i = 0; i < NV; ++i) store8<float, true>(sum + static_cast<long long>(mine) * C, (i * G + g) * 8, 1, C, dw[i]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += WARPS * 32) {
      float v = 0.f;
      for (int k = 0; k < batch; ++k) v += sum[k * C + c];
      a.part[static_cast<long long>(blockIdx.x) * C + c] = v;
    }
  }
}

// ---------------------------------------------------------------- dispatch
// Launch that may begin while earlier work of the stream still runs: every kernel here calls grid_dependency_wait() before
// it touches memory, so only its launch and set-up overlap (about 2 us a launch in a chain of short kernels).
// The quantising kernels let their successor, the product, start as soon as all their CTAs have: its set-up then runs under
// them (norm and product of 7 tokens 14.2 -> 13.4 us, in a graph 13.2; a training step of 4096 x 4096 x 1024 104.7 -> 103.1).
// The norm's backward pass does not (its successor's CTAs would share its SMs: 182 -> 185 us at 16384 x 4096), nor does the
// product (the next product's CTAs do not fit beside its own).
template <typename Kernel, typename Args, typename... More>
static cudaError_t launch_chained(Kernel kernel, dim3 grid, dim3 block, cudaStream_t stream, int smem, const Args& first, More... more) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, first, more...);
}

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Threads of a CTA that takes one row, `held` values each.
static inline int rms_threads(int cols, int held) { return ((cols + held - 1) / held + 31) / 32 * 32; }

// Rows of up to 1024 values: a warp each.  Longer ones: a CTA each, 32 values a thread, or 8 where there are fewer rows
// than SMs and the time is that of one row's chain of loads and sums (4096 bf16, one row: 4.5 us with 32 a thread, 2.5 with 8).
template <typename T, bool VEC, bool CODES>
static int launch_rms_fwd(const RmsArgs& a, int sm_count, cudaStream_t st) {
  const int warps = (a.rows + 7) / 8;
  if (a.rows < sm_count && a.cols > 256 && a.cols <= 8192)
    launch_chained(rms_fwd_kernel<T, 1, VEC, false, CODES, 1024>, dim3(a.rows), dim3(rms_threads(a.cols, 8)), st, 0, a);
  else if (a.cols <= 512) launch_chained(rms_fwd_kernel<T, 2, VEC, true, CODES, 256>, dim3(warps), dim3(256), st, 0, a);
  else if (a.cols <= 1024) launch_chained(rms_fwd_kernel<T, 4, VEC, true, CODES, 256>, dim3(warps), dim3(256), st, 0, a);
  else if (a.cols <= 16384) launch_chained(rms_fwd_kernel<T, 4, VEC, false, CODES, 512>, dim3(a.rows), dim3(rms_threads(a.cols, 32)), st, 0, a);
  else launch_chained(rms_fwd_kernel<T, 4, VEC, false, CODES, 1024>, dim3(a.rows), dim3(rms_threads(a.cols, 32)), st, 0, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

// How the backward pass cuts its work.  Ring: two CTAs of eight warps an SM where two batches of a row fit each (16-bit rows
// up to 8192), one of sixteen otherwise; NV is the one of 2, 3, 4 that leaves the fewest threads idle.  fp32 rows beyond 8192
// and rows beyond 16384 do not fit.  Otherwise (and for rows that are not on 16-byte boundaries) direct loads: a thread holds
// row, gradient, partial sums and the next row, 16 values of each up to 8192 columns and 32 beyond; rows beyond 16384 spill.
struct RmsBwdPlan {
  int nv, warps, team, batch, stages, ring_bytes, ctas;    // nv = 0: direct loads
};
static inline RmsBwdPlan rms_bwd_ring(int rows, int cols, int bytes_per_value, int sm_count) {
  RmsBwdPlan best{};
  for (int warps = 8; warps <= 16 && best.nv == 0; warps += 8) {
    const int most = sm_count * (16 / warps);
    int used = 0;
    for (int nv = 2; nv <= 4; ++nv) {
      const int team = (cols + 256 * nv - 1) / (256 * nv);
      if (team > warps) continue;
      // few rows: smaller batches, so that every CTA has one
      int batch = warps / team;
      const int fair = (rows + most - 1) / most;
      if (batch > fair) batch = fair;
      const int share = static_cast<int>(1000LL * cols * (warps / team) / (warps * 256 * nv));
      const int stage = batch * cols * bytes_per_value;
      int stages = (warps == 8 ? 104 : 208) * 1024 / stage;
      if (stages > 6) stages = 6;
      if (stages < 2 || share <= used) continue;
      const int need = batch * cols * 4;         // the partial sums of the teams, at the end
      const long long batches = (static_cast<long long>(rows) + batch - 1) / batch;
      used = share;
      best = RmsBwdPlan{nv, warps, team, batch, stages, stages * stage > need ? stages * stage : need,
                        static_cast<int>(batches < most ? batches : most)};
    }
  }
  return best;
}
static inline bool rms_bwd_by_warp(int cols) { return cols <= 512; }
static inline int rms_bwd_threads(int cols) {
  return rms_bwd_by_warp(cols) ? 256 : rms_threads(cols, cols <= 8192 ? 16 : 32);
}
static inline int rms_bwd_ctas(int rows, int cols, int sm_count) {
  const int threads = rms_bwd_threads(cols);
  const int resident = threads > 256 ? 1 : 512 / threads < 8 ? 512 / threads : 8;
  const long long want = rms_bwd_by_warp(cols) ? (static_cast<long long>(rows) + 7) / 8 : rows;
  const long long most = static_cast<long long>(sm_count) * resident;
  return static_cast<int>(want < most ? want : most);
}
// Wide loads are possible: the ring's condition too.
static inline bool rms_bwd_wide(const JbRmsBwd* q) {
  const long long size = q->type == 0 ? 4 : 2;
  return q->cols % 8 == 0 && (q->ldt * size) % 16 == 0 && aligned16(q->t) && aligned16(q->g) && aligned16(q->gsum) &&
         aligned16(q->gain) && aligned16(q->dx);
}
static inline int rms_bwd_bytes(const JbRmsBwd* q) {
  const int size = q->type == 0 ? 4 : 2;
  return size + (q->g_f32 ? 4 : size) + (q->gsum != nullptr ? size : 0);
}

template <typename T, typename TG>
static int launch_rms_bwd(const RmsBwdArgs& a, bool wide, const RmsBwdPlan& plan, int sm_count, int* status, cudaStream_t st) {
  if (plan.nv != 0) {
    auto go = [&](auto kernel) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, plan.ring_bytes) != cudaSuccess) return -3;
      return launch_chained(kernel, dim3(plan.ctas), dim3(plan.warps * 32), st, plan.ring_bytes, a, plan.team, plan.batch, plan.stages, status) == cudaSuccess ? 0 : -4;
    };
    if (plan.warps == 8) {
      if (plan.nv == 2) return go(rms_bwd_ring_kernel<T, TG, 2, 8>);
      if (plan.nv == 3) return go(rms_bwd_ring_kernel<T, TG, 3, 8>);
      return go(rms_bwd_ring_kernel<T, TG, 4, 8>);
    }
    if (plan.nv == 2) return go(rms_bwd_ring_kernel<T, TG, 2, 16>);
    if (plan.nv == 3) return go(rms_bwd_ring_kernel<T, TG, 3, 16>);
    return go(rms_bwd_ring_kernel<T, TG, 4, 16>);
  }
  const int grid = rms_bwd_ctas(a.rows, a.cols, sm_count), threads = rms_bwd_threads(a.cols);
#define JB_BWD(NV, VEC, WARP, MOST) launch_chained(rms_bwd_kernel<T, TG, NV, VEC, WARP, MOST>, dim3(grid), dim3(threads), st, 0, a)
  if (a.cols > 16384) {
    if (wide) JB_BWD(4, true, false, 1024);
    else JB_BWD(4, false, false, 1024);
  } else if (a.cols > 8192) {
    if (wide) JB_BWD(4, true, false, 512);
    else JB_BWD(4, false, false, 512);
  } else if (rms_bwd_by_warp(a.cols)) {          // the ring takes every wide case up to here
    JB_BWD(2, false, true, 256);
  } else if (threads <= 256) {
    JB_BWD(2, false, false, 256);
  } else {
    JB_BWD(2, false, false, 512);
  }
#undef JB_BWD
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

template <typename T>
static int launch_quant(const QuantArgs& a, bool tiles, int sm_count, cudaStream_t st) {
  const long long size = static_cast<long long>(sizeof(T));
  const int kblocks = (a.cols + 127) / 128, rblocks = (a.rows + 127) / 128;
  if (tiles) {
    const bool vec = (a.cols * size) % 16 == 0 && (a.ldx * size) % 16 == 0 && aligned16(a.x);
    const long long n = static_cast<long long>(rblocks) * kblocks;
    if (n > 0x7fffffffLL - 1024) return -1;
    constexpr int FAST = sizeof(T) == 2 ? QT_AHEAD : QT_WIDE;
    auto go = [&](auto kernel, int smem) {
      // two CTAs an SM where the next tile is copied ahead; without that a CTA a tile
      const long long most = vec && FAST == QT_AHEAD ? 2LL * sm_count : n;
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -3;
      return launch_chained(kernel, dim3(static_cast<unsigned>(n < most ? n : most)), dim3(512), st, smem, a, rblocks, static_cast<int>(n)) == cudaSuccess ? 0 : -4;
    };
#define JB_TILE(NORM)                                                                                   \
  return vec ? go(quant_tile_kernel<T, FAST, NORM>, quant_tile_smem<T, FAST>())                         \
             : go(quant_tile_kernel<T, QT_PLAIN, NORM>, quant_tile_smem<T, QT_PLAIN>());
    if (a.rstd != nullptr) { JB_TILE(true) }
    JB_TILE(false)
#undef JB_TILE
  } else {
    const bool vec = a.cols % 8 == 0 && (a.ldx * size) % 16 == 0 && aligned16(a.x);
    const dim3 grid((a.rows + 31) / 32, (kblocks + 7) / 8);
    if (vec) launch_chained(quant_rows_kernel<T, true>, dim3(grid), dim3(256), st, 0, a);
    else launch_chained(quant_rows_kernel<T, false>, dim3(grid), dim3(256), st, 0, a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace jb

// Codes and scales of x (times rstd and gain) by rows, by columns (transposed), both, or in squares of 128 x 128 (both
// layouts share the scales).  Pitches are multiples of 16; bytes between the last value and the pitch are written as 0
// within the last 8 (transposed: 16) bytes only.
extern "C" int jb_quantize(const JbQuant* q, int sm_count, void* stream) {
  using namespace jb;
  if (q == nullptr || q->rows < 1 || q->cols < 1 || (q->codes == nullptr && q->codes_t == nullptr)) return -1;
  if (q->codes != nullptr && ((q->pitch & 15) || !aligned16(q->codes) || q->pitch < q->cols)) return -1;
  if (q->codes_t != nullptr && ((q->pitch_t & 15) || !aligned16(q->codes_t) || q->pitch_t < q->rows)) return -1;
  QuantArgs a{};
  a.x = q->x; a.ldx = q->ldx; a.rows = q->rows; a.cols = q->cols;
  a.codes = static_cast<uint8_t*>(q->codes); a.pitch = q->pitch;
  a.scales = static_cast<uint8_t*>(q->scales); a.scale_row = q->scale_row; a.scale_k = q->scale_k;
  a.codes_t = static_cast<uint8_t*>(q->codes_t); a.pitch_t = q->pitch_t;
  a.scales_t = static_cast<uint8_t*>(q->scales_t); a.scale_t_row = q->scale_t_row; a.scale_t_k = q->scale_t_k;
  a.rstd = static_cast<const float*>(q->rstd); a.gain = q->gain; a.gain_type = q->gain_type;
  a.colsum = static_cast<float*>(q->colsum); a.square = q->square;
  // rows alone: a warp per 32 rows of one block column is quick for few rows, tiles for many (8192 x 11008 bf16: 94 us
  // against 51); nor do 8 x 65535 block columns fit the grid of the first
  const bool tiles = q->square || q->codes_t != nullptr || q->rstd != nullptr || q->colsum != nullptr || q->rows >= 128 ||
                     q->cols > 65535 * 1024;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (q->type == 0) return launch_quant<float>(a, tiles, sm_count, st);
  if (q->type == 1) return launch_quant<__nv_bfloat16>(a, tiles, sm_count, st);
  if (q->type == 2) return launch_quant<__half>(a, tiles, sm_count, st);
  return -1;
}

extern "C" int jb_column_sum(const float* part, int P, int C, void* out, int out_type, void* stream) {
  if (P < 1 || C < 1) return -1;
  return jb::launch_chained(jb::column_sum_kernel, dim3((C + 31) / 32), dim3(32, 32), static_cast<cudaStream_t>(stream), 0, part, P, C, out, out_type) == cudaSuccess ? 0 : -4;
}

// Longest row that the kernels keep in registers.
extern "C" int jb_rms_max_cols() { return 32768; }

extern "C" int jb_rms_norm_fwd(const JbRms* q, int sm_count, void* stream) {
  using namespace jb;
  if (q == nullptr || q->rows < 1 || q->cols < 1 || q->cols > jb_rms_max_cols() || q->type < 0 || q->type > 2) return -1;
  if ((q->residual == nullptr) != (q->sum == nullptr) || (q->codes == nullptr) == (q->y == nullptr)) return -1;
  if (q->codes != nullptr && ((q->pitch & 15) || !aligned16(q->codes) || q->pitch < q->cols)) return -1;
  if (q->y != nullptr && q->y_type != 0 && q->y_type != q->type) return -1;
  RmsArgs a{};
  a.x = q->x; a.residual = q->residual; a.ldx = q->ldx; a.ldr = q->ldr; a.rows = q->rows; a.cols = q->cols; a.eps = q->eps;
  a.gain = q->gain; a.gain_type = q->gain_type; a.sum = q->sum; a.rstd = static_cast<float*>(q->rstd);
  a.y = q->y; a.y_type = q->y_type; a.codes = static_cast<uint8_t*>(q->codes); a.pitch = q->pitch;
  a.scales = static_cast<uint8_t*>(q->scales); a.scale_row = q->scale_row; a.scale_k = q->scale_k;
  const long long size = q->type == 0 ? 4 : 2;
  const bool vec = q->cols % 8 == 0 && (q->ldx * size) % 16 == 0 && (q->ldr * size) % 16 == 0 && aligned16(q->x) &&
                   aligned16(q->residual) && aligned16(q->sum) && aligned16(q->y) && aligned16(q->gain);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define JB_RMS(T)                                                                                              \
  if (q->codes != nullptr) return vec ? launch_rms_fwd<T, true, true>(a, sm_count, st) : launch_rms_fwd<T, false, true>(a, sm_count, st); \
  return vec ? launch_rms_fwd<T, true, false>(a, sm_count, st) : launch_rms_fwd<T, false, false>(a, sm_count, st);
  if (q->type == 0) { JB_RMS(float) }
  if (q->type == 1) { JB_RMS(__nv_bfloat16) }
  JB_RMS(__half)
#undef JB_RMS
}

// Rows of the gain's partial sums that jb_rms_norm_bwd writes for these arguments.
extern "C" int jb_rms_bwd_parts(const JbRmsBwd* q, int sm_count) {
  using namespace jb;
  const RmsBwdPlan plan = rms_bwd_wide(q) ? rms_bwd_ring(q->rows, q->cols, rms_bwd_bytes(q), sm_count) : RmsBwdPlan{};
  if (plan.nv != 0) return plan.ctas;
  return rms_bwd_ctas(q->rows, q->cols, sm_count) * (rms_bwd_by_warp(q->cols) ? 8 : 1);
}

extern "C" int jb_rms_norm_bwd(const JbRmsBwd* q, int sm_count, int* status, void* stream) {
  using namespace jb;
  if (q == nullptr || q->rows < 1 || q->cols < 1 || q->cols > jb_rms_max_cols() || q->type < 0 || q->type > 2) return -1;
  RmsBwdArgs a{};
  a.t = q->t; a.ldt = q->ldt; a.g = q->g; a.gsum = q->gsum;
  a.rstd = static_cast<const float*>(q->rstd); a.gain = q->gain; a.gain_type = q->gain_type; a.rows = q->rows; a.cols = q->cols;
  a.dx = q->dx; a.part = static_cast<float*>(q->part);
  const bool wide = rms_bwd_wide(q);
  const RmsBwdPlan plan = wide ? rms_bwd_ring(q->rows, q->cols, rms_bwd_bytes(q), sm_count) : RmsBwdPlan{};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define JB_RMS(T, TG) return launch_rms_bwd<T, TG>(a, wide && aligned16(q->part), plan, sm_count, status, st);
  if (q->type == 0) { JB_RMS(float, float) }
  if (q->type == 1) {
    if (q->g_f32) { JB_RMS(__nv_bfloat16, float) }
    JB_RMS(__nv_bfloat16, __nv_bfloat16)
  }
  if (q->g_f32) { JB_RMS(__half, float) }
  JB_RMS(__half, __half)
#undef JB_RMS
}
