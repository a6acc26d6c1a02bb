// Block quantisation to 8 bits (e4m3 codes, power-of-two scales) and the root-mean-square norm that feeds it.
//
// A block of 128 values with the largest finite magnitude A has the scale s = the smallest power of two with
// A <= 448 s (448 is the largest e4m3 value), at least 2^-116, and 1 for a block of zeros; the codes are v / s rounded to
// nearest even.  s is a power of two, so v / s is exact and the codes are decided by one rounding: no other program
// that follows the definition gets other codes.  Below 2^-116 nothing is lost that fp32 holds as a normal number (the
// smallest code is 2^-9 s).  Infinities and NaN become NaN codes and do not count towards A.
//
// All kernels here are bound by memory: each input byte is read once and each output byte written once.
#include <cuda_fp8.h>

#include "ptx.cuh"
#include "scaled_abi.h"

namespace jb {

// ---------------------------------------------------------------- values and codes
// The magnitude of a value as an integer that orders like it; 0 for infinities and NaN.
__device__ __forceinline__ uint32_t finite_magnitude(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// e8m0 byte of the scale of a block whose largest finite magnitude has these bits: 1.75 * 2^(e - 127) >= A with the
// least e (adding 0x1fffff carries into the exponent exactly when the fraction is above .75), then 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_byte(uint32_t magnitude) {
  if (magnitude == 0u) return 127u;
  const int e = static_cast<int>((magnitude + 0x1fffffu) >> 23) - 8;
  return static_cast<uint32_t>(e < 11 ? 11 : e);
}
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float code_input(float v, float inv) {
  const float q = v * inv;
  return (__float_as_uint(v) & 0x7fffffffu) < 0x7f800000u ? q : __uint_as_float(0x7fffffffu);
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
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

// A warp takes 32 rows of one block column, two rows at a time (16 lanes x 8 values); its 32 scale bytes leave together.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quant_rows_kernel(const QuantArgs a) {
  const int lane = threadIdx.x & 31, sub = lane & 15;
  const int kb = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int col = kb * 128 + sub * 8;
  if (kb * 128 >= a.cols) return;
  const int live = min(8, max(0, a.cols - col));
  const T* x = static_cast<const T*>(a.x);
  for (long long row0 = static_cast<long long>(blockIdx.x) * 32; row0 < a.rows; row0 += static_cast<long long>(gridDim.x) * 32) {
    uint32_t mine = 127u;
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
        const long long row = row0 + 2 * (i0 + i) + (lane >> 4);
        uint32_t m = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, finite_magnitude(v[i][e]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const uint32_t byte = scale_byte(m);
        const float inv = inverse_scale(byte);
        if (row < a.rows && col < a.pitch) {
          uint2 q;
          q.x = codes4(code_input(v[i][0], inv), code_input(v[i][1], inv), code_input(v[i][2], inv), code_input(v[i][3], inv));
          q.y = codes4(code_input(v[i][4], inv), code_input(v[i][5], inv), code_input(v[i][6], inv), code_input(v[i][7], inv));
          *reinterpret_cast<uint2*>(a.codes + row * a.pitch + col) = q;
        }
        // row 2 (i0 + i) + h was reduced by lanes 16 h .. 16 h + 15
        const uint32_t other = __shfl_xor_sync(0xffffffffu, byte, 16);
        if ((lane >> 1) == i0 + i) mine = (lane & 1) == (lane >> 4) ? byte : other;
      }
    }
    const long long row = row0 + lane;
    if (row < a.rows) a.scales[row * a.scale_row + kb * a.scale_k] = static_cast<uint8_t>(mine);
  }
}

// ---------------------------------------------------------------- tiles of 128 x 128
// One CTA, one tile: values in registers (warp w: rows 16 w .. 16 w + 15, lane l: columns 4 l .. 4 l + 3), scales by
// row (shuffles), by column (shared memory) or of the whole tile; the transposed codes turn in shared memory, 16 bytes
// of one column at a time.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quant_tile_kernel(const QuantArgs a) {
  __shared__ __align__(16) uint8_t turned[128 * 128];
  __shared__ uint32_t col_mag[8][128];
  __shared__ float col_sum[8][128];
  __shared__ uint32_t row_mag[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tile_r = blockIdx.x, tile_c = blockIdx.y;
  const long long row0 = static_cast<long long>(tile_r) * 128 + warp * 16;
  const int col = tile_c * 128 + lane * 4;
  const int live = min(4, max(0, a.cols - col));
  const T* x = static_cast<const T*>(a.x);
  float v[16][4];
#pragma unroll
  for (int i = 0; i < 16; ++i) load_vec<T, 4, VEC>(x + (row0 + i) * a.ldx + col, row0 + i < a.rows ? live : 0, v[i]);
  if (a.rstd != nullptr) {
    float g[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      g[j] = (a.gain == nullptr || j >= live) ? 1.f
             : a.gain_type == 1 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.gain)[col + j])
             : a.gain_type == 2 ? __half2float(static_cast<const __half*>(a.gain)[col + j])
                                : static_cast<const float*>(a.gain)[col + j];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float r = row0 + i < a.rows ? __ldg(a.rstd + row0 + i) : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = v[i][j] * r * g[j];
    }
  }
  uint32_t cm[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) cm[j] = max(cm[j], finite_magnitude(v[i][j]));
  if (a.colsum != nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) t += v[i][j];
      col_sum[warp][lane * 4 + j] = t;
    }
  }
  if (a.square) {
    uint32_t m = max(max(cm[0], cm[1]), max(cm[2], cm[3]));
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) row_mag[warp] = m;
  } else if (a.codes_t != nullptr) {
    *reinterpret_cast<uint4*>(&col_mag[warp][lane * 4]) = make_uint4(cm[0], cm[1], cm[2], cm[3]);
  }
  __syncthreads();
  if (a.colsum != nullptr && threadIdx.x < 128 && tile_c * 128 + threadIdx.x < a.cols) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += col_sum[w][threadIdx.x];
    a.colsum[static_cast<long long>(tile_r) * a.cols + tile_c * 128 + threadIdx.x] = t;
  }

  uint32_t square_byte = 0u;
  if (a.square) {
    uint32_t m = 0u;
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, row_mag[w]);
    square_byte = scale_byte(m);
    if (threadIdx.x == 0) a.scales[tile_r * a.scale_row + tile_c * a.scale_k] = static_cast<uint8_t>(square_byte);
  }
  if (a.codes != nullptr) {
    uint32_t mine = 0u;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      uint32_t byte = square_byte;
      if (!a.square) {
        uint32_t m = max(max(finite_magnitude(v[i][0]), finite_magnitude(v[i][1])), max(finite_magnitude(v[i][2]), finite_magnitude(v[i][3])));
        byte = scale_byte(__reduce_max_sync(0xffffffffu, m));
        if (lane == i) mine = byte;
      }
      const float inv = inverse_scale(byte);
      if (row0 + i < a.rows && col < a.pitch)
        *reinterpret_cast<uint32_t*>(a.codes + (row0 + i) * a.pitch + col) =
            codes4(code_input(v[i][0], inv), code_input(v[i][1], inv), code_input(v[i][2], inv), code_input(v[i][3], inv));
    }
    if (!a.square && lane < 16 && row0 + lane < a.rows)
      a.scales[(row0 + lane) * a.scale_row + tile_c * a.scale_k] = static_cast<uint8_t>(mine);
  }
  if (a.codes_t != nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t byte = square_byte;
      if (!a.square) {
        uint32_t m = 0u;
#pragma unroll
        for (int w = 0; w < 8; ++w) m = max(m, col_mag[w][lane * 4 + j]);
        byte = scale_byte(m);
        if (warp == j && col + j < a.cols)      // each warp writes one of the four
          a.scales_t[(col + j) * a.scale_t_row + tile_r * a.scale_t_k] = static_cast<uint8_t>(byte);
      }
      const float inv = inverse_scale(byte);
      uint4 q;
      q.x = codes4(code_input(v[0][j], inv), code_input(v[1][j], inv), code_input(v[2][j], inv), code_input(v[3][j], inv));
      q.y = codes4(code_input(v[4][j], inv), code_input(v[5][j], inv), code_input(v[6][j], inv), code_input(v[7][j], inv));
      q.z = codes4(code_input(v[8][j], inv), code_input(v[9][j], inv), code_input(v[10][j], inv), code_input(v[11][j], inv));
      q.w = codes4(code_input(v[12][j], inv), code_input(v[13][j], inv), code_input(v[14][j], inv), code_input(v[15][j], inv));
      const int c = lane * 4 + j;
      *reinterpret_cast<uint4*>(turned + c * 128 + ((warp ^ (lane & 7)) << 4)) = q;       // lane & 7 = (c >> 2) & 7
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = warp * 16 + i * 4 + (lane >> 3);
      const int piece = lane & 7;
      const long long at = static_cast<long long>(tile_r) * 128 + piece * 16;
      if (tile_c * 128 + c < a.cols && at < a.pitch_t)
        *reinterpret_cast<uint4*>(a.codes_t + (static_cast<long long>(tile_c) * 128 + c) * a.pitch_t + at) =
            *reinterpret_cast<const uint4*>(turned + c * 128 + ((piece ^ ((c >> 2) & 7)) << 4));
    }
  }
}

// out[c] = sum over the rows of part [P, C], 32 columns a CTA; the order of the additions is fixed.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* part, int P, int C, void* out, int out_type) {
  __shared__ float sums[32][33];
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

__device__ __forceinline__ float gain_at(const void* gain, int type, int c) {
  if (gain == nullptr) return 1.f;
  if (type == 1) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(gain) + c));
  if (type == 2) return __half2float(__ldg(static_cast<const __half*>(gain) + c));
  return __ldg(static_cast<const float*>(gain) + c);
}
__device__ __forceinline__ void gain_vec(const void* gain, int type, int c, int live, bool vec, float (&g)[8]) {
  if (gain != nullptr && vec && live == 8) {
    if (type == 1) return load_vec<__nv_bfloat16, 8, true>(static_cast<const __nv_bfloat16*>(gain) + c, 8, g);
    if (type == 2) return load_vec<__half, 8, true>(static_cast<const __half*>(gain) + c, 8, g);
    return load_vec<float, 8, true>(static_cast<const float*>(gain) + c, 8, g);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) g[e] = e < live ? gain_at(gain, type, c + e) : 0.f;
}

// Sum of `v` over the G threads of a row (G a multiple of 32; `slot` separates the rows of a CTA).
template <int G>
__device__ __forceinline__ double row_sum(double v, double* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (G > 32) {
    const int warp = threadIdx.x >> 5;
    constexpr int W = G / 32;
    if ((threadIdx.x & 31) == 0) shared[warp] = v;
    __syncthreads();
    v = 0.0;
    const int first = warp / W * W;
#pragma unroll
    for (int w = 0; w < W; ++w) v += shared[first + w];
  }
  return v;
}

// G threads a row, NV vectors of 8 values each (vector i of thread g starts at 8 (i G + g)); rows up to 8 G NV values
// stay in registers between the sum of squares and the output, so that every byte is read once.  The squares of a
// thread are added in fp32, the threads in fp64: the sum is good to the last bit of fp32 or nearly so, whatever the
// length of the row.
template <typename T, int G, int NV, bool VEC>
__global__ void __launch_bounds__(G < 256 ? 256 : G) rms_fwd_kernel(const RmsArgs a) {
  constexpr int THREADS = G < 256 ? 256 : G;
  constexpr int ROWS = THREADS / G;
  __shared__ double shared[THREADS / 32];
  const int g = threadIdx.x % G;
  const long long row = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / G;
  const bool in = row < a.rows;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* res = a.residual == nullptr ? nullptr : static_cast<const T*>(a.residual) + row * a.ldr;
  float t[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + g) * 8;
    load_vec<T, 8, VEC>(x + c, in ? min(8, max(0, a.cols - c)) : 0, t[i]);
  }
  if (res != nullptr) {
    float r[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + g) * 8;
      load_vec<T, 8, VEC>(res + c, in ? min(8, max(0, a.cols - c)) : 0, r[i]);
    }
    T* sum = static_cast<T*>(a.sum) + row * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + g) * 8;
      // the norm is of the sum as it is stored: the backward pass, which reads the stored one, differentiates this function
#pragma unroll
      for (int e = 0; e < 8; ++e) t[i][e] = to_f32<T>(from_f32<T>(t[i][e] + r[i][e]));
      store_vec<T, 8, VEC>(sum + c, in ? min(8, max(0, a.cols - c)) : 0, t[i]);
    }
  }
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sq = fmaf(t[i][e], t[i][e], sq);
  const double mean = row_sum<G>(static_cast<double>(sq), shared) / a.cols;
  const float rstd = static_cast<float>(1.0 / sqrt(mean + static_cast<double>(a.eps)));
  if (a.rstd != nullptr && g == 0 && in) a.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + g) * 8;
    const int live = in ? min(8, max(0, a.cols - c)) : 0;
    float w[8];
    gain_vec(a.gain, a.gain_type, c, live, VEC, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[i][e] = t[i][e] * rstd * w[e];
    if (a.y != nullptr) {
      const long long at = row * a.cols + c;
      if (a.y_type == 0) store_vec<float, 8, VEC>(static_cast<float*>(a.y) + at, live, t[i]);
      else store_vec<T, 8, VEC>(static_cast<T*>(a.y) + at, live, t[i]);
    }
    if (a.codes != nullptr) {
      uint32_t m = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, finite_magnitude(t[i][e]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));   // 16 lanes = 128 columns
      const uint32_t byte = scale_byte(m);
      const float inv = inverse_scale(byte);
      if (in && c < a.pitch) {
        uint2 q;
        q.x = codes4(code_input(t[i][0], inv), code_input(t[i][1], inv), code_input(t[i][2], inv), code_input(t[i][3], inv));
        q.y = codes4(code_input(t[i][4], inv), code_input(t[i][5], inv), code_input(t[i][6], inv), code_input(t[i][7], inv));
        *reinterpret_cast<uint2*>(a.codes + row * a.pitch + c) = q;
      }
      if (in && (g & 15) == 0 && c < a.cols) a.scales[row * a.scale_row + (c >> 7) * a.scale_k] = static_cast<uint8_t>(byte);
    }
  }
}

// dx = r (w g - t r^2 mean(w g t)) + gsum and the gain's gradient sum_rows g t r.  A CTA keeps the gain's partial sums
// of its rows in registers and writes them once at the end; column_sum_kernel adds the CTAs' rows in a fixed order.
struct RmsBwdArgs {
  const void* t;             // the normalised sum, contiguous rows ldt apart
  long long ldt;
  const void* g;             // gradient of y: type of t, or fp32
  int g_f32;
  const void* gsum;          // gradient of the sum, type of t, contiguous, or null
  const float* rstd;
  const void* gain;
  int gain_type;
  int rows, cols;
  void* dx;                  // contiguous
  float* part;               // [gridDim.x * ROWS, cols], or null
};

template <typename T, int G, int NV, bool VEC>
__global__ void __launch_bounds__(G < 256 ? 256 : G) rms_bwd_kernel(const RmsBwdArgs a) {
  constexpr int THREADS = G < 256 ? 256 : G;
  constexpr int ROWS = THREADS / G;
  __shared__ double shared[2][THREADS / 32];
  const int g = threadIdx.x % G;
  const int lane_row = threadIdx.x / G;
  float dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
  int turn = 0;
  const long long stride = static_cast<long long>(gridDim.x) * ROWS;
  const long long rounds = (a.rows + stride - 1) / stride;       // the same for every thread: row_sum has barriers
  for (long long k = 0; k < rounds; ++k, turn ^= 1) {
    const long long row = k * stride + static_cast<long long>(blockIdx.x) * ROWS + lane_row;
    const bool in = row < a.rows;
    float t[NV][8], y[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + g) * 8;
      const int live = in ? min(8, max(0, a.cols - c)) : 0;
      load_vec<T, 8, VEC>(static_cast<const T*>(a.t) + row * a.ldt + c, live, t[i]);
      if (a.g_f32) load_vec<float, 8, VEC>(static_cast<const float*>(a.g) + row * a.cols + c, live, y[i]);
      else load_vec<T, 8, VEC>(static_cast<const T*>(a.g) + row * a.cols + c, live, y[i]);
    }
    const float r = in ? __ldg(a.rstd + row) : 0.f;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + g) * 8;
      const int live = in ? min(8, max(0, a.cols - c)) : 0;
      float w[8];
      gain_vec(a.gain, a.gain_type, c, live, VEC, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dw[i][e] = fmaf(y[i][e], t[i][e] * r, dw[i][e]);
        y[i][e] *= w[e];
        dot = fmaf(y[i][e], t[i][e], dot);
      }
    }
    const float inner = static_cast<float>(row_sum<G>(static_cast<double>(dot), shared[turn]) / a.cols);
    const float k3 = r * r * inner;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + g) * 8;
      const int live = in ? min(8, max(0, a.cols - c)) : 0;
      float s[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = 0.f;
      if (a.gsum != nullptr) load_vec<T, 8, VEC>(static_cast<const T*>(a.gsum) + row * a.cols + c, live, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = fmaf(r, y[i][e] - t[i][e] * k3, s[e]);
      store_vec<T, 8, VEC>(static_cast<T*>(a.dx) + row * a.cols + c, live, s);
    }
  }
  if (a.part != nullptr) {
    float* out = a.part + (static_cast<long long>(blockIdx.x) * ROWS + lane_row) * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + g) * 8;
      store_vec<float, 8, VEC>(out + c, min(8, max(0, a.cols - c)), dw[i]);
    }
  }
}

// ---------------------------------------------------------------- dispatch
static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Threads per row when each keeps `held` values: a row of up to 1024 * held stays in registers.
static inline int rms_group(int cols, int held) {
  int g = 32;
  while (g < 1024 && g * held < cols) g *= 2;
  return g;
}
// Forward: 32 values a thread (60 registers).  Backward: 16, because it holds three arrays (row, gradient, partial sums
// of the gain); rows beyond 16384 take 32 and spill.
constexpr int RMS_FWD_HELD = 32;
static inline int rms_bwd_held(int cols) { return cols <= 16384 ? 16 : 32; }

template <typename T, bool VEC>
static int launch_rms_fwd(const RmsArgs& a, cudaStream_t st) {
#define JB_RMS_FWD(G)                                                                                          \
  case G: {                                                                                                    \
    constexpr int ROWS = (G < 256 ? 256 : G) / G;                                                              \
    rms_fwd_kernel<T, G, 4, VEC><<<(a.rows + ROWS - 1) / ROWS, G < 256 ? 256 : G, 0, st>>>(a);                 \
    break;                                                                                                     \
  }
  switch (rms_group(a.cols, RMS_FWD_HELD)) { JB_RMS_FWD(32) JB_RMS_FWD(64) JB_RMS_FWD(128) JB_RMS_FWD(256) JB_RMS_FWD(512) JB_RMS_FWD(1024) }
#undef JB_RMS_FWD
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

template <typename T, bool VEC>
static int launch_rms_bwd(const RmsBwdArgs& a, int grid, cudaStream_t st) {
  if (rms_bwd_held(a.cols) == 32) {
    rms_bwd_kernel<T, 1024, 4, VEC><<<grid, 1024, 0, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? 0 : -4;
  }
#define JB_RMS_BWD(G)                                                               \
  case G:                                                                           \
    rms_bwd_kernel<T, G, 2, VEC><<<grid, G < 256 ? 256 : G, 0, st>>>(a);            \
    break;
  switch (rms_group(a.cols, 16)) { JB_RMS_BWD(32) JB_RMS_BWD(64) JB_RMS_BWD(128) JB_RMS_BWD(256) JB_RMS_BWD(512) JB_RMS_BWD(1024) }
#undef JB_RMS_BWD
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

template <typename T>
static int launch_quant(const QuantArgs& a, bool tiles, cudaStream_t st) {
  const long long size = static_cast<long long>(sizeof(T));
  const int kblocks = (a.cols + 127) / 128, rblocks = (a.rows + 127) / 128;
  if (tiles) {
    const bool vec = a.cols % 4 == 0 && (a.ldx * size) % (4 * size) == 0 && (reinterpret_cast<uintptr_t>(a.x) & (4 * size - 1)) == 0;
    if (kblocks > 65535) return -1;
    const dim3 grid(rblocks, kblocks);
    if (vec) quant_tile_kernel<T, true><<<grid, 256, 0, st>>>(a);
    else quant_tile_kernel<T, false><<<grid, 256, 0, st>>>(a);
  } else {
    const bool vec = a.cols % 8 == 0 && (a.ldx * size) % 16 == 0 && aligned16(a.x);
    if ((kblocks + 7) / 8 > 65535) return -1;
    const dim3 grid((a.rows + 31) / 32, (kblocks + 7) / 8);
    if (vec) quant_rows_kernel<T, true><<<grid, 256, 0, st>>>(a);
    else quant_rows_kernel<T, false><<<grid, 256, 0, st>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace jb

// Codes and scales of x (times rstd and gain) by rows, by columns (transposed), both, or in squares of 128 x 128 (both
// layouts share the scales).  Pitches are multiples of 16; bytes between the last value and the pitch are written as 0
// within the last 8 (transposed: 16) bytes only.
extern "C" int jb_quantize(const JbQuant* q, void* stream) {
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
  const bool tiles = q->square || q->codes_t != nullptr || q->rstd != nullptr || q->colsum != nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (q->type == 0) return launch_quant<float>(a, tiles, st);
  if (q->type == 1) return launch_quant<__nv_bfloat16>(a, tiles, st);
  if (q->type == 2) return launch_quant<__half>(a, tiles, st);
  return -1;
}

extern "C" int jb_column_sum(const float* part, int P, int C, void* out, int out_type, void* stream) {
  if (P < 1 || C < 1) return -1;
  jb::column_sum_kernel<<<(C + 31) / 32, dim3(32, 32), 0, static_cast<cudaStream_t>(stream)>>>(part, P, C, out, out_type);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

// Longest row that the kernels keep in registers.
extern "C" int jb_rms_max_cols() { return 32768; }

extern "C" int jb_rms_norm_fwd(const JbRms* q, void* stream) {
  using namespace jb;
  if (q == nullptr || q->rows < 1 || q->cols < 1 || q->cols > jb_rms_max_cols()) return -1;
  if ((q->residual == nullptr) != (q->sum == nullptr)) return -1;
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
  if (q->type == 0) return vec ? launch_rms_fwd<float, true>(a, st) : launch_rms_fwd<float, false>(a, st);
  if (q->type == 1) return vec ? launch_rms_fwd<__nv_bfloat16, true>(a, st) : launch_rms_fwd<__nv_bfloat16, false>(a, st);
  if (q->type == 2) return vec ? launch_rms_fwd<__half, true>(a, st) : launch_rms_fwd<__half, false>(a, st);
  return -1;
}

// CTAs of the backward pass and rows of its partial sums.  Two CTAs an SM fill it; a CTA takes at least four rounds of
// rows, so that the partial sums stay a small part of the traffic.
extern "C" int jb_rms_bwd_grid(int rows, int cols, int sm_count) {
  const int g = jb::rms_group(cols, jb::rms_bwd_held(cols));
  const int per = (g < 256 ? 256 : g) / g;
  const int most = sm_count * (g <= 256 ? 2 : 1);
  const long long want = (static_cast<long long>(rows) + 4 * per - 1) / (4 * per);
  return static_cast<int>(want < 1 ? 1 : (want < most ? want : most));
}
extern "C" int jb_rms_bwd_parts(int rows, int cols, int sm_count) {
  const int g = jb::rms_group(cols, jb::rms_bwd_held(cols));
  return jb_rms_bwd_grid(rows, cols, sm_count) * ((g < 256 ? 256 : g) / g);
}

extern "C" int jb_rms_norm_bwd(const JbRmsBwd* q, int sm_count, void* stream) {
  using namespace jb;
  if (q == nullptr || q->rows < 1 || q->cols < 1 || q->cols > jb_rms_max_cols()) return -1;
  RmsBwdArgs a{};
  a.t = q->t; a.ldt = q->ldt; a.g = q->g; a.g_f32 = q->g_f32 || q->type == 0; a.gsum = q->gsum;
  a.rstd = static_cast<const float*>(q->rstd); a.gain = q->gain; a.gain_type = q->gain_type; a.rows = q->rows; a.cols = q->cols;
  a.dx = q->dx; a.part = static_cast<float*>(q->part);
  const long long size = q->type == 0 ? 4 : 2;
  const bool vec = q->cols % 8 == 0 && (q->ldt * size) % 16 == 0 && aligned16(q->t) && aligned16(q->g) && aligned16(q->gsum) &&
                   aligned16(q->gain) && aligned16(q->dx) && aligned16(q->part);
  const int grid = jb_rms_bwd_grid(q->rows, q->cols, sm_count);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (q->type == 0) return vec ? launch_rms_bwd<float, true>(a, grid, st) : launch_rms_bwd<float, false>(a, grid, st);
  if (q->type == 1) return vec ? launch_rms_bwd<__nv_bfloat16, true>(a, grid, st) : launch_rms_bwd<__nv_bfloat16, false>(a, grid, st);
  if (q->type == 2) return vec ? launch_rms_bwd<__half, true>(a, grid, st) : launch_rms_bwd<__half, false>(a, grid, st);
  return -1;
}
