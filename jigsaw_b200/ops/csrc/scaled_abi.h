// C interface of the 8-bit kernels (scaled_quant.cu, scaled_gemm.cu), shared with the torch binding.  Element types: 0 fp32,
// 1 bf16, 2 fp16.  Every function returns 0, or a negative code if the launch could not be set up.
#pragma once

// Operand of the scaled product: e4m3 codes [rows, K] (K contiguous, rows `pitch` bytes apart, base and pitch multiples of
// 16) and their e8m0 scales, strides in bytes per scale row and per block of 128 along K.
struct JbScaledOperand {
  const void* codes;
  long long pitch;
  const void* scales;
  long long scale_row, scale_k;
  int rows;
  int square;                // 0: a scale per row, 1: per 128 rows
};

struct JbQuant {
  const void* x;
  long long ldx;             // elements between rows
  int rows, cols, type, square;
  void* codes;               // [rows, pitch] or null
  long long pitch;
  void* scales;              // byte of (row, block of columns) at row * scale_row + block * scale_k
  long long scale_row, scale_k;
  void* codes_t;             // transposed [cols, pitch_t] or null
  long long pitch_t;
  void* scales_t;
  long long scale_t_row, scale_t_k;
  const void* rstd;          // fp32 per row, or null: values are x * rstd * gain
  const void* gain;          // per column, or null
  int gain_type;
  void* colsum;              // fp32 [ceil(rows / 128), cols], or null
};

struct JbRms {
  const void* x;
  const void* residual;      // or null
  long long ldx, ldr;
  int rows, cols, type;
  float eps;
  const void* gain;          // or null
  int gain_type;
  void* sum;                 // contiguous, given exactly with a residual
  void* rstd;                // fp32 per row, or null
  void* y;                   // contiguous, or null
  int y_type;                // the type of x, or 0
  void* codes;               // [rows, pitch], or null
  long long pitch;
  void* scales;
  long long scale_row, scale_k;
};

struct JbRmsBwd {
  const void* t;             // the normalised sum
  long long ldt;
  const void* g;             // gradient of the output, contiguous: the type of t, or fp32
  int g_f32;
  const void* gsum;          // gradient of the sum, type of t, contiguous, or null
  const void* rstd;
  const void* gain;
  int gain_type;
  int rows, cols, type;
  void* dx;                  // contiguous
  void* part;                // fp32 [jb_rms_bwd_parts, cols], or null
};

extern "C" {
int jb_scaled_gemm(const JbScaledOperand* a, const JbScaledOperand* b, long long K, void* out, long long ldo, int out_type,
                   const void* bias, int bias_type, int sm_count, int* status, void* stream);
int jb_quantize(const JbQuant* q, int sm_count, void* stream);
int jb_column_sum(const float* part, int P, int C, void* out, int out_type, void* stream);
int jb_rms_max_cols();
int jb_rms_norm_fwd(const JbRms* q, int sm_count, void* stream);
int jb_rms_bwd_parts(const JbRmsBwd* q, int sm_count);
int jb_rms_norm_bwd(const JbRmsBwd* q, int sm_count, int* status, void* stream);
}
