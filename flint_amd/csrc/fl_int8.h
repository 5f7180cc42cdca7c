// 8-bit integer products between the files that launch them: the entry points (fl_int8.hip) and the
// scoring of features through an 8-bit vocabulary head (fl_logprobs.hip).
#pragma once
#include "fl_common.h"

constexpr int I8_MAX_K = 65536;  // |sum| <= 128 * 128 * 65536 = 2^30: the int32 sums cannot wrap
constexpr int I8_MAX_ROWS = 1 << 23;  // of either operand (a grid's threads are counted in 32 bits)

inline bool i8_shape_ok(int32_t m, int32_t n, int32_t k) {
  return m >= 1 && n >= 1 && m <= I8_MAX_ROWS && n <= I8_MAX_ROWS && k >= 16 && k % 16 == 0 && k <= I8_MAX_K;
}
inline bool i8_aligned(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int64_t i8_pad(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// bytes of the product's own workspace (0: none)
int64_t i8_gemm_bytes(int32_t m, int32_t n, int32_t k);
// y [m, n] (bf16, or fp32) = (xq . wq^T) xs ws; arguments already checked
int i8_gemm(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, void* y, bool y_fp32, void* work,
            int32_t m, int32_t n, int32_t k, hipStream_t s);
// rows of x [rows, k] (bf16) in 8 bits; arguments already checked
int i8_quantize(const uint16_t* x, int8_t* q, float* scale, int32_t rows, int32_t k, hipStream_t s);
// the same from bf16 rows x, quantised on the way
int64_t i8_linear_bytes(int32_t m, int32_t n, int32_t k);
int i8_linear(const uint16_t* x, const int8_t* wq, const float* ws, void* y, bool y_fp32, void* work, int32_t m,
              int32_t n, int32_t k, hipStream_t s);
