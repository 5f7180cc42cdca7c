// Matrix products of 8-bit integers with one scale per row of either operand (per token and per
// channel), and the quantisation of bf16 rows that feeds them.
//
// A row r in 8 bits: scale s = max|r| times fp32(1 / 127), rounded to fp32 (within an ulp of max|r| / 127, without
// a division), q = r / s rounded to nearest, ties to even, exactly (below). y[m, n] = fp32(sum_k xq[m, k] wq[n, k]) * fp32(xs[m] * ws[n]): the sum is a whole number and
// exact in int32 whatever the order (|sum| <= 2^30), so every kernel and every split here gives the same bits,
// whatever the batch.
#include "fl_int8.h"
#include <algorithm>

namespace {

typedef int i8_x4 __attribute__((ext_vector_type(4)));

// ---- quantisation -------------------------------------------------------------------------------

// x / s rounded to the nearest whole number, ties to even, for |x| <= 127 s (1 + 2^-22). The product with
// 1 / s is off by a few ulp, which matters next to a half (x = max / 2 gives 63.5, often), so the remainder
// r = x - q s decides. It is exact in one fma: q s has at most 31 bits and |r| <= s, a multiple of an ulp
// of the smaller of x and s.
struct Q8Row {
  float s, inv, up;  // scale; 1 / (s up); up: a power of two that keeps 1 / s of tiny rows finite
};
__device__ __forceinline__ Q8Row q8_row(float amax) {
  Q8Row r;
  r.s = amax < INFINITY ? amax * (1.0f / 127.0f) : __builtin_nanf("");
  r.up = amax < 0x1p-64f ? 0x1p80f : 1.0f;
  r.inv = r.s > 0.0f ? 1.0f / (r.s * r.up) : 0.0f;  // zero rows and rows with a NaN or an infinity: q = 0
  return r;
}
__device__ __forceinline__ int q8_of(float x, const Q8Row& row) {
  float q = __builtin_rintf(x * row.up * row.inv);
  const float r = __builtin_fmaf(-q, row.s, x), two = r + r;
  const bool odd = ((int)q & 1) != 0;
  if (two > row.s || (two == row.s && odd)) q += 1.0f;
  if (two < -row.s || (two == -row.s && odd)) q -= 1.0f;
  return row.inv != 0.0f ? (int)fminf(fmaxf(q, -127.0f), 127.0f) : 0;
}

constexpr int Q8_NT = 256, Q8_KEEP = 4;  // threads of a row; 8-value pieces that a thread keeps in registers

// One workgroup per row; rows of up to 8192 values are read once.
__global__ __launch_bounds__(Q8_NT) void k_quantize_i8(const uint16_t* __restrict__ x, int8_t* __restrict__ qo,
                                                       float* __restrict__ scale, int k) {
  __shared__ float red[Q8_NT / FL_WAVE];
  const int tid = threadIdx.x, nc = k >> 3;
  const int64_t row = blockIdx.x;
  const uint4* xr = reinterpret_cast<const uint4*>(x + row * k);
  uint4 v[Q8_KEEP];
  // the largest magnitude as its bf16 bits: a NaN's are above an infinity's, and both win
  uint32_t mx = 0;
  auto look = [&](const uint4& c) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = max(mx, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
  };
#pragma unroll
  for (int i = 0; i < Q8_KEEP; ++i) {
    const int c = tid + i * Q8_NT;
    v[i] = c < nc ? xr[c] : make_uint4(0, 0, 0, 0);
    look(v[i]);
  }
  for (int c = tid + Q8_KEEP * Q8_NT; c < nc; c += Q8_NT) look(xr[c]);
  // integers below 2^15 are exact floats, and larger ones stay larger
  const float wm = wave_max((float)mx);
  if ((tid & 63) == 0) red[tid >> 6] = wm;
  __syncthreads();
  const uint32_t m = (uint32_t)fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const Q8Row r = q8_row(bf2f(m));
  if (tid == 0) scale[row] = r.s;
  uint2* qr = reinterpret_cast<uint2*>(qo + row * k);
  auto put = [&](int c, const uint4& p) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
    uint32_t o[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = (uint32_t)q8_of(bflo(w[i]), r) & 0xFFu, b = (uint32_t)q8_of(bfhi(w[i]), r) & 0xFFu;
      o[i >> 1] |= (a | b << 8) << (16 * (i & 1));
    }
    qr[c] = make_uint2(o[0], o[1]);
  };
#pragma unroll
  for (int i = 0; i < Q8_KEEP; ++i) {
    const int c = tid + i * Q8_NT;
    if (c < nc) put(c, v[i]);
  }
  for (int c = tid + Q8_KEEP * Q8_NT; c < nc; c += Q8_NT) put(c, xr[c]);
}

// ---- the product ----------------------------------------------------------------------------------

template <bool F32>
__device__ __forceinline__ void i8_store(void* y, int64_t at, int acc, float s) {
  const float v = (float)acc * s;
  if (F32) reinterpret_cast<float*>(y)[at] = v;
  else reinterpret_cast<uint16_t*>(y)[at] = (uint16_t)f2bf(v);
}

// Up to 16 MB rows of x against 16 weight rows per workgroup, whose KW waves each take a part of K. Lane
// (r = l % 16, c = l / 16) of a wave holds 16 values of weight row r, and of x row r, at 64 step + 16 c: A and B
// of v_mfma_i32_16x16x64_i8, which sums over k in any order as long as both operands use the same. D: x row
// l % 16, weight rows 4 (l / 16) + 0..3.
template <int MB, int KW, bool F32>
__global__ __launch_bounds__(64 * KW) void k_i8_rows(const int8_t* __restrict__ xq, const float* __restrict__ xs,
                                                     const int8_t* __restrict__ wq, const float* __restrict__ ws,
                                                     void* __restrict__ y, int m, int n, int k) {
  __shared__ i8_x4 part[KW > 1 ? KW - 1 : 1][MB][64];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MB;
  const int steps = (k + 63) >> 6, per = (steps + KW - 1) / KW;
  const int s0 = wave * per, s1 = min(steps, s0 + per);
  // range-checked from the first row of the block: rows past the end read as zeros
  const auto wr = buf_rsrc(wq + (int64_t)n0 * k, (uint32_t)min(16, n - n0) * (uint32_t)k);
  const auto xr = buf_rsrc(xq + (int64_t)m0 * k, (uint32_t)min(16 * MB, m - m0) * (uint32_t)k);
  i8_x4 acc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) acc[b] = i8_x4{0, 0, 0, 0};
#pragma unroll 4
  for (int s = s0; s < s1; ++s) {
    const int at = s * 64 + c * 16;
    const uint32_t off = at < k ? (uint32_t)(r * k + at) : 0xFFFFFFF0u;  // past the row: zeros
    const i8_x4 w = __builtin_bit_cast(i8_x4, buf_ld128(wr, off));
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      const i8_x4 x = __builtin_bit_cast(i8_x4, buf_ld128(xr, at < k ? off + (uint32_t)(16 * b * k) : 0xFFFFFFF0u));
      acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, acc[b], 0, 0, 0);
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int b = 0; b < MB; ++b) part[wave - 1][b][lane] = acc[b];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int b = 0; b < MB; ++b) {
#pragma unroll
    for (int p = 0; p < KW - 1; ++p) acc[b] += part[p][b][lane];
    const int mm = m0 + 16 * b + r;
    if (mm >= m) continue;
    const float sx = xs[mm];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int nn = n0 + 4 * c + i;
      if (nn < n) i8_store<F32>(y, (int64_t)mm * n + nn, acc[b][i], sx * ws[nn]);
    }
  }
}

}  // namespace

int i8_quantize(const uint16_t* x, int8_t* q, float* scale, int32_t rows, int32_t k, hipStream_t s) {
  hipLaunchKernelGGL(k_quantize_i8, dim3(rows), dim3(Q8_NT), 0, s, x, q, scale, k);
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}

int64_t i8_gemm_bytes(int32_t, int32_t, int32_t) { return 0; }

int i8_gemm(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, void* y, bool y_fp32, void*,
            int32_t m, int32_t n, int32_t k, hipStream_t s) {
  constexpr int Y = 32768 * 32;  // rows per launch (the grid's second dimension)
  for (int64_t m0 = 0; m0 < m; m0 += Y) {
    const int mm = (int)std::min<int64_t>(Y, m - m0);
    void* yy = static_cast<char*>(y) + m0 * n * (y_fp32 ? 4 : 2);
    const dim3 grid((n + 15) / 16, (mm + 31) / 32);
    if (y_fp32) hipLaunchKernelGGL((k_i8_rows<2, 4, true>), grid, dim3(256), 0, s, xq + m0 * k, xs + m0, wq, ws, yy, mm, n, k);
    else hipLaunchKernelGGL((k_i8_rows<2, 4, false>), grid, dim3(256), 0, s, xq + m0 * k, xs + m0, wq, ws, yy, mm, n, k);
  }
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}

extern "C" {

int fl_quantize_int8(const uint16_t* x, int8_t* q, float* scale, int32_t rows, int32_t k, void* stream) {
  if (!i8_aligned(x) || !i8_aligned(q) || !scale || !i8_shape_ok(rows, 1, k)) return FL_E_ARG;
  return i8_quantize(x, q, scale, rows, k, reinterpret_cast<hipStream_t>(stream));
}

int fl_gemm_int8_workspace(int32_t m, int32_t n, int32_t k, int64_t* bytes) {
  if (!bytes || !i8_shape_ok(m, n, k)) return FL_E_ARG;
  *bytes = i8_gemm_bytes(m, n, k);
  return FL_OK;
}

int fl_gemm_int8(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, void* y, int32_t y_fp32,
                 void* work, int32_t m, int32_t n, int32_t k, void* stream) {
  if (!i8_shape_ok(m, n, k) || !i8_aligned(xq) || !i8_aligned(wq) || !xs || !ws || !i8_aligned(y) ||
      (i8_gemm_bytes(m, n, k) > 0 && !i8_aligned(work)))
    return FL_E_ARG;
  return i8_gemm(xq, xs, wq, ws, y, y_fp32 != 0, work, m, n, k, reinterpret_cast<hipStream_t>(stream));
}

int fl_linear_int8_workspace(int32_t m, int32_t n, int32_t k, int64_t* bytes) {
  if (!bytes || !i8_shape_ok(m, n, k)) return FL_E_ARG;
  *bytes = i8_pad((int64_t)m * k) + i8_pad((int64_t)m * 4) + i8_gemm_bytes(m, n, k);
  return FL_OK;
}

int fl_linear_int8(const uint16_t* x, const int8_t* wq, const float* ws, void* y, int32_t y_fp32, void* work,
                   int32_t m, int32_t n, int32_t k, void* stream) {
  if (!i8_shape_ok(m, n, k) || !i8_aligned(x) || !i8_aligned(wq) || !ws || !i8_aligned(y) || !i8_aligned(work))
    return FL_E_ARG;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  int8_t* xq = static_cast<int8_t*>(work);
  float* xs = reinterpret_cast<float*>(xq + i8_pad((int64_t)m * k));
  const int rc = i8_quantize(x, xq, xs, m, k, s);
  if (rc != FL_OK) return rc;
  return i8_gemm(xq, xs, wq, ws, y, y_fp32 != 0, reinterpret_cast<char*>(xs) + i8_pad((int64_t)m * 4), m, n, k, s);
}

}  // extern "C"
