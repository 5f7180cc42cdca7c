// Matrix products of 8-bit integers with one scale per row of either operand (per token and per
// channel), and the quantisation of bf16 rows that feeds them.
//
// A row r in 8 bits: scale s = max|r| times fp32(1 / 127), rounded to fp32, q = r / s rounded to nearest, ties to even,
// exactly (below). The product is the definition, as in the form that torch gives max / 127 on a device; it is not always
// the rounded quotient: where the maximum's 8 bits are 143, 144, 175, 207, 208 or 239, s is an ulp below fp32(max / 127),
// and a value of exactly max / 2 is a hair above 63.5 steps, so 64, where the quotient's scale would make it 63. No other
// q differs. Either is within half a step.
// y[m, n] = fp32(sum_k xq[m, k] wq[n, k]) * fp32(xs[m] * ws[n]): the sum is a whole number and exact in int32 whatever
// the order (|sum| <= 2^30), so every kernel and every split here gives the same bits, whatever the batch. Rounded: the
// sum to fp32 (24 bits of at most 30), the scales' product, theirs with the sum, and that to bf16 where y is.
#include "fl_int8.h"
#include <algorithm>
#include <type_traits>

namespace {

typedef int i8_x4 __attribute__((ext_vector_type(4)));

// ---- quantisation -------------------------------------------------------------------------------

// x / s rounded to the nearest whole number, ties to even, for |x| <= 127 s (1 + 2^-22) (127.008 s where s is
// subnormal and has few bits). t = x (1 / s) is off by at most 127.008 * 2^-22, so its nearest whole number q may be one off next to a half, and x = max / 2, which gives 63.5,
// is frequent: the remainder r = x - q s decides. It is exact in one fma: q s has at most 31 bits and |r| <= s is a
// multiple of an ulp of the smaller of x and s. An exact half needs s to be a power of two (x has 8 bits, and max / 127
// to 24 bits has few only if 127 divides max's), and then t is exact and its rounding went to the even side.
struct Q8Row {
  float s;           // the scale
  float w, h, inv;   // s, half of it and 1 / s; of tiny rows, whose 1 / s is not finite, of s times 2^80
  bool tiny;
};
constexpr float Q8_UP = 0x1p80f;
__device__ __forceinline__ Q8Row q8_row(float amax) {
  Q8Row r;
  r.s = amax < INFINITY ? amax * (1.0f / 127.0f) : __builtin_nanf("");
  r.tiny = amax < 0x1p-64f;
  r.w = r.tiny ? r.s * Q8_UP : r.s;
  r.h = 0.5f * r.w;
  r.inv = r.s > 0.0f ? __builtin_amdgcn_rcpf(r.w) : 0.0f;  // zero rows and rows with a NaN or an infinity: q = 0
  return r;
}
// eight bf16 values
__device__ __forceinline__ uint2 q8_pack(const uint4& p, const Q8Row& row) {
  if (!(row.inv != 0.0f)) return make_uint2(0, 0);
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = bflo(w[i]), x[2 * i + 1] = bfhi(w[i]);
  if (row.tiny) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= Q8_UP;
  }
  uint32_t o[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = __builtin_rintf(x[i] * row.inv), r = __builtin_fmaf(-q, row.w, x[i]);
    const float one = fabsf(r) > row.h ? __builtin_copysignf(1.0f, r) : 0.0f;
    o[i >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(q + 128.0f + one, i & 3, o[i >> 2]);  // 1..255
  }
  return make_uint2(o[0] ^ 0x80808080u, o[1] ^ 0x80808080u);
}

constexpr int Q8_NT = 256, Q8_KEEP = 5;  // threads of a workgroup; 8-value pieces that a lane keeps in registers

// WR waves per row, 4 / WR rows per workgroup; rows of up to 2560 WR values are read once. Bound by the launch up to some
// hundred rows (32 x 2560 3.0 us), then by memory: 2048 x 2560 5.3 us, 3 TB/s, with 11 vector instructions a value beside.
template <int WR>
__global__ __launch_bounds__(Q8_NT) void k_quantize_i8(const uint16_t* __restrict__ x, int8_t* __restrict__ qo,
                                                       float* __restrict__ scale, int rows, int k) {
  constexpr int LANES = 64 * WR;
  __shared__ float red[Q8_NT / FL_WAVE];
  const int tid = threadIdx.x % LANES, nc = k >> 3;
  const int64_t row = (int64_t)blockIdx.x * (Q8_NT / LANES) + threadIdx.x / LANES;
  if (WR < 4 && row >= rows) return;
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
    const int c = tid + i * LANES;
    v[i] = c < nc ? xr[c] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < Q8_KEEP; ++i) look(v[i]);
  for (int c = tid + Q8_KEEP * LANES; c < nc; c += LANES) look(xr[c]);
  // integers below 2^15 are exact floats, and larger ones stay larger
  float am = wave_max((float)mx);
  if constexpr (WR > 1) {
    if ((tid & 63) == 0) red[threadIdx.x >> 6] = am;
    __syncthreads();
    am = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    static_assert(WR == 4, "all waves on one row");
  }
  const Q8Row r = q8_row(bf2f((uint32_t)am));
  if (tid == 0) scale[row] = r.s;
  uint2* qr = reinterpret_cast<uint2*>(qo + row * k);
#pragma unroll
  for (int i = 0; i < Q8_KEEP; ++i) {
    const int c = tid + i * LANES;
    if (c < nc) qr[c] = q8_pack(v[i], r);
  }
  for (int c = tid + Q8_KEEP * LANES; c < nc; c += LANES) qr[c] = q8_pack(xr[c], r);
}

// ---- the product ----------------------------------------------------------------------------------

template <bool F32>
__device__ __forceinline__ void i8_store(void* y, int64_t at, int acc, float s) {
  const float v = (float)acc * s;
  if (F32) reinterpret_cast<float*>(y)[at] = v;
  else reinterpret_cast<uint16_t*>(y)[at] = (uint16_t)f2bf(v);
}

// Up to 16 MB rows of x against all weights, 16 weight rows (a block) at a time: the eight waves of a workgroup
// each take a part of K. Lane (r = l % 16, c = l / 16) of a wave holds 16 values of weight row r, and of x row r, at
// 64 step + 16 c: A and B of v_mfma_i32_16x16x64_i8, which sums over k in any order as long as both operands use
// the same. D: x row l % 16, weight rows 4 (l / 16) + 0..3. Weights go from memory to registers, U steps at once, and
// the waves' sums meet in LDS.
// XKB = 0: one block per workgroup, x from memory beside the weights. XKB > 0: the workgroups that fit the chip at
// once take blocks in turn, with two sets of registers in turn across them and x in XKB KB of LDS: every block reading x
// again would cost as much as the weights at 16 rows. QUANT: x is bf16 and the workgroup quantises the rows for itself
// into LDS, behind its first weight loads.
// Bound by the weights' way from memory: 8 x 49152 x 2560 26.6 us, 4.7 TB/s (matrix pipes 1% busy; a wave per block,
// without the sums' meeting, is no faster); below some 10 MB of weights by one launch's start, a memory latency and the end:
// 2560 x 2560 with one row quantised here 5.1 us.
constexpr int FEW_KW = 8;
constexpr int QF_MOST = 32768, QF_KEEP = 8;  // values that a workgroup quantises; 8-value pieces of a lane
// log2 of the waves of a row, so that the eight hold as many rows at once as there are (all eight one row at most)
__host__ __device__ inline int qf_log_waves(int m) { return m > 4 ? 0 : m > 2 ? 1 : m > 1 ? 2 : 3; }
// Whether the product's workgroups quantise the rows themselves: if the waves hold them in QF_KEEP pieces a lane, and if
// it beats a launch of its own before the product. us, on the way and before it, of the kernels alone; called one by one
// the two launches take 8 at least.
// - up to 4 rows: 2 x 5003 x 2560 7.3 and 8.0, 4 x 8192 x 2560 8.4 and 9.3, 4 x 16384 x 4096 15.2 and 17.0; but
//   4 x 49152 x 512 11.7 and 10.4, the rows again in every workgroup beside a short K;
// - up to 8: 8 x 8192 x 1024 6.0 and 7.0, 8 x 5003 x 1600 6.5 and 6.5, 8 x 8192 x 2560 9.2 and 9.3, 8 x 49152 x 2560 26.8
//   and 29.8; 8 x 4096 x 4096 9.4 and 8.7, 8 x 16384 x 1600 10.5 and 9.8; between the two lines 8 x 16384 x 2560 12.8 and
//   12.6, 5 x 16384 x 2560 12.5 both, but 8 x 24576 x 2560 15.0 and 15.6, 8 x 32752 x 2560 17.0 and 18.8: the upper line could
//   lie lower;
// - up to 16: 12 x 8192 x 1024 6.5 and 7.2, 16 x 5003 x 1024 7.1 and 7.2 (10 x 5003 x 1600 7.5 and 6.5: then the calls
//   decide); 16 x 12000 x 1024 8.5 and 8.0, 16 x 49152 x 2048 24.0 and 23.5.
inline bool qf_pays(int m, int n, int k) {
  const int lw = qf_log_waves(m), slots = FEW_KW >> lw, w = 64 << lw;
  const int64_t values = (int64_t)m * k;
  if (m > 16 || values > QF_MOST || (m + slots - 1) / slots * ((k / 8 + w - 1) / w) > QF_KEEP) return false;
  if (m <= 4) return k >= 1024 || n < 32768;
  if (m <= 8) return n <= 12288 ? values <= 20480 : n >= 32768 && k > 1024;
  return n <= 8192 && values <= 16384;
}
// of x rows in LDS: r and r + 8 on the same banks
__host__ __device__ inline int few_pitch(int k) { return ((k + 63) >> 6) * 64 + 16; }
struct I8Few {
  const void* x;     // int8 [m, k], or (QUANT) bf16
  const float* xs;   // not with QUANT
  const int8_t* wq;
  const float* ws;
  void* y;
  int m, n, k;
};
template <int MB, int XKB, bool QUANT, bool F32>
__global__ __launch_bounds__(64 * FEW_KW, 4) void k_i8_few(I8Few a) {
  constexpr int KW = FEW_KW, U = 5;
  static_assert(!QUANT || (MB == 1 && XKB * 1024 >= QF_MOST + 16 * 64), "the rows, each up to 64 bytes longer");
  __shared__ __align__(16) int part[XKB ? 2 : 1][KW][MB][256];
  __shared__ __align__(16) unsigned char xl[XKB ? XKB * 1024 : 16];
  __shared__ float most[16][KW], sx[16];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int m = a.m, k = a.k;
  const int steps = (k + 63) >> 6, per = (steps + KW - 1) / KW, turns = (per + U - 1) / U;
  const int s0 = wave * per, s1 = min(steps, s0 + per);
  const int blocks = (a.n + 15) >> 4;
  const auto xr = buf_rsrc(a.x, (uint32_t)m * (uint32_t)k);
  const int pitch = few_pitch(k);
  // this thread's outputs: x row `row`, weight row tn of a block
  const int tn = threadIdx.x & 15, row = threadIdx.x >> 4;
  struct Set {
    i8_x4 w[U], x[U][XKB ? 1 : MB];
    float s;  // the scale of weight row tn
  };
  // the U steps of block b from turn t on; range-checked: rows past the end, steps past the wave's part: zeros
  auto load = [&](int b, int t, Set& v) {
    const bool live = b < blocks;  // wave-uniform
    const int n0 = b * 16;
    const uint32_t rows = live ? (uint32_t)min(16, a.n - n0) : 0u;
    const auto wr = buf_rsrc(a.wq + (int64_t)(live ? n0 : 0) * k, rows * (uint32_t)k);
    if (t == turns - 1) v.s = live ? a.ws[min(n0 + tn, a.n - 1)] : 0.0f;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int s = s0 + t * U + i, at = s * 64 + c * 16;
      const bool in = s < s1 && at < k;
      v.w[i] = __builtin_bit_cast(i8_x4, buf_ld128(wr, in ? (uint32_t)(r * k + at) : 0x80000000u));
      if constexpr (XKB == 0) {
#pragma unroll
        for (int j = 0; j < MB; ++j)
          v.x[i][j] = __builtin_bit_cast(i8_x4, buf_ld128(xr, in ? (uint32_t)((16 * j + r) * k + at) : 0x80000000u));
      }
    }
  };
  i8_x4 acc[MB];
  Set A, B;
  int b = blockIdx.x, t = 0;
  // (block, turn) pairs in order
  auto next = [&](int& nb, int& nt) {
    nt = t + 1, nb = b;
    if (nt == turns) nt = 0, nb = b + (int)gridDim.x;
  };
  if constexpr (XKB > 0 && !QUANT) {  // a row per wave; beyond k of the last step: what LDS holds, times zeros
    const uint32_t at = (uint32_t)(uintptr_t)(lds_byte*)xl;
    const fl_u32x4 xv = buffer_words(a.x, (uint32_t)m * (uint32_t)k);
    for (int i = wave; i < m; i += KW)
      for (int p = 0; p < k; p += 1024)
        if (p + lane * 16 < k) dma_1k(xv, at + (uint32_t)(i * pitch + p), (uint32_t)(lane * 16), (uint32_t)(i * k + p));
  }
  load(b, 0, A);
  if constexpr (XKB > 0) {
    int nb, nt;
    next(nb, nt);
    load(nb, nt, B);
    if constexpr (!QUANT) {
      wait_loads<2 * U>();  // x is here; the weights, requested after it, need not be
      __syncthreads();
    }
  }
  if constexpr (QUANT) {
    // Waves in `slots` groups of W: a group takes rows slot, slot + slots, ..., its waves 64 W pieces of 8 values at a
    // time; the pieces (QF_KEEP a lane at most, by qf_pays) stay in registers between the maximum
    // and the quotients.
    const int lw = qf_log_waves(m), W = 1 << lw, slots = KW >> lw, slot = wave >> lw, sub = wave & (W - 1);
    const int nc = k >> 3, cpr = (nc + 64 * W - 1) >> (6 + lw);
    const uint4* xb = static_cast<const uint4*>(a.x);
    uint4 v[QF_KEEP];
    int qr = slot, j = 0;  // of piece i
#pragma unroll
    for (int i = 0; i < QF_KEEP; ++i) {
      const int ch = (j * W + sub) * 64 + lane;
      v[i] = qr < m && ch < nc ? xb[qr * nc + ch] : make_uint4(0, 0, 0, 0);
      if (++j == cpr) j = 0, qr += slots;
    }
    uint32_t mx = 0;
    qr = slot, j = 0;
#pragma unroll
    for (int i = 0; i < QF_KEEP; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = max(mx, max(w[e] & 0x7FFFu, (w[e] >> 16) & 0x7FFFu));
      if (++j == cpr) {
        if (qr < m) {  // wave-uniform
          const float wm = wave_max((float)mx);
          if (lane == 0) most[qr][sub] = wm;
        }
        mx = 0, j = 0, qr += slots;
      }
    }
    __syncthreads();
    Q8Row q{};
    qr = slot, j = 0;
#pragma unroll
    for (int i = 0; i < QF_KEEP; ++i) {
      const int ch = (j * W + sub) * 64 + lane;
      if (qr < m) {
        if (j == 0) {
          q = q8_row(bf2f((uint32_t)wave_max(most[qr][lane & (W - 1)])));
          if (lane == 0) sx[qr] = q.s;
        }
        if (ch < nc) *reinterpret_cast<uint2*>(xl + qr * pitch + ch * 8) = q8_pack(v[i], q);
      }
      if (++j == cpr) j = 0, qr += slots;
    }
    __syncthreads();
  }
  const float sr = row < 16 * MB && row < m ? (QUANT ? sx[row & 15] : a.xs[row]) : 0.0f;
  int buf = 0;
  // one turn of a block; the last one ends it
  auto turn = [&](int t, const Set& v) {
    if (t == 0) {
#pragma unroll
      for (int j = 0; j < MB; ++j) acc[j] = i8_x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        i8_x4 x;
        if constexpr (XKB == 0) x = v.x[i][j];
        else  // the last row again for lanes behind it (not stored); a step within the row
          x = *reinterpret_cast<const i8_x4*>(xl + min(16 * j + r, m - 1) * pitch + min(s0 + t * U + i, steps - 1) * 64 +
                                              c * 16);
        acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v.w[i], x, acc[j], 0, 0, 0);
      }
    }
    if (t < turns - 1) return;
#pragma unroll
    for (int j = 0; j < MB; ++j) *reinterpret_cast<i8_x4*>(&part[buf][wave][j][lane * 4]) = acc[j];
    lds_barrier();
    // a thread adds up and stores one value, 16 weight rows side by side. The next block's sums go to the other
    // buffer, and a wave that is there has passed this barrier: the one after is enough for this buffer.
    const int nn = b * 16 + tn;
    if (row < 16 * MB && row < m && nn < a.n) {
      int sum = 0;
#pragma unroll
      for (int p = 0; p < KW; ++p) sum += part[buf][p][row >> 4][((tn >> 2) * 16 + (row & 15)) * 4 + (tn & 3)];
      i8_store<F32>(a.y, (int64_t)row * a.n + nn, sum, sr * v.s);
    }
    if (XKB) buf ^= 1;
  };
  if constexpr (XKB == 0) {
    for (; t < turns; ++t) {
      turn(t, A);
      if (t + 1 < turns) load(b, t + 1, A);
    }
    return;
  }
  // the loads of the two pairs after the one at work are in flight
  auto go = [&](Set& v) {
    turn(t, v);
    int nb, nt;
    next(nb, nt);
    b = nb, t = nt;
    next(nb, nt);
    load(nb, nt, v);
  };
  while (b < blocks) {
    go(A);
    if (b >= blocks) break;
    go(B);
  }
}

// ---- tiles ------------------------------------------------------------------------------------------
// A workgroup of WM x WN waves computes T rows of x against T weight rows over one part of K, in steps of 128
// bytes of K. The two units of a step, weights and x, go straight from memory into LDS (buffer_load ... lds, 1 KB = 8
// rows of 128 bytes per wave instruction), into a ring of NR units. In LDS the 16-byte piece c of row r sits at
// c ^ (r / 2 % 8), so that 16 lanes on one piece of 16 rows take all 64 banks once (c ^ r % 8: 8.5 M conflict cycles in
// 90 us); the lanes of the load fetch the pieces in that order. Waves use 32x32x32 MFMAs: a lane (r = l % 32, h = l /
// 32) holds piece 2 j + h of row r at sub-step j. Weights are operand A: a lane ends with x row l % 32 and weight
// rows 8 (i / 4) + 4 h + i % 4.
// What bounds the tiles of 256, at 2048 x 16384 x 2560 (two rounds of 256 tiles, 84 us, 2.0 POPS, the matrix pipes busy in
// 0.48 of the cycles at 2.04 GHz): 1.59 us a step, of which the MFMAs and their reads of LDS alone take 1.39, at the clock
// that the card then keeps; 6 us a round for its start and end, 5.5 for bf16 results (8.3 for fp32). Hiding the ends does
// not pay, the time goes with the work done: tiles started 0 to 8 us apart, so that few store at a time, take 85 to 86, and
// two workgroups a CU of 192 x 128, with 1.7 times the reads from L2, 97.

typedef int i8_x16 __attribute__((ext_vector_type(16)));
typedef int i8_out32 __attribute__((ext_vector_type(4), aligned(4)));
typedef float i8_scale4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t i8_out16 __attribute__((ext_vector_type(4), aligned(2)));

struct I8Tile {
  const int8_t *xq, *wq;
  const float *xs, *ws;
  void* y;       // bf16 or fp32 [m, n]; with splits int32 [splits, m, n] part sums
  int m, n, k;
  int mblk, nblk, splits, sps;  // tiles along m and n; parts of K and their steps of 128
};

// KW > 1: the waves are KW ways of one wave, each over its own steps with a ring of its own, for calls of few tiles,
// where a step's latency counts: a way needs no barrier, and its products are four times those of a wave that shares the
// tile with three others (333 x 2570 x 2560 11 -> 8.8 us). The ways' sums meet in LDS.
template <int T, int KW, int WM, int WN, int NR, int OUT>  // OUT: 0 bf16, 1 fp32, 2 int32 part sums
__global__ __launch_bounds__(64 * KW * WM * WN, KW * WM * WN > 4 ? 2 : 1) void k_i8_tile(I8Tile a) {
  constexpr int NW = WM * WN, TM = T / WM, TN = T / WN, FM = TM / 32, FN = TN / 32;
  constexpr int PER = T / 8 / NW, UNIT = T * 128;  // loads of a wave for a unit; its bytes
  static_assert(T % (8 * NW) == 0 && TM % 32 == 0 && TN % 32 == 0 && NR >= 4, "whole loads, two steps");
  static_assert(KW == 1 || NW == 1, "ways take their own numbers of steps: no barrier between them");
  // at the end, in the units' place: 32 rows of x by TN sums of a wave at a time; with ways all sums of each
  constexpr int LD = KW == 1 ? TN + 4 : T + 4, SLAB = (KW == 1 ? 32 : T) * LD * 4, SLABS = KW == 1 ? NW : KW;
  constexpr int SMEM = KW * NR * UNIT > SLABS * SLAB ? KW * NR * UNIT : SLABS * SLAB;
  __shared__ __align__(1024) unsigned char smem[SMEM];
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int wv0 = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int way = wv0 / NW, wave = wv0 % NW, wm = wave % WM, wn = wave / WM;
  // an XCD's workgroups (blockIdx % 8) take neighbouring tiles: up to 8 along m, then along n
  const int tiles = a.mblk * a.nblk * a.splits, share = (tiles + 7) >> 3;
  const int t = (int)(blockIdx.x & 7) * share + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= share || t >= tiles) return;
  const int split = t / (a.mblk * a.nblk), tt = t - split * (a.mblk * a.nblk);
  const int grp = tt / (8 * a.nblk), gm = min(8, a.mblk - grp * 8), in = tt - grp * 8 * a.nblk;
  const int m0 = (grp * 8 + in % gm) * T, n0 = (in / gm) * T;
  const int steps = (a.k + 127) >> 7;
  // the workgroup's part of K, the way's of that
  const int p0 = split * a.sps, p1 = min(steps, p0 + a.sps), per = (p1 - p0 + KW - 1) / KW;
  const int s0 = p0 + way * per, s1 = min(p1, s0 + per);
  const int rows_n = min(T, a.n - n0), rows_m = min(T, a.m - m0);
  const fl_u32x4 wv = buffer_words(a.wq + (int64_t)n0 * a.k, (uint32_t)rows_n * (uint32_t)a.k);
  const fl_u32x4 xv = buffer_words(a.xq + (int64_t)m0 * a.k, (uint32_t)rows_m * (uint32_t)a.k);
  // this lane's piece of the wave's loads of a unit; the buffers' range check makes rows past the end zeros
  auto piece = [&](int i) { return (lane & 7) ^ (((wave * PER + i) & 1) * 4 + (lane >> 4)); };
  uint32_t off[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    off[i] = (uint32_t)((wave * PER + i) * 8 + (lane >> 3)) * (uint32_t)a.k + (uint32_t)piece(i) * 16u;
  unsigned char* const ring = smem + way * (NR * UNIT);
  const uint32_t base = (uint32_t)(uintptr_t)(lds_byte*)smem + (uint32_t)(way * NR * UNIT + wave * PER * 1024);
  const int tail = a.k & 127;  // bytes of the last step, if it is not whole
  // unit u of this part of K (2 s: weights of step s0 + s, 2 s + 1: x) into its slot, if there is such a step
  auto load = [&](int u, int slot) {
    const int s = s0 + (u >> 1);
    if (s >= s1) return;
    const bool cut = s == steps - 1 && tail != 0;  // pieces past the end of a row are zeros too
    const fl_u32x4 v = u & 1 ? xv : wv;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      dma_1k(v, base + (uint32_t)(slot * UNIT + i * 1024), cut && piece(i) * 16 >= tail ? 0x80000000u : off[i],
             (uint32_t)s * 128u);
  };
  auto meet = [&] {  // one wave's loads and reads are its own
    if (NW > 1) __builtin_amdgcn_s_barrier();
  };
  i8_x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  // Sub-step j of a step: fragments of 32 bytes of K. They are read one sub-step ahead; the last one of a step reads
  // the next step's first, behind the step's one barrier, when the next step's units have landed for every wave
  // and this step's have been read by every wave, so that their slots can be loaded again.
  struct Frag {
    i8_x4 w[FN], x[FM];
  };
  auto read = [&](int ws, int xs, int j, Frag& f) {
    const unsigned char* wt = ring + ws * UNIT + (wn * TN + r) * 128;
    const unsigned char* xt = ring + xs * UNIT + (wm * TM + r) * 128;
    const int at = ((2 * j + h) ^ ((r >> 1) & 7)) * 16;
#pragma unroll
    for (int i = 0; i < FN; ++i) f.w[i] = *reinterpret_cast<const i8_x4*>(wt + i * 32 * 128 + at);
#pragma unroll
    for (int i = 0; i < FM; ++i) f.x[i] = *reinterpret_cast<const i8_x4*>(xt + i * 32 * 128 + at);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](const Frag& f) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[j], f.x[i], acc[i][j], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int u = 0; u < NR; ++u) load(u, u);
  if (s0 + (NR - 1) / 2 < s1) wait_loads<(NR - 2) * PER>();
  else wait_loads<0>();
  meet();
  Frag A, B;
  read(0, 1, 0, A);
  int ws = 0, xs = 1;  // this step's slots
  for (int s = 0; s < s1 - s0; ++s) {
    const int wn_ = ws + 2 >= NR ? ws + 2 - NR : ws + 2, xn_ = xs + 2 >= NR ? xs + 2 - NR : xs + 2;
    read(ws, xs, 1, B);
    // the second of the two units that follow the last step's, whose slots are free since its barrier: not both at
    // once, a load instruction takes 16 cycles
    if (s > 0) load(2 * s - 1 + NR, xs >= 2 ? xs - 2 : xs - 2 + NR);
    multiply(A);
    read(ws, xs, 2, A);
    multiply(B);
    read(ws, xs, 3, B);
    multiply(A);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): B is here, this step's units are read
    // in flight behind the next step's units: those after them, NR - 4, fewer in the last steps
    if (s0 + s + (NR - 1) / 2 < s1) wait_loads<(NR - 4) * PER>();
    else wait_loads<0>();
    meet();
    load(2 * s + NR, ws);
    read(wn_, xn_, 0, A);  // (after the last step: what is there, not used)
    multiply(B);
    ws = wn_, xs = xn_;
  }
  // out through LDS, so that a wave stores whole lines
  __syncthreads();
  constexpr int V = OUT == 0 ? 8 : 4;  // values of a lane's store
  auto put = [&](const int* v, int mm, int nn, float sx, const float* sw) {  // V sums of x row mm from weight row nn on
    const int64_t at = ((int64_t)split * a.m + mm) * a.n + nn;
    float o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = OUT == 2 ? 0.0f : (float)v[e] * (sx * sw[e]);
    if (nn + V <= a.n) {  // 16 bytes, aligned to the type only where n is odd
      if (OUT == 2) *reinterpret_cast<i8_out32*>(static_cast<int*>(a.y) + at) = i8_out32{v[0], v[1], v[2], v[3]};
      else if (OUT == 1)
        *reinterpret_cast<i8_out32*>(static_cast<float*>(a.y) + at) =
            i8_out32{__float_as_int(o[0]), __float_as_int(o[1]), __float_as_int(o[2]), __float_as_int(o[3])};
      else
        *reinterpret_cast<i8_out16*>(static_cast<uint16_t*>(a.y) + at) =
            i8_out16{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4 % V], o[5 % V]),
                     pack_bf16x2(o[6 % V], o[7 % V])};
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (nn + e >= a.n) break;
        if (OUT == 2) static_cast<int*>(a.y)[at + e] = v[e];
        else if (OUT == 1) static_cast<float*>(a.y)[at + e] = o[e];
        else static_cast<uint16_t*>(a.y)[at + e] = (uint16_t)f2bf(o[e]);
      }
    }
  };
  constexpr int COLS = KW == 1 ? TN : T, LR = COLS / V;  // lanes of a row
  const int lc = (lane % LR) * V, nn = n0 + (KW == 1 ? wn * TN : 0) + lc;
  float sw[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sw[e] = OUT < 2 && nn + e < a.n ? a.ws[nn + e] : 0.0f;
  auto keep = [&](int* slab, int i, int row) {  // sums of x rows 32 i + r of the wave
#pragma unroll
    for (int f = 0; f < FN; ++f)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<i8_x4*>(slab + row * LD + f * 32 + 8 * q + 4 * h) =
            i8_x4{acc[i][f][4 * q], acc[i][f][4 * q + 1], acc[i][f][4 * q + 2], acc[i][f][4 * q + 3]};
  };
  if constexpr (KW == 1) {
    int* slab = reinterpret_cast<int*>(smem + wave * SLAB);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      keep(slab, i, r);
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int p = 0; p < 32 * LR / 64; ++p) {
        const int row = (p * 64 + lane) / LR, mm = m0 + wm * TM + i * 32 + row;
        int v[V];
#pragma unroll
        for (int e = 0; e < V; e += 4)
          *reinterpret_cast<i8_x4*>(v + e) = *reinterpret_cast<const i8_x4*>(slab + row * LD + lc + e);
        if (mm < a.m) put(v, mm, nn, OUT < 2 ? a.xs[mm] : 0.0f, sw);
      }
      __builtin_amdgcn_wave_barrier();
    }
  } else {
    int* slab = reinterpret_cast<int*>(smem);
#pragma unroll
    for (int i = 0; i < FM; ++i) keep(slab + way * (T * LD) + wn * TN, i, wm * TM + i * 32 + r);
    __syncthreads();
    for (int at = threadIdx.x; at < T * LR; at += 64 * KW * NW) {  // at % LR is lane % LR
      const int row = at / LR, mm = m0 + row;
      if (mm >= a.m) break;
      int v[V];
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        i8_x4 z = *reinterpret_cast<const i8_x4*>(slab + row * LD + lc + e);
#pragma unroll
        for (int w = 1; w < KW; ++w) z += *reinterpret_cast<const i8_x4*>(slab + w * (T * LD) + row * LD + lc + e);
        *reinterpret_cast<i8_x4*>(v + e) = z;
      }
      put(v, mm, nn, OUT < 2 ? a.xs[mm] : 0.0f, sw);
    }
  }
}

// y = the sum of the part sums, scaled: four values a thread. A launch's time: the parts are those of a few tiles
// (64 x 2560 in five parts 3.9 us)
template <bool F32>
__global__ __launch_bounds__(256) void k_i8_join(const int* __restrict__ part, int splits, const float* __restrict__ xs,
                                                 const float* __restrict__ ws, void* __restrict__ y, int m, int n) {
  const int64_t mn = (int64_t)m * n, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= mn) return;
  if ((n & 3) == 0) {
    i8_x4 v = *reinterpret_cast<const i8_x4*>(part + at);
    for (int p = 1; p < splits; ++p) v += *reinterpret_cast<const i8_x4*>(part + p * mn + at);
    const int64_t row = at / n;
    const int c = (int)(at - row * n);
    const float sx = xs[row];
    const i8_scale4 w = *reinterpret_cast<const i8_scale4*>(ws + c);
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (float)v[e] * (sx * w[e]);
    if (F32) *reinterpret_cast<float4*>(static_cast<float*>(y) + at) = make_float4(o[0], o[1], o[2], o[3]);
    else
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(y) + at) =
          make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
  } else {
    for (int64_t i = at; i < at + 4 && i < mn; ++i) {
      int v = 0;
      for (int p = 0; p < splits; ++p) v += part[p * mn + i];
      const int64_t row = i / n;
      i8_store<F32>(y, i, v, xs[row] * ws[i - row * n]);
    }
  }
}

// How a product is cut
enum I8Kind { I8_FEW, I8_T64, I8_T128, I8_T256 };
struct I8Plan {
  I8Kind kind;
  int mblk, nblk, splits, sps;  // of tiles
};

// Whether x of up to 32 rows goes through k_i8_few, which reads x once per 16 weight rows (from LDS where a workgroup
// takes several blocks) and has more weights in flight than tiles, which read x once per 64. us, few and tiles of 64:
// - 8 / 16 / 32 rows x 2560 x 2560 4.1 / 4.4 / 5.5 and 6.8 / 6.9 / 7.1;
//   x 2560 x 8192 7.6 / 9.9 / 13.7 and 10.2 / 10.2 / 10.6; 16 x 5003 x 8192 17.9 and 14.7;
// - 16 rows x 49152 x 2560, the weights from HBM, 27.7 and 29.2; 8 x 16384 x 2560 9.8 and 10.3;
//   beyond 48 KB of x in LDS 16 x 49152 x 4096 42.9 and 42.7, 16 x 16384 x 4096 15.8 and 15.1;
// - 32 rows x 16384 x 2560 11.8 and 10.9, 24 x 32768 x 2560 20.8 and 18.0, 32 x 49152 x 2560 29.9 and 31.4;
// - short rows, whose K is too little for eight waves: 16 x 16384 x 512 6.1 and 4.7.
constexpr int FEW_LDS_KB = 48;
bool i8_few_rows(int m, int n, int k) {
  if (m > 16) return m <= 32 && n <= 4096 && k < 4096;
  if (n >= 8192) return k > 1024 && (m <= 2 || m * few_pitch(k) <= FEW_LDS_KB << 10);
  return (int64_t)m * k < 131072;
}

I8Plan i8_plan(int m, int n, int k) {
  I8Plan p{I8_FEW, 0, 0, 1, 0};
  if (i8_few_rows(m, n, k)) return p;
  const int steps = (k + 127) / 128;
  auto tiles = [&](int b) { return (int64_t)((m + b - 1) / b) * ((n + b - 1) / b); };
  // us of a round of 256 tiles: its start and end and each step, as measured over m 33..2048, n 512..16384 and
  // k 512..8192 (252 products: 1% over the best kind for each in the mean, 30% at most)
  auto rounds = [&](int b, double ends, double step) {
    return (double)((tiles(b) + 255) / 256) * (ends + step * steps);
  };
  double t64 = rounds(64, 1.0, 0.19);
  const double t128 = rounds(128, 2.0, 0.48), t256 = rounds(256, 4.0, 1.4);
  // few tiles: K in parts of twelve steps at least, 2.5 us to join them (64 x 2560 x 8192: 11.0 in five parts,
  // 17 in one)
  const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(steps / 12, 256 / tiles(64)));
  if (parts > 1) t64 = 3.5 + 0.19 * steps / parts;
  p.kind = t64 <= t128 && t64 <= t256 ? I8_T64 : t128 <= t256 ? I8_T128 : I8_T256;
  const int b = p.kind == I8_T256 ? 256 : p.kind == I8_T128 ? 128 : 64;
  p.mblk = (m + b - 1) / b;
  p.nblk = (n + b - 1) / b;
  p.splits = p.kind == I8_T64 ? parts : 1;
  p.sps = (steps + p.splits - 1) / p.splits;
  p.splits = (steps + p.sps - 1) / p.sps;
  return p;
}

template <int MB, int XKB, bool QUANT>
void i8_few(const I8Few& a, int per_cu, bool f32, hipStream_t s) {
  const int blocks = (a.n + 15) / 16;
  const dim3 grid(XKB ? std::min(blocks, 256 * per_cu) : blocks), nt(64 * FEW_KW);
  if (f32) hipLaunchKernelGGL((k_i8_few<MB, XKB, QUANT, true>), grid, nt, 0, s, a);
  else hipLaunchKernelGGL((k_i8_few<MB, XKB, QUANT, false>), grid, nt, 0, s, a);
}

template <int T, int KW, int WM, int WN, int NR>
void i8_tiles(const I8Tile& a, bool f32, hipStream_t s) {
  const unsigned grid = 8u * (unsigned)(((int64_t)a.mblk * a.nblk * a.splits + 7) / 8);
  const dim3 nt(64 * KW * WM * WN);
  if constexpr (KW > 1) {  // parts of K come with few tiles only
    if (a.splits > 1) {
      hipLaunchKernelGGL((k_i8_tile<T, KW, WM, WN, NR, 2>), dim3(grid), nt, 0, s, a);
      return;
    }
  }
  if (f32) hipLaunchKernelGGL((k_i8_tile<T, KW, WM, WN, NR, 1>), dim3(grid), nt, 0, s, a);
  else hipLaunchKernelGGL((k_i8_tile<T, KW, WM, WN, NR, 0>), dim3(grid), nt, 0, s, a);
}

}  // namespace

int i8_quantize(const uint16_t* x, int8_t* q, float* scale, int32_t rows, int32_t k, hipStream_t s) {
  // us, wave per row and workgroup per row: 32 x 2560 3.5 and 3.0, 1024 x 2560 3.9 and 4.0, 2048 x 2560 5.3 and 5.8;
  // 1024 x 8192, which a wave reads twice, 12.0 and 7.5
  const dim3 nt(Q8_NT);
  if (rows >= 1024 && k <= 64 * 8 * Q8_KEEP)
    hipLaunchKernelGGL(k_quantize_i8<1>, dim3((rows + 3) / 4), nt, 0, s, x, q, scale, rows, k);
  else
    hipLaunchKernelGGL(k_quantize_i8<4>, dim3(rows), nt, 0, s, x, q, scale, rows, k);
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}

int64_t i8_gemm_bytes(int32_t m, int32_t n, int32_t k) {
  const I8Plan p = i8_plan(m, n, k);
  return p.splits > 1 ? i8_pad((int64_t)p.splits * m * n * 4) : 0;
}

int i8_gemm(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, void* y, bool y_fp32, void* work,
            int32_t m, int32_t n, int32_t k, hipStream_t s) {
  const I8Plan p = i8_plan(m, n, k);
  if (p.kind == I8_FEW) {
    const I8Few a{xq, xs, wq, ws, y, m, n, k};
    if (m > 16) i8_few<2, 0, false>(a, 0, y_fp32, s);
    // x in LDS and blocks in turn, and x from memory with a block a workgroup: us, 8 / 16 x 49152 x 2560 27 / 28 and
    // 31 / 38, 1 x 49152 x 2560 26 and 24, 8 x 5003 x 1600 4.4 and 4.0; 8 x 5003 x 4096 8.4 and 9.0, 2 x 6500 x 8192 11.9
    // and 13.2, 1 x 10000 x 8192 17.1 and 18.3, 2 x 4096 x 4096 5.6 and 5.5. One workgroup a CU, and two: 4 x 5003 x 8192
    // 12.3 and 12.9, 8 x 16384 x 2560 10.1 and 9.7
    else if (m * few_pitch(k) <= FEW_LDS_KB << 10 && (k < 4096 ? n >= 8192 && m > 2 : n > 4096))
      i8_few<1, FEW_LDS_KB, false>(a, n <= 8192 ? 1 : 2, y_fp32, s);
    else i8_few<1, 0, false>(a, 0, y_fp32, s);
  } else {
    const I8Tile a{xq, wq, xs, ws, p.splits > 1 ? work : y, m, n, k, p.mblk, p.nblk, p.splits, p.sps};
    // up to 256 tiles a CU holds one workgroup, which may have all of its LDS; beyond, two that take turns at waiting:
    // us, two and one, 128 x 128 tiles of 1500 x 5003 x 2560 (480) 27 and 31, 64 x 64 of 2048 x 2560 x 512 (1280) 11
    // and 17
    const bool one = (int64_t)p.mblk * p.nblk * p.splits <= 256;
    if (p.kind == I8_T256) i8_tiles<256, 1, 2, 4, 5>(a, y_fp32, s);
    else if (p.kind == I8_T128) one ? i8_tiles<128, 1, 2, 4, 8>(a, y_fp32, s) : i8_tiles<128, 1, 2, 2, 4>(a, y_fp32, s);
    else one ? i8_tiles<64, 4, 1, 1, 4>(a, y_fp32, s) : i8_tiles<64, 1, 2, 2, 8>(a, y_fp32, s);
    if (p.splits > 1) {
      const dim3 grid((unsigned)(((int64_t)m * n + 1023) / 1024)), nt(256);
      const int* part = static_cast<const int*>(work);
      if (y_fp32) hipLaunchKernelGGL(k_i8_join<true>, grid, nt, 0, s, part, p.splits, xs, ws, y, m, n);
      else hipLaunchKernelGGL(k_i8_join<false>, grid, nt, 0, s, part, p.splits, xs, ws, y, m, n);
    }
  }
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}

int64_t i8_linear_bytes(int32_t m, int32_t n, int32_t k) {
  if (qf_pays(m, n, k)) return 0;
  return i8_pad((int64_t)m * k) + i8_pad((int64_t)m * 4) + i8_gemm_bytes(m, n, k);
}

int i8_linear(const uint16_t* x, const int8_t* wq, const float* ws, void* y, bool y_fp32, void* work, int32_t m,
              int32_t n, int32_t k, hipStream_t s) {
  if (qf_pays(m, n, k)) {
    // one workgroup a CU, which quantises once for the blocks that it takes in turn, or two, which have more weights in
    // flight: us, 7 x 5003 x 1408 6.5 and 7.5, 8 x 8000 x 2048 8.1 and 9.5, 8 x 12000 x 2560 10.9 and 11.6; 4 x 12000 x 4096
    // 14.1 and 12.3, 4 x 16384 x 2560 12.0 and 11.8, 1 x 49152 x 2560 28.3 and 25.6
    const bool one = n <= 8192 || (n <= 12288 && k < 4096);
    i8_few<1, 36, true>(I8Few{x, nullptr, wq, ws, y, m, n, k}, one ? 1 : 2, y_fp32, s);
    return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
  }
  int8_t* xq = static_cast<int8_t*>(work);
  float* xs = reinterpret_cast<float*>(xq + i8_pad((int64_t)m * k));
  const int rc = i8_quantize(x, xq, xs, m, k, s);
  if (rc != FL_OK) return rc;
  return i8_gemm(xq, xs, wq, ws, y, y_fp32, reinterpret_cast<char*>(xs) + i8_pad((int64_t)m * 4), m, n, k, s);
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
  *bytes = i8_linear_bytes(m, n, k);
  return FL_OK;
}

int fl_linear_int8(const uint16_t* x, const int8_t* wq, const float* ws, void* y, int32_t y_fp32, void* work,
                   int32_t m, int32_t n, int32_t k, void* stream) {
  if (!i8_shape_ok(m, n, k) || !i8_aligned(x) || !i8_aligned(wq) || !ws || !i8_aligned(y) ||
      (i8_linear_bytes(m, n, k) > 0 && !i8_aligned(work)))
    return FL_E_ARG;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return i8_linear(x, wq, ws, y, y_fp32 != 0, work, m, n, k, s);
}

}  // extern "C"
