// Log probabilities of given tokens, with entropy, rank and the top alternatives, of rows of logits;
// and the same from features, through an 8-bit vocabulary head.
//
// Of a row l with maximum m: s = sum e_i, u = sum e_i d_i with d_i = l_i - m, e_i = exp(d_i); then
//   logprob(t) = d_t - log s,   entropy = log s - u / s,   rank(t) = #{i before t},
// where indices are ordered by value, larger first, NaN above all, equal values by rising index (-0 equals
// 0). Everything in fp32. A row without a finite maximum (all -inf, or with a +inf) or with a NaN has no
// distribution: its log probabilities and entropy are NaN, its order is what it is.
//
// One pass over the logits: a workgroup holds a chunk of a row in registers, finds its maximum, then its
// sums, its rank count and its first `top` indices. Rows of several chunks end in a merge launch of one
// workgroup per row.
#include "fl_int8.h"
#include <algorithm>

namespace {

typedef unsigned long long u64;

constexpr int LP_NT = 512, LP_NW = LP_NT / FL_WAVE;
constexpr int LP_TOP = 32;     // alternatives at most
constexpr int LP_CHUNKS = 32;  // of a row at most
constexpr int LP_CAP = 1024;   // candidates kept in LDS
constexpr int LP_MAXV = 1 << 20;
static_assert(LP_CHUNKS * LP_TOP <= LP_CAP, "a merge's candidates always fit");
static_assert(LP_MAXV <= LP_CHUNKS * LP_NT * 64, "every vocabulary fits its chunks");

// Keys that order as the values do, as unsigned numbers (NaN, made positive, above +inf), with the index below
// them: all keys of a row differ, and none is 0.
__device__ __forceinline__ u64 lp_key(float x, int i) {
  const uint32_t b = x != x ? 0x7FC00000u : __float_as_uint(x + 0.0f);  // -0 becomes 0
  const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return ((u64)o << 32) | (0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ float lp_value(u64 key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

struct LpArgs {
  const void* logits;
  int64_t stride;               // of a row, in values
  int vocab, top, chunks, per;  // chunks of a row, values of a chunk (a multiple of 8)
  const int32_t* tokens;        // [rows] or null (then logprob and rank are not written)
  float *logprob, *entropy;     // [rows]
  int32_t* rank;                // [rows]
  int32_t* top_ids;             // [rows, top]
  float* top_lp;                // [rows, top]
  float4* part;                 // chunks > 1: per (row, chunk) maximum, s, u, rank count (its bits) ...
  u64* cand;                    // ... and its first `top` keys, in order, then zeros
};

struct LpShared {
  float red[5][LP_NW];
  int count;
  u64 cand[LP_CAP], first[LP_TOP];
};

// the row's token and its logit; in = false (no token asked for, or an id outside the vocabulary): NaN
struct LpToken {
  int t;
  bool in;
  float l;
};
template <bool BF16>
__device__ __forceinline__ LpToken lp_token(const LpArgs& a, int64_t row) {
  LpToken k{-1, false, __builtin_nanf("")};
  if (a.tokens) k.t = a.tokens[row];
  k.in = k.t >= 0 && k.t < a.vocab;
  if (k.in) {
    const int64_t at = row * a.stride + k.t;
    k.l = BF16 ? bf2f(reinterpret_cast<const uint16_t*>(a.logits)[at]) : reinterpret_cast<const float*>(a.logits)[at];
  }
  return k;
}

// The first a.top of the sh.count (<= LP_CAP) keys in sh.cand, in order, into sh.first: a key's place is the
// number of larger ones.
__device__ __forceinline__ void lp_sort(LpShared& sh, int top) {
  const int tid = threadIdx.x, c = sh.count;
  if (tid < top) sh.first[tid] = 0;
  __syncthreads();
  for (int i = tid; i < c; i += LP_NT) {
    const u64 key = sh.cand[i];
    int at = 0;
    for (int j = 0; j < c; ++j) at += sh.cand[j] > key;
    if (at < top) sh.first[at] = key;
  }
  __syncthreads();
}

// what the whole row says, from its maximum, sums and rank count, and sh.first
__device__ __forceinline__ void lp_write(const LpArgs& a, int64_t row, const LpToken& tok, float m, float s, float u,
                                         int before, const LpShared& sh) {
  const float nan = __builtin_nanf("");
  const bool fine = fabsf(m) < INFINITY;
  const float logs = fine ? logf(s) : nan;  // s is NaN if a value is
  const int tid = threadIdx.x;
  if (tid == 0) {
    if (a.tokens) {
      a.logprob[row] = tok.in ? (tok.l - m) - logs : nan;
      a.rank[row] = tok.in ? before : -1;
    }
    const float h = logs - u / s;
    a.entropy[row] = h < 0.0f ? 0.0f : h;  // rounding
  }
  if (tid < a.top) {
    const u64 key = sh.first[tid];
    a.top_ids[row * a.top + tid] = (int32_t)(0xFFFFFFFFu - (uint32_t)key);
    a.top_lp[row * a.top + tid] = (lp_value(key) - m) - logs;
  }
}

// One chunk of a row per workgroup, E values per thread in registers. VEC: rows are 16-byte aligned.
template <bool BF16, bool VEC, int E>
__global__ __launch_bounds__(LP_NT, E <= 64 ? 4 : 2) void k_logprobs(LpArgs a) {
  constexpr int V = !VEC ? 1 : BF16 ? 8 : 4;  // consecutive values of a load
  __shared__ LpShared sh;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int64_t row = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x % a.chunks);
  const int j0 = chunk * a.per, j1 = min(a.vocab, j0 + a.per), len = j1 - j0;
  const LpToken tok = lp_token<BF16>(a, row);
  const float* lf = reinterpret_cast<const float*>(a.logits) + row * a.stride;
  const uint16_t* lh = reinterpret_cast<const uint16_t*>(a.logits) + row * a.stride;
  auto index = [&](int e) { return j0 + ((e / V) * LP_NT + tid) * V + e % V; };
  float x[E];
#pragma unroll
  for (int i = 0; i < E / V; ++i) {
    const int j = index(i * V);
    if (V > 1 && j + V <= j1) {
      if constexpr (BF16) {
        const uint4 w = *reinterpret_cast<const uint4*>(lh + j);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < V; ++k) x[i * V + k] = k & 1 ? bfhi(ww[(k / 2) & 3]) : bflo(ww[(k / 2) & 3]);
      } else {
        const float4 w = *reinterpret_cast<const float4*>(lf + j);
        const float ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < V; ++k) x[i * V + k] = ww[k & 3];
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) x[i * V + k] = j + k < j1 ? (BF16 ? bf2f(lh[j + k]) : lf[j + k]) : -INFINITY;
    }
  }
  float mine = -INFINITY;  // NaN is passed over here; it comes back through s
#pragma unroll
  for (int e = 0; e < E; ++e) mine = fmaxf(mine, x[e]);
  // A value that at least `top` of the chunk reach: of each of the waves whose lanes all hold values, the q-th
  // largest of its lanes' maxima; the smallest of these. Few others reach it.
  const int full = min(LP_NW, len / (FL_WAVE * V)), q = full > 0 ? (a.top + full - 1) / full : 0;
  float left = mine, wm = -INFINITY, wq = -INFINITY;
  for (int i = 0; i < max(q, 1); ++i) {
    wq = wave_max(left);
    if (i == 0) wm = wq;
    const int first = __builtin_ctzll(__ballot(left == wq) | (1ull << 63));
    if ((tid & 63) == first) left = -INFINITY;
  }
  if ((tid & 63) == 0) sh.red[0][wave] = wm, sh.red[1][wave] = wq;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  float m = -INFINITY, T = full > 0 ? INFINITY : -INFINITY;
#pragma unroll
  for (int w = 0; w < LP_NW; ++w) {
    m = fmaxf(m, sh.red[0][w]);
    if (w < full) T = fminf(T, sh.red[1][w]);
  }
  // sums and rank count; values past the chunk are -inf and add nothing
  const float mu = m == -INFINITY ? 0.0f : m;
  float s = 0.0f, u = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float d = x[e] - mu;
    d = d < -1000.0f ? -1000.0f : d;  // e = 0, and 0 * d = 0 for masked values; NaN stays
    const float p = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
    s += p;
    u += p * d;
  }
  const bool odd = s != s;  // this thread holds a NaN, or the +inf that is the maximum
  int before = 0;
  if (tok.in) {
    const int tm = min(tok.t, j1);
    if (tok.l == tok.l) {
#pragma unroll
      for (int e = 0; e < E; ++e) before += !(x[e] <= tok.l) || (x[e] == tok.l && index(e) < tm);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) before += x[e] != x[e] && index(e) < tm;
    }
  }
  if (a.top > 0 && (odd || mine >= T)) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = index(e);
      // over -inf alone: its first values by index besides whatever is larger
      const bool is = T == -INFINITY ? !(x[e] <= T) || j < j0 + a.top : !(x[e] < T);
      if (is && j < j1) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < LP_CAP) sh.cand[at] = lp_key(x[e], j);
      }
    }
  }
  s = wave_sum(s);
  u = wave_sum(u);
  const float bf = wave_sum((float)before);  // at most 64 x 96: exact
  if ((tid & 63) == 0) sh.red[2][wave] = s, sh.red[3][wave] = u, sh.red[4][wave] = bf;
  __syncthreads();
  s = u = 0.0f, before = 0;
#pragma unroll
  for (int w = 0; w < LP_NW; ++w) s += sh.red[2][w], u += sh.red[3][w], before += (int)sh.red[4][w];
  if (a.top > 0) {
    if (sh.count <= LP_CAP) {
      lp_sort(sh, a.top);
    } else {  // a crowd of equal values: one after the other, from memory
      u64 last = ~0ull;
      for (int r = 0; r < a.top; ++r) {
        u64 best = 0;
        for (int j = j0 + tid; j < j1; j += LP_NT) {
          const u64 k = lp_key(BF16 ? bf2f(lh[j]) : lf[j], j);
          if (k < last) best = u64max(best, k);
        }
        best = wave_max_u64(best);
        __syncthreads();
        if ((tid & 63) == 0) sh.cand[wave] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < LP_NW; ++w) best = u64max(best, sh.cand[w]);
        if (tid == 0) sh.first[r] = best;
        last = best;
      }
      __syncthreads();
    }
  }
  if (a.chunks == 1) {
    lp_write(a, row, tok, m, s, u, before, sh);
    return;
  }
  const int64_t at = row * a.chunks + chunk;
  if (tid == 0) a.part[at] = make_float4(m, s, u, __int_as_float(before));
  if (tid < a.top) a.cand[at * a.top + tid] = sh.first[tid];
}

// The chunks of a row in order: one workgroup per row
template <bool BF16>
__global__ __launch_bounds__(LP_NT) void k_logprobs_merge(LpArgs a) {
  __shared__ LpShared sh;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const LpToken tok = lp_token<BF16>(a, row);
  const float4* part = a.part + row * a.chunks;
  float m = -INFINITY, s = 0.0f, u = 0.0f;
  int before = 0;
  for (int c = 0; c < a.chunks; ++c) m = fmaxf(m, part[c].x);
  for (int c = 0; c < a.chunks; ++c) {
    const float4 p = part[c];
    before += __float_as_int(p.w);
    if (p.y == 0.0f) continue;  // nothing but -inf
    // a NaN (or +inf) chunk has s = NaN, whatever its maximum
    const float d = fmaxf(p.x - m, -1000.0f), e = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
    s += p.y * e;
    u += (p.z + p.y * d) * e;
  }
  if (a.top > 0) {
    const u64* cand = a.cand + row * a.chunks * a.top;
    if (tid == 0) sh.count = 0;
    // at least `top` keys reach the largest of the chunks' last ones
    u64 T = 0;
    for (int c = 0; c < a.chunks; ++c) T = u64max(T, cand[(c + 1) * a.top - 1]);
    __syncthreads();
    for (int i = tid; i < a.chunks * a.top; i += LP_NT) {
      const u64 k = cand[i];
      if (k >= T && k != 0) sh.cand[atomicAdd(&sh.count, 1)] = k;
    }
    __syncthreads();
    lp_sort(sh, a.top);
  }
  lp_write(a, row, tok, m, s, u, before, sh);
}

// Chunks of a row: one, or as many as give `want` workgroups in all, of 4096 values at least.
void lp_plan(LpArgs& a, int rows) {
  const int most = std::min(LP_CHUNKS, std::max(1, a.vocab / 4096)), least = (a.vocab + LP_NT * 96 - 1) / (LP_NT * 96);
  a.chunks = std::max(least, std::min(most, std::max(1, 512 / rows)));
  a.per = ((a.vocab + a.chunks - 1) / a.chunks + 7) / 8 * 8;
  a.chunks = (a.vocab + a.per - 1) / a.per;
}

template <bool BF16, bool VEC>
void lp_launch(const LpArgs& a, int rows, hipStream_t s) {
  const dim3 grid((unsigned)rows * (unsigned)a.chunks);
  const int e = (a.per + LP_NT - 1) / LP_NT;
  if (e <= 8) hipLaunchKernelGGL((k_logprobs<BF16, VEC, 8>), grid, dim3(LP_NT), 0, s, a);
  else if (e <= 16) hipLaunchKernelGGL((k_logprobs<BF16, VEC, 16>), grid, dim3(LP_NT), 0, s, a);
  else if (e <= 32) hipLaunchKernelGGL((k_logprobs<BF16, VEC, 32>), grid, dim3(LP_NT), 0, s, a);
  else if (e <= 64) hipLaunchKernelGGL((k_logprobs<BF16, VEC, 64>), grid, dim3(LP_NT), 0, s, a);
  else hipLaunchKernelGGL((k_logprobs<BF16, VEC, 96>), grid, dim3(LP_NT), 0, s, a);
  if (a.chunks > 1) hipLaunchKernelGGL(k_logprobs_merge<BF16>, dim3(rows), dim3(LP_NT), 0, s, a);
}

int64_t lp_part_bytes(const LpArgs& a, int rows) { return a.chunks > 1 ? i8_pad((int64_t)rows * a.chunks * 16) : 0; }
int64_t lp_bytes(const LpArgs& a, int rows) {
  return a.chunks > 1 ? lp_part_bytes(a, rows) + i8_pad((int64_t)rows * a.chunks * a.top * 8) : 0;
}

constexpr int LP_MAXROWS = 1 << 17;  // rows x LP_CHUNKS workgroups of 512 threads in one grid

bool lp_shape_ok(int rows, int vocab, int top) {
  return rows >= 1 && rows <= LP_MAXROWS && vocab >= 1 && vocab <= LP_MAXV && top >= 0 && top <= LP_TOP && top <= vocab;
}
bool lp_outputs_ok(const int32_t* tokens, int top, const float* logprob, const float* entropy, const int32_t* rank,
                   const int32_t* top_ids, const float* top_lp) {
  return entropy && (!tokens || (logprob && rank)) && (top == 0 || (top_ids && top_lp));
}

int lp_run(LpArgs a, bool bf16, int rows, void* work, hipStream_t s) {
  lp_plan(a, rows);
  a.part = static_cast<float4*>(work);
  a.cand = reinterpret_cast<u64*>(static_cast<char*>(work) + lp_part_bytes(a, rows));
  const int esize = bf16 ? 2 : 4;
  const bool vec = i8_aligned(a.logits) && (a.stride * esize) % 16 == 0;
  if (bf16 && vec) lp_launch<true, true>(a, rows, s);
  else if (bf16) lp_launch<true, false>(a, rows, s);
  else if (vec) lp_launch<false, true>(a, rows, s);
  else lp_launch<false, false>(a, rows, s);
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}

// Features -> log probabilities: the rows of x in 8 bits, then blocks of rows through the head, whose fp32
// logits stay in the workspace (up to 128 MB of them, half of what the last-level cache holds).
struct HeadPlan {
  int rows;  // of a block
  int64_t xq, xs, logits, gemm, lp, bytes;
};
HeadPlan head_plan(int m, int n, int k, int top) {
  HeadPlan p{};
  const int64_t fit = std::max<int64_t>(1, (128ll << 20) / ((int64_t)n * 4));
  p.rows = (int)std::min<int64_t>(m, fit >= 256 ? fit / 256 * 256 : fit);
  LpArgs a{};
  a.vocab = n;
  a.top = top;
  int64_t lp = 0;
  for (const int r : {p.rows, m % p.rows}) {
    if (r == 0) continue;
    lp_plan(a, r);
    lp = std::max(lp, lp_bytes(a, r));
    p.gemm = std::max(p.gemm, i8_gemm_bytes(r, n, k));
  }
  const int64_t gemm = p.gemm;
  p.xq = 0;
  p.xs = i8_pad((int64_t)m * k);
  p.logits = p.xs + i8_pad((int64_t)m * 4);
  p.gemm = p.logits + i8_pad((int64_t)p.rows * n * 4);
  p.lp = p.gemm + i8_pad(gemm);
  p.bytes = p.lp + lp;
  return p;
}

}  // namespace

extern "C" {

int fl_logprobs_workspace(int32_t rows, int32_t vocab, int32_t top, int64_t* bytes) {
  if (!bytes || !lp_shape_ok(rows, vocab, top)) return FL_E_ARG;
  LpArgs a{};
  a.vocab = vocab;
  a.top = top;
  lp_plan(a, rows);
  *bytes = lp_bytes(a, rows);
  return FL_OK;
}

int fl_logprobs(const void* logits, int32_t bf16, int64_t stride, int32_t rows, int32_t vocab, const int32_t* tokens,
                int32_t top, float* logprob, float* entropy, int32_t* rank, int32_t* top_ids, float* top_logprobs,
                void* work, void* stream) {
  if (!logits || !lp_shape_ok(rows, vocab, top) || (rows > 1 && stride < vocab) ||
      !lp_outputs_ok(tokens, top, logprob, entropy, rank, top_ids, top_logprobs))
    return FL_E_ARG;
  LpArgs a{logits, rows > 1 ? stride : 0, vocab, top, 0, 0, tokens, logprob, entropy, rank, top_ids, top_logprobs,
           nullptr, nullptr};
  lp_plan(a, rows);
  if (lp_bytes(a, rows) > 0 && !i8_aligned(work)) return FL_E_ARG;
  return lp_run(a, bf16 != 0, rows, work, reinterpret_cast<hipStream_t>(stream));
}

int fl_head_logprobs_workspace(int32_t m, int32_t n, int32_t k, int32_t top, int64_t* bytes) {
  if (!bytes || !i8_shape_ok(m, n, k) || !lp_shape_ok(m, n, top)) return FL_E_ARG;
  *bytes = head_plan(m, n, k, top).bytes;
  return FL_OK;
}

int fl_head_logprobs(const uint16_t* x, const int8_t* wq, const float* ws, const int32_t* tokens, int32_t top,
                     float* logprob, float* entropy, int32_t* rank, int32_t* top_ids, float* top_logprobs, void* work,
                     int32_t m, int32_t n, int32_t k, void* stream) {
  if (!i8_shape_ok(m, n, k) || !lp_shape_ok(m, n, top) || !i8_aligned(x) || !i8_aligned(wq) || !ws ||
      !i8_aligned(work) || !lp_outputs_ok(tokens, top, logprob, entropy, rank, top_ids, top_logprobs))
    return FL_E_ARG;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const HeadPlan p = head_plan(m, n, k, top);
  char* base = static_cast<char*>(work);
  int8_t* xq = reinterpret_cast<int8_t*>(base + p.xq);
  float* xs = reinterpret_cast<float*>(base + p.xs);
  int rc = i8_quantize(x, xq, xs, m, k, s);
  for (int r0 = 0; r0 < m && rc == FL_OK; r0 += p.rows) {
    const int r = std::min(p.rows, m - r0);
    rc = i8_gemm(xq + (int64_t)r0 * k, xs + r0, wq, ws, base + p.logits, true, base + p.gemm, r, n, k, s);
    if (rc != FL_OK) break;
    const int64_t t0 = (int64_t)r0 * top;
    LpArgs a{base + p.logits, n, n, top, 0, 0, tokens ? tokens + r0 : nullptr, tokens ? logprob + r0 : nullptr,
             entropy + r0, tokens ? rank + r0 : nullptr, top ? top_ids + t0 : nullptr, top ? top_logprobs + t0 : nullptr,
             nullptr, nullptr};
    rc = lp_run(a, false, r, base + p.lp, s);
  }
  return rc;
}

}  // extern "C"
