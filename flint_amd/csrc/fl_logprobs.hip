// Log probabilities of given tokens, with entropy, rank and the top alternatives, of rows of logits;
// and the same from features, through an 8-bit vocabulary head.
//
// Of a row l with maximum m: s = sum e_i, u = sum e_i d_i with d_i = l_i - m, e_i = exp(d_i); then
//   logprob(t) = d_t - log s,   entropy = log s - u / s,   rank(t) = #{i before t},
// where indices are ordered by value, larger first, NaN above all, equal values by rising index (-0 equals
// 0). Everything in fp32. A row without a finite maximum (all -inf, or with a +inf) or with a NaN has no
// distribution: its log probabilities and entropy are NaN, its order is what it is.
//
// One pass over the logits: a workgroup streams a row, or a chunk of one, through registers; every thread keeps the
// running maximum and sums of its values. Rows of several chunks end in a merge launch of one workgroup per row.
#include "fl_int8.h"
#include <algorithm>
#include <type_traits>

namespace {

typedef unsigned long long u64;

constexpr float LP_LOG2E = 1.4426950408889634f;
constexpr int LP_NT = 256, LP_NW = LP_NT / FL_WAVE;
constexpr int LP_E = 16;                // values of a thread in a step
constexpr int LP_STEP = LP_NT * LP_E;   // of a workgroup
constexpr int LP_TOP = 32;     // alternatives at most
constexpr int LP_CHUNKS = 32;  // of a row at most
constexpr int LP_KEEP = 256;   // candidates that a wave keeps in LDS
constexpr int LP_MAXV = 1 << 20;
static_assert(LP_CHUNKS * LP_TOP <= LP_NW * LP_KEEP, "a merge's candidates always fit");

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

// 16 bytes of a row, which starts where its type may
typedef uint32_t lp_raw_f32 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t lp_raw_bf16 __attribute__((ext_vector_type(4), aligned(2)));

struct LpArgs {
  const void* logits;
  int64_t stride;               // of a row, in values
  int vocab, top, chunks, per;  // chunks of a row, values of a chunk (a multiple of 8)
  const int32_t* tokens;        // [rows] or null (then logprob and rank are not written)
  float *logprob, *entropy;     // [rows]
  int32_t* rank;                // [rows]
  int32_t* top_ids;             // [rows, top]
  float* top_lp;                // [rows, top]
  // chunks > 1: per (row, chunk) maximum, s, u, rank count (its bits) and the first `top` keys, in order, then zeros;
  // per row the token's logit and whether there is one
  float4* part;
  u64* cand;
  float2* given;
};

struct LpShared {
  uint32_t bound[LP_NW];
  float4 red[LP_NW];  // maximum, s, u, rank count of each wave
  int kept[LP_NW];    // candidates of each wave
  int place[LP_NW][FL_WAVE];
  u64 cand[LP_NW][LP_KEEP];  // their keys, zeros up to the next multiple of eight
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

// The first `top` of the waves' candidates (sh.kept of them each, <= LP_KEEP; a barrier lies behind them), in order:
// out(place, key) in wave 0, key 0 past the last. A key's place is the number of larger ones: lanes take candidates,
// each wave counts over its own.
template <class F>
__device__ __forceinline__ void lp_sort(LpShared& sh, int top, F out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int n[LP_NW], c = 0;
#pragma unroll
  for (int w = 0; w < LP_NW; ++w) c += n[w] = sh.kept[w];
  const int own = sh.kept[wave];
  if (wave == 0 && lane >= c && lane < top) out(lane, (u64)0);
  for (int b = 0; b < c; b += FL_WAVE) {
    int i = b + lane, w = 0;
#pragma unroll
    for (int v = 0; v < LP_NW - 1; ++v)
      if (w == v && i >= n[v]) i -= n[v], ++w;
    const u64 key = b + lane < c ? sh.cand[w][i] : 0;
    int larger = 0;
    for (int j = 0; j < own; j += 8)  // zeros behind the last
#pragma unroll
      for (int i = 0; i < 8; ++i) larger += sh.cand[wave][j + i] > key;
    sh.place[wave][lane] = larger;
    __syncthreads();
    if (wave == 0 && key != 0) {
      int at = 0;
#pragma unroll
      for (int v = 0; v < LP_NW; ++v) at += sh.place[v][lane];
      if (at < top) out(at, key);
    }
    if (b + FL_WAVE < c) __syncthreads();
  }
}

// A value that q of G groups of N lanes reach (of the wave's first lanes), close to the q-th largest of theirs: v orders
// as unsigned, agrees in a group and is 0 in the lanes behind. The last bits tell equal groups apart and are dropped from
// the answer. Every group counts the larger ones: 16 groups 300 cycles, against 190 for each of q rounds of maxima; whole
// 64-bit keys in a loop over the chunks there are: 0.7 us more than 32 chunks in 32 bits.
template <int G, int N>
__device__ __forceinline__ uint32_t lp_reached(uint32_t v, int q) {
  v = (v & ~(uint32_t)(G - 1)) | (uint32_t)((threadIdx.x & 63) / N % G);
  int larger = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) larger += (uint32_t)__builtin_amdgcn_readlane((int)v, g * N) > v;
  const u64 at = __ballot(larger == q - 1);  // q = 0: nowhere, any value will do
  return (uint32_t)__builtin_amdgcn_readlane((int)v, __builtin_ctzll(at | (1ull << 63))) & ~(uint32_t)(G - 1);
}
template <int CTRL>
__device__ __forceinline__ uint32_t umax_dpp(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_umax32(uint32_t v) {
  v = umax_dpp<0x4E>(umax_dpp<0xB1>(v));  // of 4 lanes
  v = umax_dpp<0x140>(umax_dpp<0x141>(v));  // of 16
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(r[0], r[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(q[0], q[1]);
}
// Of values with a lane each, one that q of the wave's lanes reach, stored for the other waves to read at any time
// (rising values only make it rise): close to the q-th largest where it is asked for once, the chunk being one step; else
// the q-th largest, in q rounds, as a higher bound spares candidates in all the steps that follow (1024 rows of 49152,
// top 32: 49 us, 55 without).
__device__ __forceinline__ void lp_publish(uint32_t* bound, float mine, int q, bool once) {
  const uint32_t b = __float_as_uint(mine + 0.0f);  // -0 becomes 0
  uint32_t v = mine == mine ? b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u) : 0u, t = 0;
  if (once && q <= 16) t = lp_reached<16, 4>(umax_dpp<0x4E>(umax_dpp<0xB1>(v)), q);
  else
    for (int r = 0; r < q; ++r) {
      t = wave_umax32(v);
      if ((threadIdx.x & 63) == __builtin_ctzll(__ballot(v == t) | (1ull << 63))) v = 0;
    }
  if ((threadIdx.x & 63) == 0)
    __hip_atomic_store(bound + (threadIdx.x >> 6), t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}
// the smallest of the first waves' bounds: a value that LP_NW q reach
__device__ __forceinline__ float lp_least(uint32_t* bound, int waves) {
  uint32_t t = waves > 0 ? ~0u : 0u;
#pragma unroll
  for (int k = 0; k < LP_NW; ++k)
    if (k < waves) t = min(t, __hip_atomic_load(bound + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
  return t <= 0x007FFFFFu ? -INFINITY : lp_value((u64)t << 32);  // -inf's ordered bits
}

// what the whole row says, from its maximum, sums and rank count: by wave 1, beside wave 0's sort
__device__ __forceinline__ float lp_logsum(float m, float s) {  // NaN without a distribution; s is NaN if a value is
  return fabsf(m) < INFINITY ? logf(s) : __builtin_nanf("");
}
__device__ __forceinline__ void lp_write(const LpArgs& a, int64_t row, const LpToken& tok, float m, float logs, float s,
                                         float u, int before) {
  if (threadIdx.x != FL_WAVE) return;
  if (a.tokens) {
    a.logprob[row] = tok.in ? (tok.l - m) - logs : __builtin_nanf("");
    a.rank[row] = tok.in ? before : -1;
  }
  const float h = logs - u / s;
  a.entropy[row] = h < 0.0f ? 0.0f : h;  // rounding
}
__device__ __forceinline__ void lp_place(const LpArgs& a, int64_t row, float m, float logs, int place, u64 key) {
  a.top_ids[row * a.top + place] = (int32_t)(0xFFFFFFFFu - (uint32_t)key);
  a.top_lp[row * a.top + place] = (lp_value(key) - m) - logs;
}

// v_max3_f32 without the operation per operand that makes a loaded value canonical
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// how many of these lanes are below this one
__device__ __forceinline__ int lp_below(u64 lanes) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
}
// how many lanes of the wave
__device__ __forceinline__ int lp_count(bool is) { return __builtin_popcountll(__ballot(is)); }

// (maximum, s, u) of a wave's lanes joined, in every lane
__device__ __forceinline__ void lp_join(float& m, float& s, float& u) {
  const float mm = wave_max(m), mu = mm == -INFINITY ? 0.0f : mm;
  const float d = fmaxf(m - mu, -1000.0f), e = __builtin_amdgcn_exp2f(d * LP_LOG2E);  // nothing seen: s = u = 0
  u = wave_sum((u + s * d) * e);
  s = wave_sum(s * e);
  m = mm;
}

// One chunk of a row per workgroup, in steps of LP_E values per thread; the next step's loads are in flight meanwhile.
// 1024 rows of 49152 (fp32, top 5) 37 us, 5.4 TB/s with part of them in the last-level cache, the vector ALUs busy in more
// than half of the cycles (16 instructions a value; bf16, 32 us, is bound by these); 34 without alternatives, two steps in
// flight no faster. One row of 49152, top 20, twelve chunks, 5.5 us and 3.0 to merge them (5.8 in all without
// alternatives): a launch and a memory latency each, then one dependent step after another.
template <bool BF16>
__global__ __launch_bounds__(LP_NT, 4) void k_logprobs(LpArgs a) {
  constexpr int V = BF16 ? 8 : 4;  // consecutive values of a load (16 bytes, aligned to the type only)
  using raw4 = std::conditional_t<BF16, lp_raw_bf16, lp_raw_f32>;
  __shared__ LpShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x % a.chunks);
  const int j0 = chunk * a.per, j1 = min(a.vocab, j0 + a.per);
  const float* lf = reinterpret_cast<const float*>(a.logits) + row * a.stride;
  const uint16_t* lh = reinterpret_cast<const uint16_t*>(a.logits) + row * a.stride;
  constexpr uint32_t NINF = BF16 ? 0xFF80FF80u : 0xFF800000u;
  // kept as loaded until used: anything done to a value here would wait for it
  auto load = [&](int jb, raw4 (&x)[LP_E / V]) {
#pragma unroll
    for (int i = 0; i < LP_E / V; ++i) {
      const int j = jb + (i * LP_NT + tid) * V;
      x[i] = raw4{NINF, NINF, NINF, NINF};
      if (jb + (i + 1) * LP_NT * V <= j1 || j + V <= j1)
        x[i] = *reinterpret_cast<const raw4*>(BF16 ? (const void*)(lh + j) : (const void*)(lf + j));
      else if (j < j1) {  // the one lane where the row ends inside 16 bytes
        uint32_t v[V];
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = BF16 ? lh[min(j + k, j1 - 1)] : __float_as_uint(lf[min(j + k, j1 - 1)]);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = j + k < j1 ? v[k] : NINF & (BF16 ? 0xFFFFu : ~0u);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[i][k] = BF16 ? v[(2 * k) % V] | v[(2 * k + 1) % V] << 16 : v[k % V];
      }
    }
  };
  raw4 cur[LP_E / V];
  load(j0, cur);
  const LpToken tok = lp_token<BF16>(a, row);
  // Candidates for the first `top` places: of each of the waves whose lanes all hold values, the q-th largest of
  // its lanes' maxima so far; at least `top` values of the chunk reach the smallest of these, T, and few others do. T
  // only rises, so what is collected with an earlier T is too much at worst.
  const int full = min(LP_NW, (j1 - j0) / (FL_WAVE * V)), q = full > 0 ? (a.top + full - 1) / full : 0;
  float m = -INFINITY, s = 0.0f, u = 0.0f, T = -INFINITY;
  int before = 0, kept = 0, i = 0;  // `before` and kept: of the wave
  bool masked = false;              // whether the wave has met a -inf: without one its sums spare an operation a value
  for (int jb = j0; jb < j1; jb += LP_STEP, ++i) {
    raw4 ahead[LP_E / V];
    if (jb + LP_STEP < j1) load(jb + LP_STEP, ahead);
    float x[LP_E];
#pragma unroll
    for (int e = 0; e < LP_E; ++e) {
      const uint32_t w = cur[e / V][(BF16 ? e / 2 : e) & 3];
      x[e] = !BF16 ? __uint_as_float(w) : e & 1 ? bfhi(w) : bflo(w);
    }
    // NaN is passed over; it comes back through s
    float top = max3(max3(max3(x[0], x[1], x[2]), x[3], x[4]), x[5], x[6]);
    top = max3(max3(max3(max3(top, x[7], x[8]), x[9], x[10]), x[11], x[12]), x[13], x[14]);
    top = max3(top, x[15], x[15]);
    const float old = m;
    m = fmaxf(m, top);
    // sums over the maximum so far; values past the chunk are -inf and add nothing
    const float mu = m == -INFINITY ? 0.0f : m;
    const float d0 = fmaxf(old - mu, -1000.0f), e0 = __builtin_amdgcn_exp2f(d0 * LP_LOG2E);
    u = (u + s * d0) * e0;
    s *= e0;
    auto sums = [&](float& s, float& u, auto low) {
#pragma unroll
      for (int e = 0; e < LP_E; ++e) {
        const float d = x[e] - mu, p = __builtin_amdgcn_exp2f(d * LP_LOG2E);
        s += p;
        u = __builtin_fmaf(p, low(d), u);
      }
    };
    float s1 = s, u1 = u;
    masked = masked || jb + LP_STEP > j1;
    if (!masked) {
      sums(s1, u1, [](float d) { return d; });
      masked = __ballot(u1 != u1) != 0;  // 0 times -inf
    }
    if (masked) s1 = s, u1 = u, sums(s1, u1, [](float d) { return fmaxf(d, -1000.0f); });  // 0 times -1000
    s = s1, u = u1;
    const int jt = jb + tid * V;  // e's index: jt + (e / V) * LP_NT * V + e % V
    if (a.top > 0) {
      if ((i & (i + 1)) == 0) {  // steps 0, 1, 3, 7, ...
        lp_publish(sh.bound, m, q, j1 - j0 <= LP_STEP);
        if (i == 0) __syncthreads();
        T = lp_least(sh.bound, full);
      }
      const float least = fmaxf(T, -3.4028235e38f);
      if (i == 0) {
        // The first step has most of them, in any of a lane's values: a candidate of every lane that has one at a time
        // (16 ballots in a row take twice as long).
        uint32_t mask = 0;  // value e: bit 15 - e
#pragma unroll
        for (int e = 0; e < LP_E; ++e) mask = mask << 1 | (uint32_t)!(x[e] < least);
        for (u64 lanes; (lanes = __ballot(mask != 0)) != 0; mask &= mask - 1) {
          const int b = __builtin_ctz(mask | 1u << LP_E), e = LP_E - 1 - b;
          float half[LP_E];
#pragma unroll
          for (int i = 0; i < LP_E; ++i) half[i] = x[LP_E - 1 - i];
#pragma unroll
          for (int w = LP_E / 2, bit = 1; w > 0; w /= 2, bit *= 2)
#pragma unroll
            for (int i = 0; i < w; ++i) half[i] = b & bit ? half[2 * i + 1] : half[2 * i];
          const int at = kept + lp_below(lanes);
          if (mask != 0 && at < LP_KEEP) sh.cand[wave][at] = lp_key(half[0], jt + e / V * (LP_NT * V) + e % V);
          kept += __builtin_popcountll(lanes);
        }
        if (T == -INFINITY && wave == 0) {
          // all that is larger may be too little: the values of -inf among the chunk's first `top`, which come next
          const int j = j0 + lane;
          float v = 0.0f;
          if (lane < a.top && j < j1) v = BF16 ? bf2f(lh[j]) : lf[j];
          const u64 lanes = __ballot(v == -INFINITY);
          const int at = kept + lp_below(lanes);
          if (v == -INFINITY && at < LP_KEEP) sh.cand[wave][at] = lp_key(v, j);
          kept += __builtin_popcountll(lanes);
        }
      } else if (__ballot(s != s || top >= least) != 0) {
#pragma unroll
        for (int e = 0; e < LP_E; ++e) {
          const u64 lanes = __ballot(!(x[e] < least));
          if (lanes == 0) continue;
          const int at = kept + lp_below(lanes);
          if (!(x[e] < least) && at < LP_KEEP) sh.cand[wave][at] = lp_key(x[e], jt + (e / V) * LP_NT * V + e % V);
          kept += __builtin_popcountll(lanes);
        }
      }
    }
    // last: the token's logit comes from two loads in a row; mostly a likely token's, which few steps have anything above
    if (tok.in && (tok.l != tok.l || __ballot(s != s || !(top < tok.l)) != 0)) {
      if (tok.l != tok.l || (tok.t >= jb && tok.t < jb + LP_STEP) || (tok.l == -INFINITY && jb + LP_STEP > j1)) {
        const int tm = min(tok.t, j1) - jt;
#pragma unroll
        for (int e = 0; e < LP_E; ++e) {
          const bool lower = (e / V) * LP_NT * V + e % V < tm;
          before += lp_count(tok.l == tok.l ? !(x[e] <= tok.l) || (x[e] == tok.l && lower) : x[e] != x[e] && lower);
        }
      } else if (tok.t < jb) {  // all of the step is behind the token: what is larger comes before it
#pragma unroll
        for (int e = 0; e < LP_E; ++e) before += lp_count(!(x[e] <= tok.l));
      } else {  // a whole step before it: equal values, too
#pragma unroll
        for (int e = 0; e < LP_E; ++e) before += lp_count(!(x[e] < tok.l));
      }
    }
#pragma unroll
    for (int v = 0; v < LP_E / V; ++v) cur[v] = ahead[v];
  }
  lp_join(m, s, u);
  if (lane == 0) sh.red[wave] = make_float4(m, s, u, __int_as_float(before)), sh.kept[wave] = kept;
  if (lane < 8 && (kept & 7) + lane < 8 && kept + lane < LP_KEEP) sh.cand[wave][kept + lane] = 0;
  __syncthreads();
  int most = 0;
  before = 0;
  {
    float4 w[LP_NW];
#pragma unroll
    for (int k = 0; k < LP_NW; ++k) {
      w[k] = sh.red[k];
      m = fmaxf(m, w[k].x);
      before += __float_as_int(w[k].w);
      most = max(most, sh.kept[k]);
    }
    const float mu = m == -INFINITY ? 0.0f : m;
    s = u = 0.0f;
#pragma unroll
    for (int k = 0; k < LP_NW; ++k) {
      const float d = fmaxf(w[k].x - mu, -1000.0f), e = __builtin_amdgcn_exp2f(d * LP_LOG2E);
      s += w[k].y * e;
      u += (w[k].z + w[k].y * d) * e;
    }
  }
  const float logs = a.chunks == 1 ? lp_logsum(m, s) : 0.0f;
  const int64_t at = row * a.chunks + chunk;
  auto out = [&](int place, u64 key) {
    if (a.chunks == 1) lp_place(a, row, m, logs, place, key);
    else a.cand[at * a.top + place] = key;
  };
  if (a.chunks == 1) lp_write(a, row, tok, m, logs, s, u, before);
  else if (tid == FL_WAVE) {
    a.part[at] = make_float4(m, s, u, __int_as_float(before));
    if (chunk == 0) a.given[row] = make_float2(tok.l, tok.in ? 1.0f : 0.0f);
  }
  if (a.top == 0) return;
  if (most <= LP_KEEP) {
    lp_sort(sh, a.top, out);
    return;
  }
  // Too many candidates: one after the other, from memory. Crowds of equal values come here, so do masks of the type's lowest
  // value that leave a chunk fewer tokens than its bound asks for, and masks of -inf that leave a range of ids in a chunk
  // whose first steps hold nothing, as there is no bound yet when it begins. 31 / 1024 rows of 49152 with five tokens left
  // by the lowest value, top 8, 35 / 586 us, against 11 / 37 by -inf; a range by either, 1024 rows, 376, top 32 2217.
  u64 last = ~0ull;
  for (int r = 0; r < a.top; ++r) {
    u64 best = 0;
    for (int j = j0 + tid; j < j1; j += LP_NT) {
      const u64 k = lp_key(BF16 ? bf2f(lh[j]) : lf[j], j);
      if (k < last) best = u64max(best, k);
    }
    best = wave_max_u64(best);
    __syncthreads();
    if (lane == 0) sh.cand[0][wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < LP_NW; ++w) best = u64max(best, sh.cand[0][w]);
    if (tid == 0) out(r, best);
    last = best;
  }
}

// The chunks of a row joined: one workgroup per row, lane = chunk
__global__ __launch_bounds__(LP_NT) void k_logprobs_merge(LpArgs a) {
  constexpr int E = LP_CHUNKS * LP_TOP / LP_NT;  // keys of a thread
  __shared__ LpShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, keys = a.chunks * a.top;
  const int64_t row = blockIdx.x;
  const u64* cand = a.cand + row * keys;
  const float4 p = lane < a.chunks ? a.part[row * a.chunks + lane] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
  if (a.top > 0) {
    u64 mine[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {  // neighbours to different waves: a chunk's first keys are the larger ones
      const int k = i * LP_NT + lane * LP_NW + wave;
      mine[i] = k < keys ? cand[k] : 0;
    }
    // At least `top` keys reach what q chunks' keys at place `at` do, with at so that q is about half of the chunks.
    const int at = min((2 * a.top + a.chunks - 1) / a.chunks, a.top) - 1, q = (a.top + at) / (at + 1);
    const uint32_t t = lp_reached<LP_CHUNKS, 1>(lane < a.chunks ? (uint32_t)(cand[lane * a.top + at] >> 32) : 0u, q);
    int kept = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const bool is = mine[i] != 0 && (uint32_t)(mine[i] >> 32) >= t;
      const u64 lanes = __ballot(is);
      const int at = kept + lp_below(lanes);
      if (is) sh.cand[wave][at] = mine[i];
      kept += __builtin_popcountll(lanes);
    }
    if (lane == 0) sh.kept[wave] = kept;
    if (lane < 8 && (kept & 7) + lane < 8 && kept + lane < LP_KEEP) sh.cand[wave][kept + lane] = 0;
  }
  LpToken tok{-1, false, 0.0f};
  if (a.tokens) {
    const float2 g = a.given[row];
    tok.l = g.x, tok.in = g.y != 0.0f;
  }
  float m = p.x, s = p.y, u = p.z;
  lp_join(m, s, u);
  const float logs = lp_logsum(m, s);
  lp_write(a, row, tok, m, logs, s, u, (int)wave_sum((float)__float_as_int(p.w)));  // below 2^24: exact
  if (a.top == 0) return;
  __syncthreads();
  lp_sort(sh, a.top, [&](int place, u64 key) { lp_place(a, row, m, logs, place, key); });
}

// Chunks of a row: one, or as many as give 1024 workgroups in all (what the chip holds at once: 512 / 640 / 768 rows of
// 49152 in 1024 29.6 / 35 / 37 us, in up to 1536 33 / 40 / 43), each of as many whole steps as the largest needs
// (100 / 128 / 200 rows 15.0 / 15.8 / 18.7 us, cut evenly in values 17.0 / 17.4 / 20.3).
void lp_plan(LpArgs& a, int rows) {
  const int steps = (a.vocab + LP_STEP - 1) / LP_STEP;
  const int most = std::max(1, std::min({LP_CHUNKS, steps, 1024 / rows})), each = (steps + most - 1) / most;
  a.chunks = (steps + each - 1) / each;
  a.per = ((a.vocab + a.chunks - 1) / a.chunks + 7) / 8 * 8;
  a.chunks = (a.vocab + a.per - 1) / a.per;
}

template <bool BF16>
void lp_launch(const LpArgs& a, int rows, hipStream_t s) {
  hipLaunchKernelGGL(k_logprobs<BF16>, dim3((unsigned)rows * (unsigned)a.chunks), dim3(LP_NT), 0, s, a);
  if (a.chunks > 1) hipLaunchKernelGGL(k_logprobs_merge, dim3(rows), dim3(LP_NT), 0, s, a);
}

int64_t lp_part_bytes(const LpArgs& a, int rows) { return i8_pad((int64_t)rows * a.chunks * 16); }
int64_t lp_cand_bytes(const LpArgs& a, int rows) { return i8_pad((int64_t)rows * a.chunks * a.top * 8); }
int64_t lp_bytes(const LpArgs& a, int rows) {
  return a.chunks > 1 ? lp_part_bytes(a, rows) + lp_cand_bytes(a, rows) + (int64_t)rows * 8 : 0;
}

constexpr int LP_MAXROWS = 1 << 17;  // rows x LP_CHUNKS workgroups of 256 threads in one grid

bool lp_shape_ok(int rows, int vocab, int top) {
  return rows >= 1 && rows <= LP_MAXROWS && vocab >= 1 && vocab <= LP_MAXV && top >= 0 && top <= LP_TOP && top <= vocab;
}
bool lp_outputs_ok(const int32_t* tokens, int top, const float* logprob, const float* entropy, const int32_t* rank,
                   const int32_t* top_ids, const float* top_lp) {
  return entropy && (!tokens || (logprob && rank)) && (top == 0 || (top_ids && top_lp));
}

int lp_run(LpArgs a, bool bf16, int rows, void* work, hipStream_t s) {
  lp_plan(a, rows);
  char* const base = static_cast<char*>(work);
  a.part = reinterpret_cast<float4*>(base);
  a.cand = reinterpret_cast<u64*>(base + lp_part_bytes(a, rows));
  a.given = reinterpret_cast<float2*>(base + lp_part_bytes(a, rows) + lp_cand_bytes(a, rows));
  if (bf16) lp_launch<true>(a, rows, s);
  else lp_launch<false>(a, rows, s);
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}

// Features -> log probabilities: blocks of rows through the 8-bit head, whose fp32 logits stay in the workspace, up to
// 256 MB of them. 1024 rows of 49152 in one block are three whole rounds of 256 x 256 tiles, 512 one and a half, which
// take two: 185 us in one block, 215 in two (2048 rows in blocks of 256 / 512 MB: 395 / 379).
struct HeadPlan {
  int rows;  // of a block
  int64_t logits, linear, lp, bytes;
};
HeadPlan head_plan(int m, int n, int k, int top) {
  HeadPlan p{};
  const int64_t fit = std::max<int64_t>(1, (256ll << 20) / ((int64_t)n * 4));
  p.rows = (int)std::min<int64_t>(m, fit >= 256 ? fit / 256 * 256 : fit);
  LpArgs a{};
  a.vocab = n;
  a.top = top;
  int64_t lp = 0, linear = 0;
  for (const int r : {p.rows, m % p.rows}) {  // whole blocks and the last one
    if (r == 0) continue;
    lp_plan(a, r);
    lp = std::max(lp, lp_bytes(a, r));
    linear = std::max(linear, i8_linear_bytes(r, n, k));
  }
  p.logits = 0;
  p.linear = i8_pad((int64_t)p.rows * n * 4);
  p.lp = p.linear + i8_pad(linear);
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
           nullptr, nullptr, nullptr};
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
  for (int r0 = 0; r0 < m; r0 += p.rows) {
    const int r = std::min(p.rows, m - r0);
    int rc = i8_linear(x + (int64_t)r0 * k, wq, ws, base + p.logits, true, base + p.linear, r, n, k, s);
    if (rc != FL_OK) return rc;
    const int64_t t0 = (int64_t)r0 * top;
    LpArgs a{base + p.logits, n, n, top, 0, 0, tokens ? tokens + r0 : nullptr, tokens ? logprob + r0 : nullptr,
             entropy + r0, tokens ? rank + r0 : nullptr, top ? top_ids + t0 : nullptr, top ? top_logprobs + t0 : nullptr,
             nullptr, nullptr, nullptr};
    rc = lp_run(a, false, r, base + p.lp, s);
    if (rc != FL_OK) return rc;
  }
  return FL_OK;
}

}  // extern "C"
