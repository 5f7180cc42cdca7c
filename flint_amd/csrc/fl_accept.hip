// Verification of drafted tokens against the target's probabilities, from given random numbers (speculative
// sampling): which path of the tree stays, and the token behind it.
//
// At a node whose target row is p, the children are tried in order. After some rejections the target's distribution is
// w = max(p - C q, 0) up to its sum Z, where each rejection adds Z to C (C = 0, Z = 1 before the first): taking Z q off
// a w that is already max(p - C q, 0) and cutting at 0 is the same as max(p - (C + Z) q, 0), so w needs no memory, only
// C. Without draft probabilities (q all at the token) w is p without the rejected tokens. Child t is accepted where u
// q(t) Z < w(t). All of it in 64 bits: sums of 49152 values in another order than the caller's own must not move a
// token across a border.
#include <algorithm>
#include "fl_common.h"

namespace {

constexpr int AC_NT = 1024, AC_NW = AC_NT / FL_WAVE, AC_M = 1024;

struct AcceptArgs {
  const void *p, *q;              // [B][M][V] and [B][M - 1][V] (or null), fp32 or bf16
  const int32_t *tokens, *parents;  // [B][M]; parents null: a chain
  const float *ua, *us;           // [B][M], [B]
  int32_t *path, *count, *token;  // [B][M], [B], [B]
  int m, v;
};

template <bool BF>
__device__ __forceinline__ float at(const void* p, int64_t i) {
  if constexpr (BF) return bf2f(static_cast<const uint16_t*>(p)[i]);
  else return static_cast<const float*>(p)[i];
}

__device__ __forceinline__ double wave_dsum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// One workgroup per sequence.
template <bool BF>
__global__ __launch_bounds__(AC_NT) void k_accept(AcceptArgs a) {
  __shared__ int par[AC_M], tok[AC_M], gone[AC_M];
  __shared__ float pt[AC_M], qt[AC_M];
  __shared__ double red[AC_NW], red2[AC_NW];
  __shared__ int found[AC_NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x, V = a.v;
  const int64_t prow = (int64_t)b * a.m, qrow = (int64_t)b * (a.m - 1);
  const bool draft = a.q != nullptr;
  for (int i = tid; i < a.m; i += AC_NT) {
    int p = i == 0 ? -1 : a.parents ? a.parents[prow + i] : i - 1, t = i == 0 ? -1 : a.tokens[prow + i];
    if (p < 0 || p >= i) p = -1;  // no node of the tree: nothing leads to it
    if (t < 0 || t >= V) t = -1;
    par[i] = p, tok[i] = t;
    const bool real = p >= 0 && t >= 0;
    pt[i] = real ? at<BF>(a.p, (prow + p) * V + t) : 0.0f;
    qt[i] = !draft ? 1.0f : real ? at<BF>(a.q, (qrow + p) * V + t) : 0.0f;
  }
  __syncthreads();
  // w of an index of node `cur`'s row
  int cur = 0, n = 1, ngone = 0;
  double C = 0.0, Z = 1.0;
  bool zok = true;  // Z is that of C (with no draft: of the tokens gone)
  auto weight = [&](int i) -> double {
    const float p = at<BF>(a.p, (prow + cur) * V + i);
    double w = p;
    if (draft) {
      if (cur < a.m - 1 && C > 0.0) w -= C * (double)at<BF>(a.q, (qrow + cur) * V + i);
    } else {
      for (int k = 0; k < ngone; ++k)
        if (gone[k] == i) w = 0.0;
    }
    return w > 0.0 ? w : 0.0;
  };
  const int seg = (V + AC_NW - 1) / AC_NW, s0 = min(V, wave * seg), s1 = min(V, s0 + seg);
  auto total = [&]() -> double {  // red: the waves' sums over their segments
    double s = 0.0;
    for (int i = s0 + lane; i < s1; i += 64) s += weight(i);
    s = wave_dsum(s);
    __syncthreads();
    if (lane == 0) red[wave] = s;
    __syncthreads();
    s = 0.0;
    for (int i = 0; i < AC_NW; ++i) s += red[i];
    return s;
  };
  if (tid == 0) a.path[prow] = 0;
  for (int i = 1; i < a.m; ++i) {
    if (par[i] != cur || tok[i] < 0) continue;
    if (!zok) {
      Z = total();
      zok = true;
    }
    double w = pt[i];
    if (draft) w -= C * (double)qt[i];
    else
      for (int k = 0; k < ngone; ++k)
        if (gone[k] == tok[i]) w = 0.0;
    if ((double)a.ua[prow + i] * (double)qt[i] * Z < w) {
      cur = i, C = 0.0, Z = 1.0, zok = true, ngone = 0;
      if (tid == 0) a.path[prow + n] = i;
      ++n;
      __syncthreads();
    } else {
      C += Z;
      zok = false;
      if (!draft) {
        __syncthreads();
        if (tid == 0) gone[ngone] = tok[i];
        ++ngone;
        __syncthreads();
      }
    }
  }
  for (int i = n + tid; i < a.m; i += AC_NT) a.path[prow + i] = -1;
  double sum = total();
  if (!(sum > 0.0)) {  // nothing left: the row itself
    C = 0.0, ngone = 0;
    sum = total();
  }
  // the first index where the running sum passes `want`: the segment, then the piece of it, then the lane
  const double want = (double)a.us[b] * sum;
  double run = 0.0;
  int sg = -1;
  double before = 0.0;
  int last = -1;  // the last segment with any weight
  double before_last = 0.0;
  for (int i = 0; i < AC_NW; ++i) {
    if (sg < 0 && run + red[i] > want) sg = i, before = run;
    if (red[i] > 0.0) last = i, before_last = run;
    run += red[i];
  }
  if (sg < 0) sg = last, before = before_last;
  int result = -1;
  if (sg >= 0 && sum > 0.0 && sum < INFINITY) {
    const int g0 = min(V, sg * seg), g1 = min(V, g0 + seg);
    // wave 0 walks the segment, 64 values at a time
    if (wave == 0) {
      int best = -1, tail = -1;
      for (int i0 = g0; i0 < g1 && best < 0; i0 += 64) {
        const int i = i0 + lane;
        const double w = i < g1 ? weight(i) : 0.0;
        double inc = w;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const double u = __shfl_up(inc, o, 64);
          if (lane >= o) inc += u;
        }
        const unsigned long long hit = __ballot(w > 0.0 && before + inc > want), any = __ballot(w > 0.0);
        if (hit) best = i0 + __ffsll((unsigned long long)hit) - 1;
        if (any) tail = i0 + 63 - __clzll((long long)any);
        before += __shfl(inc, 63, 64);
      }
      result = best >= 0 ? best : tail;
    }
  }
  if (tid == 0) a.token[b] = result, a.count[b] = n;
  (void)red2, (void)found;
}

}  // namespace

extern "C" {

int fl_accept(const void* probs, const void* draft, int32_t bf16, const int32_t* tokens, const int32_t* parents,
              const float* accept_u, const float* sample_u, int32_t* path, int32_t* count, int32_t* token, int32_t b,
              int32_t m, int32_t vocab, void* stream) {
  if (!probs || !tokens || !accept_u || !sample_u || !path || !count || !token) return FL_E_ARG;
  if (b < 1 || b > 65536 || m < 1 || m > AC_M || vocab < 1 || vocab > 1 << 20) return FL_E_ARG;
  const AcceptArgs a{probs, m > 1 ? draft : nullptr, tokens, parents, accept_u, sample_u, path, count, token, m, vocab};
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (bf16) hipLaunchKernelGGL(k_accept<true>, dim3(b), dim3(AC_NT), 0, s, a);
  else hipLaunchKernelGGL(k_accept<false>, dim3(b), dim3(AC_NT), 0, s, a);
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}

}  // extern "C"
