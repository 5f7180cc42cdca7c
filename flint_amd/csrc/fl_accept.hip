// Verification of drafted tokens against the target's probabilities, from given random numbers (speculative
// sampling): which path of the tree stays, and the token behind it.
//
// At a node whose target row is p, the children are tried in order. After some rejections the target's distribution is
// w = max(p - C q, 0) up to its sum Z, where each rejection adds Z to C (C = 0, Z = 1 before the first): taking Z q off
// a w that is already max(p - C q, 0) and cutting at 0 is the same as max(p - (C + Z) q, 0), so w needs no memory, only
// C. Without draft probabilities (q all at the token) w is p without the rejected tokens. Child t is accepted where u
// q(t) Z < w(t). All of it in 64 bits: sums of 49152 values in another order than the caller's own must not move a
// token across a border.
#include <type_traits>
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
// a row behind a range check: 0 past its end
template <bool BF>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* p, int64_t row, int v) {
  return buf_rsrc(static_cast<const char*>(p) + row * v * (BF ? 2 : 4), (uint32_t)v * (BF ? 2u : 4u));
}
template <bool BF>
__device__ __forceinline__ float row_ld(__amdgpu_buffer_rsrc_t r, uint32_t i) {
  if constexpr (BF) return bf2f(__builtin_amdgcn_raw_buffer_load_b16(r, 2u * i, 0, 0));
  else return __uint_as_float(buf_ld32(r, 4u * i));
}
// the sum over a wave's lanes, in every lane, by VALU exchanges of both halves
template <typename F>
__device__ __forceinline__ double dsum_step(double v, F lane) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = __float_as_uint(lane(__uint_as_float((uint32_t)u))), hi = __float_as_uint(lane(__uint_as_float((uint32_t)(u >> 32))));
  return v + __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double wave_dsum(double v) {
  v = dsum_step(v, lane_xor1);
  v = dsum_step(v, lane_xor2);
  v = dsum_step(v, lane_half_mirror);
  v = dsum_step(v, lane_mirror);
  v = dsum_step(v, lane_xor16);
  return dsum_step(v, lane_xor32);
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }

// One workgroup per tree; its waves sum pieces of a row for the rejections that need Z and for the last token (without draft
// probabilities a node's row is summed once and rejected tokens are taken off, and again where little is left). One CU
// reads a row of 49152 fp32 values and its draft row in 2.6 us at its 64 bytes a cycle, about what one exchange between
// workgroups costs, so a row stays with one. (Held in registers between two sums, the row's 96 values a lane and their
// conversions spilled.)
template <bool BF, bool DRAFT>
__global__ __launch_bounds__(AC_NT) void k_accept(AcceptArgs a) {
  __shared__ double red[2][AC_NW];
  __shared__ int gone[AC_M];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), b = blockIdx.x, V = a.v;
  const int64_t prow = (int64_t)b * a.m, qrow = (int64_t)b * (a.m - 1);
  const int seg = ((V + AC_NW - 1) / AC_NW + 63) / 64 * 64;  // a wave's piece of a row
  int cur = 0, n = 1, ngone = 0, turn = 0;  // node; nodes of the path; tokens rejected at the node
  bool fresh = true;                        // Z is the sum of w (or 1)
  double C = 0.0, Z = 1.0;
  // without draft probabilities: the row's sum (once known) without the tokens gone but the last, whose p is `last`; what it
  // was when it was last summed
  double rest = -1.0, last = 0.0, whole = 0.0;
  __amdgpu_buffer_rsrc_t pr, qr;
  auto open = [&] {
    pr = row_rsrc<BF>(a.p, prow + cur, V);
    // before a rejection q does not count, and a leaf's row may hold anything (the last node has none): not read
    qr = DRAFT && C > 0.0 ? row_rsrc<BF>(a.q, qrow + cur, V) : buf_rsrc(a.p, 0);
  };
  auto cut = [&](float p, float q) -> double {
    const double w = DRAFT ? __builtin_fma(-C, (double)q, (double)p) : (double)p;
    return w > 0.0 ? w : 0.0;
  };
  // This wave's sum of w over [s0, s1), U loads of a lane and row in flight. Loads past the end cost as much as others, so
  // U is what a piece needs; the next U in flight behind the sums cost more than they gave (48 trees 23 us a call, 21 without).
  auto piece = [&](auto unroll, int s0, int s1) -> double {
    constexpr int U = decltype(unroll)::value;
    double s[4] = {};
    for (int i0 = s0; i0 < s1; i0 += 64 * U) {
      float p[U], q[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = i0 + 64 * j + lane;
        p[j] = row_ld<BF>(pr, i < s1 ? (uint32_t)i : 0x3FFFFFFFu);
        q[j] = DRAFT ? row_ld<BF>(qr, i < s1 ? (uint32_t)i : 0x3FFFFFFFu) : 0.0f;
      }
      if (!DRAFT)
        for (int k = 0; k < ngone; ++k) {
          const int d = gone[k] - i0 - lane;
#pragma unroll
          for (int j = 0; j < U; ++j) p[j] = d == 64 * j ? 0.0f : p[j];
        }
#pragma unroll
      for (int j = 0; j < U; ++j) s[j & 3] += cut(p[j], q[j]);
    }
    return wave_dsum((s[0] + s[1]) + (s[2] + s[3]));
  };
  // all waves' sums of their pieces of [g0, g1) to red[turn]
  auto pieces = [&](auto unroll, int g0, int g1, int len) {
    turn ^= 1;
    const int s0 = min(g1, g0 + wave * len);
    const double s = piece(unroll, s0, min(g1, s0 + len));
    if (lane == 0) red[turn][wave] = s;
    __syncthreads();
  };
  auto total = [&]() -> double {
    open();
    pieces(std::integral_constant<int, 16>{}, 0, V, seg);
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < AC_NW; ++i) s += red[turn][i];
    return s;
  };
  if (tid == 0) a.path[prow] = 0;
  for (int n0 = 0; n0 < a.m; n0 += 64) {  // nodes in order, 64 at a time, one per lane
    const int i = n0 + lane;
    int par = -1, tok = -1;
    float pt = 0.0f, qt = 1.0f, u = 0.0f;
    if (i > 0 && i < a.m) {
      par = a.parents ? a.parents[prow + i] : i - 1;
      tok = a.tokens[prow + i];
      u = a.ua[prow + i];
      if (par >= 0 && par < i && tok >= 0 && tok < V) {
        pt = at<BF>(a.p, (prow + par) * V + tok);
        if (DRAFT) qt = at<BF>(a.q, (qrow + par) * V + tok);
      } else {
        par = -1;  // no node of the tree, or no token: passed over
      }
    }
    unsigned long long ahead = ~0ull;  // of these 64 not yet passed
    for (;;) {
      const unsigned long long kids = __ballot(par == cur) & ahead;
      if (!kids) break;
      const int l = __ffsll(kids) - 1;
      ahead = l == 63 ? 0 : ~0ull << (l + 1);
      const int t = __builtin_amdgcn_readlane(tok, l);
      const float p1 = lane_of(pt, l), q1 = lane_of(qt, l), u1 = lane_of(u, l);
      if (!fresh) {
        if (DRAFT) {
          Z = total();
        } else {  // the row's sum without the tokens gone
          if (rest < 0.0) {  // one token is gone: taken off here, as the later ones are one by one
            ngone = 0;
            whole = rest = total();
            ngone = 1;
          }
          rest -= last;
          // where little is left, the difference is what rounding left of it: summed anew (else it is good to 2^-40)
          if (!(rest >= whole * 0x1p-10)) whole = rest = total();
          Z = rest;
        }
        fresh = true;
      }
      double w = cut(p1, q1);
      if (!DRAFT) {
        bool again = false;  // proposed and rejected before
        for (int k = lane; k < ngone; k += 64) again = again || gone[k] == t;
        if (__any(again)) w = 0.0;
      }
      if ((double)u1 * (double)q1 * Z < w) {
        cur = n0 + l, C = 0.0, Z = 1.0, rest = -1.0, ngone = 0, fresh = true;
        if (tid == 0) a.path[prow + n] = cur;
        ++n;
        if (!DRAFT) __syncthreads();  // gone is free again
      } else {
        C += Z;
        fresh = false;
        if (!DRAFT) {
          last = w;
          if (tid == 0) gone[ngone] = t;
          ++ngone;
          __syncthreads();
        }
      }
    }
  }
  for (int i = n + tid; i < a.m; i += AC_NT) a.path[prow + i] = -1;
  double sum = total();
  if (!(sum > 0.0)) {  // nothing left: the row itself
    C = 0.0, ngone = 0;
    sum = total();
  }
  int result = -1;
  if (sum > 0.0 && sum < INFINITY) {
    // the first index at which the running sum passes `want`: the wave's piece, pieces of that until 256 values are left,
    // then four in a row a lane
    const double want = (double)a.us[b] * sum;
    double before = 0.0;
    int g0 = 0, g1 = V, len = seg;
    for (;;) {
      int pick = -1, tail = 0;
      double run = before, at_pick = before, at_tail = before;
#pragma unroll
      for (int i = 0; i < AC_NW; ++i) {
        const double r = red[turn][i];
        if (pick < 0 && run + r > want) pick = i, at_pick = run;
        if (r > 0.0) tail = i, at_tail = run;
        run += r;
      }
      if (pick < 0) pick = tail, at_pick = at_tail;  // the sums of pieces differ in their last bits
      before = at_pick;
      g0 = min(g1, g0 + pick * len);
      g1 = min(g1, g0 + len);
      if (g1 - g0 <= 256) break;
      len = ((g1 - g0 + AC_NW - 1) / AC_NW + 63) / 64 * 64;
      pieces(std::integral_constant<int, 4>{}, g0, g1, len);
    }
    double w[4], own = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = g0 + 4 * lane + j;
      w[j] = i < g1 ? cut(row_ld<BF>(pr, i), DRAFT ? row_ld<BF>(qr, i) : 0.0f) : 0.0;
      if (!DRAFT)
        for (int k = 0; k < ngone; ++k)
          if (gone[k] == i) w[j] = 0.0;
      own += w[j];
    }
    double inc = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double x = __shfl_up(inc, o, 64);
      if (lane >= o) inc += x;
    }
    const unsigned long long hit = __ballot(own > 0.0 && before + inc > want), any = __ballot(own > 0.0);
    if (any) {  // none: a piece whose sum was its last bits
      const int l = hit ? __ffsll(hit) - 1 : 63 - __clzll((long long)any);
      double run = before + (inc - own);
      int mine = -1;
      bool done = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        run += w[j];
        if (!done && w[j] > 0.0) mine = g0 + 4 * lane + j, done = run > want;
      }
      result = __builtin_amdgcn_readlane(mine, l);
    }
  }
  if (tid == 0) a.token[b] = result, a.count[b] = n;
}

template <bool BF, bool DRAFT>
void accept_launch(const AcceptArgs& a, int b, hipStream_t s) {
  hipLaunchKernelGGL((k_accept<BF, DRAFT>), dim3(b), dim3(AC_NT), 0, s, a);
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
  if (a.q) bf16 ? accept_launch<true, true>(a, b, s) : accept_launch<false, true>(a, b, s);
  else bf16 ? accept_launch<true, false>(a, b, s) : accept_launch<false, false>(a, b, s);
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}

}  // extern "C"
