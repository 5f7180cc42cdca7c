// Attention of the nodes of a drafted tree (or chain, or one token) over a K/V cache, and the weight that every
// cached key gathers from them.
//
// The rows of a key head are its (node, query head) pairs, node-major: row t * rep + j. Scores are taken transposed,
// S^T = K Q^T on 32x32x16 MFMAs, so that a lane holds one row (r = lane % 32) and registers hold its keys; the softmax
// is online, per lane, in the log2 domain (p = exp2(s c - m), c = scale log2 e), in fp32; O^T += V^T P^T takes a step's
// 16 keys in the order in which the score registers already hold them, so P never crosses lanes. V^T comes out of LDS
// through the transposing read (a 16-lane group receives four rows of 16 values by column). P is split into two 16-bit
// terms. In bf16 they leave 2^-17 of a weight: with one alone 1024 tokens behind 4096 take 82 us in place of 102, but their
// outputs lie 1.3 times as far from 64 bits (0.0021 in place of 0.0016 of their norm), and the model's attention is fp32
// times V. In fp16 they share steps of 2^-24, so P is held near the top of fp16's range, tile by tile (softmax_pv): they
// leave 2^-28 of the largest weight of a tile's row, and 2^-36 of the row's largest.
#include <algorithm>
#include <type_traits>
#include "fl_gemm.h"
#include "fl_state.h"

namespace {

typedef _Float16 fl_f16x8 __attribute__((ext_vector_type(8)));
typedef short at_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) at_s16x4 at_lds4;

struct AttnArgs {
  const uint16_t *q, *k, *v;
  const int32_t* pos;   // per sequence, or null: pos0
  const uint8_t* mask;  // [M][M] per sequence, or null: a chain
  uint16_t* out;        // [B][M][heads][D]
  float* lse;           // [B][M][heads] or null (read by k_attn_weights)
  float* part;          // with key parts: o [parts][B][groups][R][D], then (m, l) [parts][B][groups][R][2]
  int b, m, heads, groups, rep, slots, pos0, R;
  int blocks, parts, kpp;  // row blocks per key head; key parts, keys of a part
  float sc;             // scale * log2 e
  int64_t q_b, q_m, q_h, k_b, k_g, k_s, v_b, v_g, v_s, mask_b;
};

template <bool H>
__device__ __forceinline__ fl_f32x16 mma(uint4 a, uint4 b, fl_f32x16 c) {
  if constexpr (H)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(fl_f16x8, a), __builtin_bit_cast(fl_f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(fl_bf16x8, a), __builtin_bit_cast(fl_bf16x8, b), c, 0, 0, 0);
}
template <bool H>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (H) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    return pack_bf16x2(a, b);
  }
}
template <bool H>
__device__ __forceinline__ float lo16(uint32_t w) {
  if constexpr (H) return (float)__builtin_bit_cast(_Float16, (uint16_t)w);
  else return bflo(w);
}
template <bool H>
__device__ __forceinline__ float hi16(uint32_t w) {
  if constexpr (H) return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
  else return bfhi(w);
}
template <bool H>
__device__ __forceinline__ bool finite16(uint32_t w) {  // both values of a pair
  constexpr uint32_t e = H ? 0x7C00u : 0x7F80u;
  return (w & e) != e && (w & (e << 16)) != (e << 16);
}
template <bool H>
__device__ __forceinline__ bool finite16(uint4 w) {
  return finite16<H>(w.x) && finite16<H>(w.y) && finite16<H>(w.z) && finite16<H>(w.w);
}
template <bool H>
__device__ __forceinline__ uint32_t only_finite(uint32_t w) {  // a value that is none becomes 0
  constexpr uint32_t e = H ? 0x7C00u : 0x7F80u;
  if ((w & e) == e) w &= 0xFFFF0000u;
  if ((w & (e << 16)) == (e << 16)) w &= 0xFFFFu;
  return w;
}
template <bool H>
__device__ __forceinline__ uint4 only_finite(uint4 w) {
  return make_uint4(only_finite<H>(w.x), only_finite<H>(w.y), only_finite<H>(w.z), only_finite<H>(w.w));
}

// Keys [0, keys) of a sequence and this workgroup's part of them; keys < 0: a pos outside the cache.
struct Span {
  int pos, keys, kb0, kend;
};
// Every part has kpp keys, so that the workgroups of a ragged batch take as long as each other; a short sequence has
// fewer parts.
__device__ __forceinline__ Span span_of(const AttnArgs& a, int b, int part) {
  Span s;
  s.pos = a.pos ? __builtin_amdgcn_readfirstlane(a.pos[b]) : a.pos0;  // the wave's, in a scalar register
  if (s.pos < 0 || s.pos > a.slots - a.m) {
    s.pos = 0, s.keys = -1, s.kb0 = s.kend = 0;
    return s;
  }
  s.keys = s.pos + a.m;
  s.kb0 = (int)min((int64_t)s.keys, (int64_t)part * a.kpp);
  s.kend = min(s.keys - s.kb0, a.kpp) + s.kb0;
  return s;
}

// Scores of the keys of a tile that node t does not see, or that lie behind `kend`, become -inf. A chain's node sees up
// to itself; a tree's bits come from the mask by range-checked byte loads, all in flight together (an offset outside
// reads 0).
template <int KT>
__device__ __forceinline__ void hide(const AttnArgs& a, const uint8_t* mask, int pos, int kend, int kb, int t, fl_f32x16 (&s)[KT]) {
  const int hf = (threadIdx.x & 63) >> 5;
  if (!mask) {
    const int lim = min(kend, pos + t + 1) - kb - 4 * hf;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kt][i] = 32 * kt + 8 * (i >> 2) + (i & 3) < lim ? s[kt][i] : -INFINITY;
    return;
  }
  const auto mr = buf_rsrc(mask, (uint32_t)a.m * (uint32_t)a.m);
  const uint32_t row = (uint32_t)t * (uint32_t)a.m;
  const int j0 = kb + 4 * hf - pos, jend = kend - pos;  // node of register 0; nodes before the end (one at least)
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    uint32_t bit[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = j0 + 32 * kt + 8 * (i >> 2) + (i & 3);
      bit[i] = __builtin_amdgcn_raw_buffer_load_b8(mr, (uint32_t)j < (uint32_t)jend ? row + (uint32_t)j : 0xFFFFFFF0u, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = j0 + 32 * kt + 8 * (i >> 2) + (i & 3);
      s[kt][i] = (bit[i] | (uint32_t)(j >> 31)) != 0 ? s[kt][i] : -INFINITY;  // a cached key: j < 0
    }
    asm volatile("" ::: "memory");  // 16 registers for the bits, not 32
  }
}

// A tile of TK keys from slot kb on: the range check makes what lies behind the part's end zeros. The base moves with
// the tile (scalar arithmetic), so lane offsets are constants and no offset passes 32 bits however long the cache is.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const uint16_t* base, int64_t stride, int kb, int kend, int tk, int d) {
  const int rem = min(kend - kb, tk);
  const uint32_t bytes = rem <= 0 ? 0u : (uint32_t)((rem - 1) * stride + d) * 2u;
  return buf_rsrc(base + (int64_t)kb * stride, bytes);
}

// 16 bytes at a lane's offset and a scalar one
__device__ __forceinline__ uint4 tile_ld(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, soff, 0));
}

// V in LDS: rows of D values, its 64-byte blocks swapped by row so that a transposing read's four rows lie on
// different banks.
template <int D>
__device__ __forceinline__ int v_swz(int row) {
  return D == 64 ? (row >> 1) & 1 : row & 3;
}
template <int D>
__device__ __forceinline__ int v_at(int row, int c) {  // byte of the 16-byte chunk c of a row
  return row * (2 * D) + ((c >> 2) ^ v_swz<D>(row)) * 64 + (c & 3) * 16;
}
__device__ __forceinline__ uint2 tr4(const unsigned char* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds4*)(p)));
}

// The state of 32 rows: this lane's row's reference (log2 domain), sum, and O^T (dims 32 d + 8 (i / 4) + 4 hf + i % 4),
// the last two in units of 2^m; fp16 also has an integer near the row's largest score, to which its reference returns at
// the end
template <bool H, int DT>
struct Rows {
  fl_f32x16 o[DT];
  float m, l, top;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    m = top = -INFINITY, l = 0.0f;
  }
  __device__ __forceinline__ void refer_to(float mn) {
    const float corr = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= corr;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] *= corr;
  }
  __device__ __forceinline__ void finish() {
    if constexpr (H) refer_to(top);
  }
};

// One tile of 32 KT keys' scores into the state. s: raw scores, s[kt][i] of key 32 kt + 8 (i / 4) + 4 hf + i % 4, -inf
// where not seen; vt: the tile's V in LDS.
template <bool H, int D, int KT>
__device__ __forceinline__ void softmax_pv(fl_f32x16 (&s)[KT], Rows<H, D / 32>& st, float sc, const unsigned char* vt) {
  constexpr int DT = D / 32;
  const int lane = threadIdx.x & 63, i16 = lane & 15, hf = lane >> 5;
  float mx = -INFINITY;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 16; i += 2) mx = fmaxf(fmaxf(s[kt][i], s[kt][i + 1]), mx);  // one three-way maximum each
  mx = xor32_max(mx) * sc;
  // Arguments are s c - m rounded once, m a rounded s c. From 2^22 on that one's own rounding would show in all of a row's
  // weights alike (from 2^31 on beyond what fp32 holds, from 2^24 on fp16): there s c is rounded first, as m is.
  if (__builtin_expect(__any(fabsf(mx) >= 0x1p22f && mx > -INFINITY), 0)) {
    const bool big = fabsf(mx) >= 0x1p22f && mx > -INFINITY;
    const float f = big ? sc : 1.0f;
    sc = big ? 1.0f : sc;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kt][i] *= f;
  }
  if constexpr (H) {
    // m is an integer, 11 below the scores of some tile: p lies below 2^15 (fp16 ends at 2^16) and a tile's largest at
    // 2^3 or more, so that what lies far below a row's maximum keeps its bits. It follows a tile's maximum both ways
    // (o and l then grow by that power of two), down to 40 below the row's: 2^-76 of its largest weight may be dropped,
    // and o stays below 2^(56 + 16) times the number of keys. 16 trees of 13 behind 8011 keys 59 us; with the reference
    // of bf16, which lost those, 57.
    if (__any(fabsf((mx - st.m) - 9.0f) > 6.0f)) {
      const float near = floorf(fmaxf(mx, st.top - 40.0f));
      const float mn = near - (near - 11.0f) > 15.0f ? near : near - 11.0f;  // no 11 below where floats lie 16 apart
      const bool move = mx - st.m > 15.0f || (mx > -INFINITY && st.m - mn > 8.0f);
      if (__any(move)) {
        st.refer_to(move ? mn : st.m);
        st.top = fmaxf(st.top, st.m + 11.0f);
      }
    }
  } else {
    // m is any reference near the maximum: it follows only where a row's passed it by 2^8 (p and l stay far inside their
    // range), which after a row's first tile hardly happens; some row of 32 has a new maximum in half of all tiles
    if (__any(mx > st.m + 8.0f)) st.refer_to(fmaxf(st.m, mx));
  }
  const float mu = st.m == -INFINITY ? 0.0f : st.m;
  const int row = 4 * hf + (i16 >> 2);
  const unsigned char* vp = vt + row * (2 * D) + (i16 & 3) * 8 + ((lane >> 4) & 1) * 32;
  float ps[4] = {};
  // 16 keys at a time: their exponentials and terms of P while the matrix cores run the 16 before
#pragma unroll
  for (int st16 = 0; st16 < 2 * KT; ++st16) {
    uint2 v0[DT], v1[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const unsigned char* vd = vp + st16 * 16 * (2 * D) + (d ^ v_swz<D>(row)) * 64;
      v0[d] = tr4(vd), v1[d] = tr4(vd + 8 * (2 * D));
    }
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[st16 >> 1][8 * (st16 & 1) + i], sc, -mu));
      ps[i & 3] += p[i];
    }
    uint32_t ph[4], pl[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ph[e] = pack16<H>(p[2 * e], p[2 * e + 1]);
      asm("" : "+v"(ph[e]));  // read back from the pair, not converted again
      pl[e] = pack16<H>(p[2 * e] - lo16<H>(ph[e]), p[2 * e + 1] - hi16<H>(ph[e]));
    }
    const uint4 bh = make_uint4(ph[0], ph[1], ph[2], ph[3]), bl = make_uint4(pl[0], pl[1], pl[2], pl[3]);
#pragma unroll
    for (int d = 0; d < DT; ++d) st.o[d] = mma<H>(make_uint4(v0[d].x, v0[d].y, v1[d].x, v1[d].y), bh, st.o[d]);
#pragma unroll
    for (int d = 0; d < DT; ++d) st.o[d] = mma<H>(make_uint4(v0[d].x, v0[d].y, v1[d].x, v1[d].y), bl, st.o[d]);
  }
  st.l += xor32_sum((ps[0] + ps[1]) + (ps[2] + ps[3]));
}

// Values of V that are not finite, once a wave's keys (tiles of TK from kb0 on, `step` apart) are through: a row that sees
// one has it in that dimension under any weight, where the sums may hold 0 times infinity, or what a second term of the
// other sign or a factor of 0 left of it. Any that met a matrix instruction shows in o; of those that were made zeros
// `odd` tells. Rows whose sum l is no number are none anyway.
template <bool H, int D, int TK>
__device__ __forceinline__ void settle_not_finite(const AttnArgs& a, const uint8_t* mask, const uint16_t* v, int pos, int kb0, int kend,
                                                  int step, int t, bool odd, Rows<H, D / 32>& st) {
  const int hf = (threadIdx.x & 63) >> 5;
  float z[4] = {};
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i & 3] = __builtin_fmaf(st.o[d][i], 0.0f, z[i & 3]);
  const bool none = __builtin_isfinite((z[0] + z[1]) + (z[2] + z[3])) || !__builtin_isfinite(st.l);
  if (__builtin_expect(!__any(odd || !none), 1)) return;
#pragma unroll
  for (int d = 0; d < D / 32; ++d) {
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.0f;
#pragma unroll 1
    for (int kb = kb0; kb < kend; kb += step) {
      const auto vr = tile_rsrc(v, a.v_s, kb, kend, TK, D);
#pragma unroll 1
      for (int key = kb; key < min(kend, kb + TK); ++key) {
        const int j = key - pos;
        const bool seen = j < 0 || (mask ? mask[(uint32_t)t * (uint32_t)a.m + (uint32_t)j] != 0 : j <= t);
        const uint32_t off = seen ? (uint32_t)((key - kb) * a.v_s + 4 * hf) * 2u : 0xFFFFFF00u;  // not seen: zeros
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint2 w = buf_ld64(vr, off + 64 * d + 16 * e);
          const float x[4] = {lo16<H>(w.x), hi16<H>(w.x), lo16<H>(w.y), hi16<H>(w.y)};
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[4 * e + i] += __builtin_isfinite(x[i]) ? 0.0f : x[i];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) st.o[d][i] = sum[i] == 0.0f ? st.o[d][i] : sum[i];
  }
}
// a part's share of a sum: what is not finite stays that under any factor
__device__ __forceinline__ float share(float f, float x) { return __builtin_isfinite(x) ? f * x : x; }

template <bool H, int D>
__device__ __forceinline__ void store_rows(const AttnArgs& a, const Rows<H, D / 32>& st, int b, int g, int part, int row, bool bad) {
  if (row >= a.R) return;
  const int hf = (threadIdx.x & 63) >> 5, t = row / a.rep, head = g * a.rep + row % a.rep;
  if (a.parts == 1) {
    const int64_t at = ((int64_t)b * a.m + t) * a.heads + head;
    const float inv = bad ? NAN : st.l == 0.0f ? 0.0f : 1.0f / st.l;
    uint16_t* d0 = a.out + at * D + 4 * hf;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<uint2*>(d0 + 32 * d + 8 * e) =
            make_uint2(pack16<H>(st.o[d][4 * e] * inv, st.o[d][4 * e + 1] * inv),
                       pack16<H>(st.o[d][4 * e + 2] * inv, st.o[d][4 * e + 3] * inv));
    if (a.lse && hf == 0)
      a.lse[at] = bad ? NAN : st.l == 0.0f ? -INFINITY : (st.m + __builtin_amdgcn_logf(st.l)) * 0.6931471805599453f;
  } else {
    const int64_t n = (int64_t)a.b * a.groups * a.R;
    const int64_t idx = (int64_t)part * n + ((int64_t)b * a.groups + g) * a.R + row;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<fl_f32x4*>(a.part + idx * D + 32 * d + 8 * e + 4 * hf) =
            fl_f32x4{st.o[d][4 * e], st.o[d][4 * e + 1], st.o[d][4 * e + 2], st.o[d][4 * e + 3]};
    if (hf == 0) {
      float* ml = a.part + (int64_t)a.parts * n * D + idx * 2;
      ml[0] = st.m;
      ml[1] = st.l;
    }
  }
}

// ---- few rows: every wave takes its own keys ------------------------------------------------------------
// 32 rows of a key head and one part of the keys per workgroup; its waves take tiles of TK keys in turn, K straight from
// memory into the MFMA's operand layout, V through a piece of LDS that only this wave uses, the next tile's loads in
// flight behind the products. No barrier until the waves' (m, l, o) meet in LDS at the end.
template <bool H, int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void k_attn_few(AttnArgs a) {
  constexpr int TK = 4096 / D, KT = TK / 32, ST = D / 16, DT = D / 32, CH = D / 8;  // CH: 16-byte chunks of a row
  constexpr int VB = TK * D * 2, MB = 18 * 64 * 4;
  __shared__ __align__(16) unsigned char smem[NW * (VB > MB ? VB : MB)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hf = lane >> 5;
  int rest = blockIdx.x;
  const int g = rest % a.groups;
  rest /= a.groups;
  const int blk = rest % a.blocks;
  rest /= a.blocks;
  const int part = rest % a.parts, b = rest / a.parts;
  const Span sp = span_of(a, b, part);
  if (a.parts > 1 && sp.kb0 >= sp.kend) return;  // the merge knows
  const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
  const uint16_t* kp = a.k + (int64_t)b * a.k_b + (int64_t)g * a.k_g;
  const uint16_t* vp = a.v + (int64_t)b * a.v_b + (int64_t)g * a.v_g;
  const int row = blk * 32 + r, rowc = min(row, a.R - 1), t = rowc / a.rep, head = g * a.rep + rowc % a.rep;
  uint4 qf[ST];
  const uint16_t* qp = a.q + (int64_t)b * a.q_b + (int64_t)t * a.q_m + (int64_t)head * a.q_h;
#pragma unroll
  for (int s = 0; s < ST; ++s) qf[s] = *reinterpret_cast<const uint4*>(qp + s * 16 + hf * 8);
  Rows<H, DT> st;
  st.clear();
  unsigned char* vt = smem + wave * VB;
  unsigned char* vw = vt + v_at<D>(lane / CH, lane % CH);  // a sweep of 64 lanes is 1 KB of rows, at the same swizzle
  const uint32_t ko = (uint32_t)(r * a.k_s + hf * 8) * 2u, kstep = (uint32_t)(32 * a.k_s) * 2u;
  const uint32_t vo = (uint32_t)((lane / CH) * a.v_s + (lane % CH) * 8) * 2u, vstep = (uint32_t)((64 / CH) * a.v_s) * 2u;
  uint4 kf[KT][ST], vf[8];
  auto load = [&](int kb) {
    const auto kr = tile_rsrc(kp, a.k_s, kb, sp.kend, TK, D), vr = tile_rsrc(vp, a.v_s, kb, sp.kend, TK, D);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int s = 0; s < ST; ++s) kf[kt][s] = tile_ld(kr, ko + s * 32, kt * kstep);
#pragma unroll
    for (int i = 0; i < 8; ++i) vf[i] = tile_ld(vr, vo, i * vstep);
  };
  bool odd = false;  // some node's V is not finite
  int kb = sp.kb0 + wave * TK;
  if (kb < sp.kend) load(kb);
  for (; kb < sp.kend; kb += NW * TK) {
    const bool nodes = kb + TK > sp.pos;  // some keys of the tile are nodes (or lie behind the end)
    if (nodes) {
      bool fin = true;
#pragma unroll
      for (int i = 0; i < 8; ++i) fin = fin && finite16<H>(vf[i]);
      if (__any(!fin)) {
        odd = true;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = kb + lane / CH + i * (64 / CH);
          if (key >= sp.pos) vf[i] = only_finite<H>(vf[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(vw + i * 1024) = vf[i];
    fl_f32x16 s[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kt][i] = 0.0f;
#pragma unroll
      for (int e = 0; e < ST; ++e) s[kt] = mma<H>(kf[kt][e], qf[e], s[kt]);
    }
    const int kn = kb + NW * TK;
    load(kn < sp.kend ? kn : sp.kend);  // behind the end: zeros, nothing read
    if (nodes) hide<KT>(a, mask, sp.pos, sp.kend, kb, t, s);
    softmax_pv<H, D, KT>(s, st, a.sc, vt);
  }
  st.finish();
  settle_not_finite<H, D, TK>(a, mask, vp, sp.pos, sp.kb0 + wave * TK, sp.kend, NW * TK, t, odd, st);
  // the waves' states, one 32-dim tile at a time: each wave sums its share of the registers over the waves
  static_assert(16 % NW == 0 && 16 / NW == 2, "two registers each");
  const int i0 = 2 * wave;  // dims 32 d + 8 (i0 / 4) + 4 hf + i0 % 4 and the next
  float mm = -INFINITY, ll = 0.0f;
  const int64_t n = (int64_t)a.b * a.groups * a.R, idx = (int64_t)part * n + ((int64_t)b * a.groups + g) * a.R + row;
  const int64_t at = ((int64_t)b * a.m + t) * a.heads + head;
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    __syncthreads();
    float* mine = reinterpret_cast<float*>(smem) + wave * 18 * 64 + lane;
#pragma unroll
    for (int i = 0; i < 16; ++i) mine[i * 64] = st.o[d][i];
    mine[16 * 64] = st.m;
    mine[17 * 64] = st.l;
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(smem) + lane;
    if (d == 0) {
#pragma unroll
      for (int w = 0; w < NW; ++w) mm = fmaxf(mm, all[(w * 18 + 16) * 64]);
    }
    const float mu = mm == -INFINITY ? 0.0f : mm;
    float o0 = 0.0f, o1 = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float e = __builtin_amdgcn_exp2f(all[(w * 18 + 16) * 64] - mu);
      l += e * all[(w * 18 + 17) * 64];
      o0 += e * all[(w * 18 + i0) * 64];
      o1 += e * all[(w * 18 + i0 + 1) * 64];
    }
    ll = l;
    if (__builtin_expect(__any(!__builtin_isfinite(o0 + o1)), 0)) {
      o0 = o1 = 0.0f;
#pragma unroll 1
      for (int w = 0; w < NW; ++w) {
        const float e = __builtin_amdgcn_exp2f(all[(w * 18 + 16) * 64] - mu);
        o0 += share(e, all[(w * 18 + i0) * 64]);
        o1 += share(e, all[(w * 18 + i0 + 1) * 64]);
      }
    }
    const int dim = 32 * d + 8 * (i0 >> 2) + 4 * hf + (i0 & 3);
    if (row < a.R) {
      if (a.parts == 1) {
        const float inv = sp.keys < 0 ? NAN : l == 0.0f ? 0.0f : 1.0f / l;
        *reinterpret_cast<uint32_t*>(a.out + at * D + dim) = pack16<H>(o0 * inv, o1 * inv);
      } else {
        *reinterpret_cast<float2*>(a.part + idx * D + dim) = make_float2(o0, o1);
      }
    }
  }
  if (wave == 0 && hf == 0 && row < a.R) {
    if (a.parts == 1) {
      if (a.lse) a.lse[at] = sp.keys < 0 ? NAN : ll == 0.0f ? -INFINITY : (mm + __builtin_amdgcn_logf(ll)) * 0.6931471805599453f;
    } else {
      float* ml = a.part + (int64_t)a.parts * n * D + idx * 2;
      ml[0] = mm;
      ml[1] = ll;
    }
  }
}

// ---- many rows: the workgroup's waves share the keys ------------------------------------------------------
// 32 rows per wave, four waves, one part of the keys in rounds of TK. K and V go straight from memory into a ring of
// three LDS stages, two rounds ahead (a round takes less than a microsecond, about what a load does; through registers,
// one round ahead, the waves waited for it every time), swizzled by what each lane loads; one barrier a round.
template <bool H, int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void k_attn_many(AttnArgs a) {
  constexpr int TK = 4096 / D, KT = TK / 32, ST = D / 16, DT = D / 32, CH = D / 8, NS = 3;
  constexpr int TILE = TK * D * 2, PW = TILE / 4096;  // bytes of K or V of a round (8 KB); 1 KB loads of a wave of each
  __shared__ __align__(16) unsigned char ring[NS][2][TILE];
  __shared__ int odd;  // some node's V is not finite
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hf = lane >> 5;
  int rest = blockIdx.x;
  const int g = rest % a.groups;
  rest /= a.groups;
  const int part = rest % a.parts;
  rest /= a.parts;
  const int blk = a.blocks - 1 - rest % a.blocks, b = rest / a.blocks;  // the longest rows first
  const Span sp = span_of(a, b, part);
  if (a.parts > 1 && sp.kb0 >= sp.kend) return;
  const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
  const uint16_t* kp = a.k + (int64_t)b * a.k_b + (int64_t)g * a.k_g;
  const uint16_t* vp = a.v + (int64_t)b * a.v_b + (int64_t)g * a.v_g;
  const int row = blk * 128 + wave * 32 + r, rowc = min(row, a.R - 1), t = rowc / a.rep;
  // a chain's rows see nothing behind their own node: the workgroup's last key, and the wave's
  int kend = sp.kend, wend = sp.kend;
  if (!mask && sp.keys > 0) {
    kend = min(kend, sp.pos + min(a.m - 1, (blk * 128 + 127) / a.rep) + 1);
    wend = min(kend, sp.pos + min(a.m - 1, (blk * 128 + wave * 32 + 31) / a.rep) + 1);
  }
  kend = __builtin_amdgcn_readfirstlane(kend);
  const int wfull = sp.pos + (mask ? 0 : min(a.m - 1, (blk * 128 + wave * 32) / a.rep) + 1);  // keys that all its rows see
  uint4 qf[ST];
  const uint16_t* qp = a.q + (int64_t)b * a.q_b + (int64_t)t * a.q_m + (int64_t)(g * a.rep + rowc % a.rep) * a.q_h;
#pragma unroll
  for (int s = 0; s < ST; ++s) qf[s] = *reinterpret_cast<const uint4*>(qp + s * 16 + hf * 8);
  Rows<H, DT> st;
  st.clear();
  // 16-byte chunk i * 256 + tid of a tile's LDS: a row of it, and there the chunk that the swizzle puts in its place
  auto k_at = [&](int key, int ch) {  // 16 rows' chunk on 16 different places
    return key * (2 * D) + (ch ^ (D == 64 ? (key >> 1) & 7 : key & 15)) * 16;
  };
  const int k0 = tid / CH, slot = tid % CH;  // a sweep of 256 threads is 256 / CH rows, at the same swizzle
  const uint32_t ko = (uint32_t)(k0 * a.k_s) * 2u + (uint32_t)(slot ^ (D == 64 ? (k0 >> 1) & 7 : k0 & 15)) * 16u;
  const uint32_t vo = (uint32_t)(k0 * a.v_s) * 2u + (uint32_t)(((slot >> 2) ^ v_swz<D>(k0)) * 4 + (slot & 3)) * 16u;
  const uint32_t kstep = (uint32_t)(256 / CH * a.k_s) * 2u, vstep = (uint32_t)(256 / CH * a.v_s) * 2u;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_byte*)&ring[0][0][0] + (uint32_t)wave * 1024u;
  auto load = [&](int kb, int stage) {  // behind the end: zeros, nothing read
    const int rem = min(max(kend - kb, 0), TK);
    const fl_u32x4 kw = buffer_words(kp + (int64_t)kb * a.k_s, rem ? (uint32_t)((rem - 1) * a.k_s + D) * 2u : 0u);
    const fl_u32x4 vw = buffer_words(vp + (int64_t)kb * a.v_s, rem ? (uint32_t)((rem - 1) * a.v_s + D) * 2u : 0u);
    const uint32_t at = lds0 + (uint32_t)stage * (2 * TILE);
#pragma unroll
    for (int i = 0; i < PW; ++i) dma_1k(kw, at + i * 4096, ko, i * kstep);
#pragma unroll
    for (int i = 0; i < PW; ++i) dma_1k(vw, at + TILE + i * 4096, vo, i * vstep);
  };
  if (tid == 0) odd = 0;
  __syncthreads();
  load(sp.kb0, 0);
  load(sp.kb0 + TK, 1);
  int stage = 0;
  for (int kb = sp.kb0; kb < kend; kb += TK) {
    unsigned char *ks = ring[stage][0], *vs = ring[stage][1];
    wait_loads<2 * PW>();  // this round's have landed, the next one's may be in flight
    if (kb + TK > sp.pos) {  // nodes: values of V that are not finite become zeros, each lane's own chunks
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        uint4* x = reinterpret_cast<uint4*>(vs + i * 4096 + tid * 16);
        if (kb + k0 + i * (256 / CH) >= sp.pos && !finite16<H>(*x)) {
          *x = only_finite<H>(*x);
          odd = 1;  // read behind the last round's barrier
        }
      }
    }
    lds_barrier();  // every wave's loads have landed, and the stage before this one has been read
    load(kb + 2 * TK, stage == 0 ? 2 : stage - 1);
    if (kb < wend) {
      fl_f32x16 s[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kt][i] = 0.0f;
#pragma unroll
        for (int e = 0; e < ST; ++e)
          s[kt] = mma<H>(*reinterpret_cast<const uint4*>(ks + k_at(kt * 32 + r, 2 * e + hf)), qf[e], s[kt]);
      }
      if (kb + TK > wfull) hide<KT>(a, mask, sp.pos, kend, kb, t, s);
      softmax_pv<H, D, KT>(s, st, a.sc, vs);
    }
    stage = stage == NS - 1 ? 0 : stage + 1;
  }
  wait_loads<0>();  // what was loaded ahead has landed before the LDS is given away
  st.finish();
  settle_not_finite<H, D, TK>(a, mask, vp, sp.pos, sp.kb0, wend, TK, t, odd != 0, st);
  store_rows<H, D>(a, st, b, g, part, row, sp.keys < 0);
}

// The key parts of a row (up to 64) merged: a wave per row, 16 bytes of a part's o a lane, 256 / D parts at a time
// and four of those loads in flight; the lanes of a dim meet at the end in a fixed order.
template <bool H, int D>
__global__ __launch_bounds__(256) void k_attn_merge(AttnArgs a) {
  constexpr int LP = D / 4, PP = 64 / LP;  // lanes of a part, parts side by side
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), b = blockIdx.y / a.groups, g = blockIdx.y % a.groups;
  if (row >= a.R) return;
  const int64_t n = (int64_t)a.b * a.groups * a.R, w = (int64_t)blockIdx.y * a.R + row;
  const Span sp = span_of(a, b, 0);
  const int parts = sp.keys < 0 ? 0 : (sp.keys - 1) / a.kpp + 1;
  const float* ml = a.part + (int64_t)a.parts * n * D;
  const int p0 = lane / LP, d0 = lane % LP * 4;
  // four groups of PP parts at a time; a group with no part in it is not loaded (uniform), a lane with none reads the last
  fl_f32x4 x[4];
  auto load = [&](int g0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (g0 + i * PP < parts)
        x[i] = *reinterpret_cast<const fl_f32x4*>(a.part + (min(g0 + i * PP + p0, parts - 1) * n + w) * D + d0);
  };
  load(0);
  float2 own = make_float2(-INFINITY, 0.0f);  // lane p: part p
  if (lane < parts) own = *reinterpret_cast<const float2*>(ml + (lane * n + w) * 2);
  const float mm = wave_max(own.x), mu = mm == -INFINITY ? 0.0f : mm;
  const float e = __builtin_amdgcn_exp2f(own.x - mu);  // 0 behind the last part
  const float L = wave_sum(e * own.y);
  fl_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int g0 = 0; g0 < parts; g0 += 4 * PP) {
    if (g0) load(g0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (g0 + i * PP < parts) {
        const float f = __shfl(e, (g0 + i * PP + p0) & 63, 64);
        o += g0 + i * PP + p0 < parts ? x[i] * f : fl_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
  }
  if (__builtin_expect(__any(!__builtin_isfinite((o[0] + o[1]) + (o[2] + o[3]))), 0)) {
    o = fl_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int g0 = 0; g0 < parts; g0 += 4 * PP) {
      load(g0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = __shfl(e, (g0 + i * PP + p0) & 63, 64);
        if (g0 + i * PP + p0 < parts)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[c] += share(f, x[i][c]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (LP == 16) o[i] = xor16_sum(o[i]);
    o[i] = xor32_sum(o[i]);
  }
  const int64_t at = ((int64_t)b * a.m + row / a.rep) * a.heads + g * a.rep + row % a.rep;
  const float inv = sp.keys < 0 ? NAN : L == 0.0f ? 0.0f : 1.0f / L;
  if (p0 == 0)
    *reinterpret_cast<uint2*>(a.out + at * D + d0) = make_uint2(pack16<H>(o[0] * inv, o[1] * inv), pack16<H>(o[2] * inv, o[3] * inv));
  if (a.lse && lane == 0)
    a.lse[at] = sp.keys < 0 ? NAN : L == 0.0f ? -INFINITY : (mm + __builtin_amdgcn_logf(L)) * 0.6931471805599453f;
}

// ---- the weight that every key gathers ---------------------------------------------------------------------
// w[key] (+)= sum over rows of exp2(s c - lse log2 e). Here the scores are taken as S = Q K^T, so that a lane is a key
// and registers are rows: the sum over rows stays in the lane. A wave holds 64 keys of a key head in its MFMA operands
// and walks over the rows, 32 at a time, which come in whole cache lines, the next 32 in flight, and turn into the
// operand layout in a piece of LDS that only this wave uses (loaded in that layout, 16 rows to an instruction's quarter,
// they took 64 cycles an instruction: 512 tokens over 8704 keys 76 us). SPLIT: the four waves of a workgroup share
// 64 keys and take the row tiles in turn (many rows), else each has 64 keys of its own. One workgroup writes a key, in a
// fixed order: no atomics, the same bits every time.
template <bool H, int D, bool SPLIT>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void k_attn_weights(AttnArgs a, float* __restrict__ w, int add) {
  constexpr int KT = 2, ST = D / 16, CH = D / 8, RS = 64 / CH;  // RS: rows of a load of the wave
  __shared__ __align__(16) unsigned char qs[4][32 * D * 2];
  __shared__ __align__(16) float refs[4][32];
  __shared__ __align__(16) int nodes[4][32];
  __shared__ float red[4][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hf = lane >> 5;
  const int g = blockIdx.x % a.groups, rest = blockIdx.x / a.groups;
  const int tiles = (a.slots + 63) / 64, per = SPLIT ? tiles : (tiles + 3) / 4;
  // the last slots first: the nodes' own tiles take longest
  const int b = rest / per, kb = (SPLIT ? per - 1 - rest % per : (per - 1 - rest % per) * 4 + wave) * 64;
  const int pos = a.pos ? __builtin_amdgcn_readfirstlane(a.pos[b]) : a.pos0;
  const bool bad = pos < 0 || pos > a.slots - a.m;
  const int keys = bad ? 0 : pos + a.m;
  const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.mask_b : nullptr;
  float acc[KT] = {0.0f, 0.0f};
  if (kb < keys) {
    const uint16_t* kp = a.k + (int64_t)b * a.k_b + (int64_t)g * a.k_g;
    const auto kr = tile_rsrc(kp, a.k_s, kb, keys, 64, D);
    uint4 kf[KT][ST];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int s = 0; s < ST; ++s) kf[kt][s] = buf_ld128(kr, (uint32_t)((kt * 32 + r) * a.k_s + hf * 8 + s * 16) * 2u);
    const int step = SPLIT ? 4 : 1, tiles_r = (a.R + 31) / 32;
    // a chain's nodes before the tile's first key see none of it
    int rt = (mask ? 0 : max(0, kb - pos) * a.rep / 32) + (SPLIT ? wave : 0);
    // queries and lse of the group's first head; of the rows that this lane loads, (node, head of the group) and the
    // offset, which move on by 32 step rows
    const uint16_t* qg = a.q + (int64_t)b * a.q_b + (int64_t)(g * a.rep) * a.q_h;
    const float* lg = a.lse + (int64_t)b * a.m * a.heads + g * a.rep;
    const auto qr = buf_rsrc(qg, (uint32_t)((a.m - 1) * a.q_m + (a.rep - 1) * a.q_h + D) * 2u);
    const int dn = 32 * step / a.rep, dj = 32 * step % a.rep;
    const uint32_t qm = (uint32_t)a.q_m * 2u, qh = (uint32_t)a.q_h * 2u;
    int rj[ST];
    uint32_t ro[ST];
#pragma unroll
    for (int i = 0; i < ST; ++i) {
      const int row = rt * 32 + lane / CH + i * RS;
      rj[i] = row % a.rep;
      ro[i] = (uint32_t)(row / a.rep) * qm + (uint32_t)rj[i] * qh + (uint32_t)(lane % CH) * 16u;
    }
    int ln = (rt * 32 + r) / a.rep, lj = (rt * 32 + r) % a.rep;  // of row r, whose lse this lane loads
    int left = a.R - rt * 32 - lane / CH;                        // rows from this lane's first one on
    uint4 qv[ST];
    float lse;
    int node;
    auto load = [&] {
#pragma unroll
      for (int i = 0; i < ST; ++i) {
        // rows behind the last are zeros, not what lies there: another head's NaN would reach keys that it does not see
        qv[i] = buf_ld128(qr, i * RS < left ? ro[i] : 0xFFFFFF00u);
        rj[i] += dj;
        ro[i] += (uint32_t)dn * qm + (uint32_t)dj * qh;
        if (rj[i] >= a.rep) rj[i] -= a.rep, ro[i] += qm - (uint32_t)a.rep * qh;
      }
      left -= 32 * step;
      node = ln;
      lse = ln < a.m ? lg[(int64_t)ln * a.heads + lj] : -INFINITY;
      ln += dn, lj += dj;
      if (lj >= a.rep) lj -= a.rep, ++ln;
    };
    unsigned char* mine = qs[wave];
    auto q_at = [&](int row, int c) { return row * (2 * D) + (c ^ (D == 64 ? (row >> 1) & 7 : row & 15)) * 16; };
    if (rt < tiles_r) load();
    for (; rt < tiles_r; rt += step) {
#pragma unroll
      for (int i = 0; i < ST; ++i) *reinterpret_cast<uint4*>(mine + q_at(lane / CH + i * RS, lane % CH)) = qv[i];
      // rows behind the last, and rows that see nothing, add nothing, not even to a key whose score is no number
      const bool gaps = __any(lse == -INFINITY);
      if (hf == 0) refs[wave][r] = lse * 1.4426950408889634f;
      if (hf == 1) nodes[wave][r] = node;
      if (rt + step < tiles_r) load();
      fl_f32x16 s[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kt][i] = 0.0f;
#pragma unroll
      for (int e = 0; e < ST; ++e) {
        const uint4 qf = *reinterpret_cast<const uint4*>(mine + q_at(r, 2 * e + hf));
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[kt] = mma<H>(qf, kf[kt][e], s[kt]);
      }
      // s[kt][i]: row 8 (i / 4) + 4 hf + i % 4 of the tile, key 32 kt + r
      // all of the tile's keys are cached, or (a chain) no later than the rows' first node
      auto add_all = [&](auto with_gaps) {
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const fl_f32x4 ref = *reinterpret_cast<const fl_f32x4*>(&refs[wave][8 * q4 + 4 * hf]);
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][4 * q4 + i], a.sc, -ref[i]));
              if (decltype(with_gaps)::value) p[i] = ref[i] == -INFINITY ? 0.0f : p[i];
            }
            acc[kt] += (p[0] + p[1]) + (p[2] + p[3]);
          }
        }
      };
      if (kb + 64 <= pos || (!mask && kb + 63 - pos <= rt * 32 / a.rep)) {
        gaps ? add_all(std::true_type{}) : add_all(std::false_type{});
      } else {
        const auto mr = buf_rsrc(mask, mask ? (uint32_t)a.m * (uint32_t)a.m : 0u);
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const fl_f32x4 ref = *reinterpret_cast<const fl_f32x4*>(&refs[wave][8 * q4 + 4 * hf]);
          const int4 at = *reinterpret_cast<const int4*>(&nodes[wave][8 * q4 + 4 * hf]);
          const int t[4] = {at.x, at.y, at.z, at.w};
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const int j = kb + 32 * kt + r - pos;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][4 * q4 + i], a.sc, -ref[i]));
              const uint32_t off = j >= 0 && j < a.m && t[i] < a.m ? (uint32_t)t[i] * (uint32_t)a.m + (uint32_t)j : 0xFFFFFFF0u;
              const bool sees = mask ? __builtin_amdgcn_raw_buffer_load_b8(mr, off, 0, 0) != 0 : j <= t[i];
              // a key behind the end is a zero: no score of its own, and j <= t holds for no node
              acc[kt] += ref[i] != -INFINITY && (j < 0 || (sees && j < a.m)) ? p : 0.0f;
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const float v = xor32_sum(acc[kt]);
    if (hf == 0) red[wave][32 * kt + r] = v;
  }
  __syncthreads();
  float* row = w + ((int64_t)b * a.groups + g) * a.slots;
  auto put = [&](int slot, float v) {
    if (slot >= a.slots) return;
    if (bad) row[slot] = NAN;
    else if (!add) row[slot] = v;
    else if (slot < keys) row[slot] += v;
  };
  if (!SPLIT) put(kb + lane, red[wave][lane]);
  else if (tid < 64) put(kb + tid, (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]));
}

// ---- host -------------------------------------------------------------------------------------------------
constexpr int AT_NW = 8;      // waves of k_attn_few
constexpr int AT_FEW = 64;    // rows that it takes at most
constexpr int AT_PARTS = 64;  // key parts at most: a lane of the merge each

bool desc_ok(const fl_attn_desc* d) {
  if (!d || d->b < 1 || d->m < 1 || d->heads < 1 || d->groups < 1 || d->slots < 1 || d->slots > 1 << 30) return false;
  if (d->heads % d->groups || (d->dim != 64 && d->dim != 128) || d->m > d->slots) return false;
  if (d->b > 65536 || d->m > 32768 || d->heads > 4096 || (int64_t)d->m * (d->heads / d->groups) > (1 << 24)) return false;
  if (!(d->scale > 0.0f) || d->scale > 3.0e38f) return false;
  const int64_t st[] = {d->q_b, d->q_m, d->q_h, d->k_b, d->k_g, d->k_s, d->v_b, d->v_g, d->v_s};
  for (int64_t x : st)
    if (x < 0 || x % 8 || x > (int64_t)1 << 40) return false;
  // a tile of 64 slots, and a sequence's queries, within 32 bits
  return d->k_s <= 1 << 23 && d->v_s <= 1 << 23 && d->mask_b >= 0 &&
         (d->m - 1) * d->q_m + (d->heads - 1) * d->q_h + d->dim <= 1 << 30;
}
bool on16(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct AttnPlan {
  bool few;
  int blocks, parts, kpp;
  int64_t bytes;
};
// The plan for sequences of up to `keys` keys. Within a kind its parts grow with the keys, so the workspace for all that
// a cache can hold is the larger of the two kinds' (attn_work_bound).
AttnPlan attn_plan_of(const fl_attn_desc& d, int keys, bool few) {
  const int R = d.m * (d.heads / d.groups);
  AttnPlan p{};
  p.few = few;
  p.blocks = few ? (R + 31) / 32 : (R + 127) / 128;
  const int unit = few ? AT_NW * 4096 / d.dim : 64, least = few ? unit : 256;
  const int64_t base = (int64_t)d.b * d.groups * p.blocks;
  // Workgroups that cutting the keys may reach. Few rows: one per CU, whose eight waves have 128 KB in flight (131072 keys
  // 55 us, with two rounds of workgroups 62). Many rows: of the three (dim 64) or two that a CU holds, one and a third
  // times as many as there are places (1024 tokens behind 4096: 640 113 us, 1024 103, 1600 109; 16 trees of 13 and
  // 128 dims: 640 59, 1024 70).
  const int64_t fill = few ? 256 : d.dim == 64 ? 1024 : 640;
  // a wave of few rows takes three tiles in less than the launch that joins parts costs (1032 keys: 11.6 uncut, 13.5 in
  // two parts; 2000: 16.0 and 13.5)
  const int most = few && keys <= 3 * unit
                       ? 1
                       : (int)std::max<int64_t>(1, std::min<int64_t>({AT_PARTS, (fill + base - 1) / base, keys / least}));
  p.kpp = (int)(((int64_t)(keys + most - 1) / most + unit - 1) / unit * unit);
  p.parts = (keys - 1) / p.kpp + 1;
  p.bytes = most == 1 ? 0 : most * ((int64_t)d.b * d.groups * R) * (d.dim + 2) * 4;
  return p;
}
// `pos_known`: the host knows how many keys there are; else up to d.slots, and sequences of any length
AttnPlan attn_plan(const fl_attn_desc& d, bool pos_known) {
  const int R = d.m * (d.heads / d.groups), keys = pos_known ? d.pos0 + d.m : d.slots;
  // Few rows: a wave's own keys need no barrier but meet in LDS at the end, which pays where one launch does (up to three
  // tiles a wave) and where memory is the bound; in between the shared ring's kernel starts and ends sooner. us, one
  // token, few / many: 1000 keys 11.2 / 11.5, 2000 13.6 / 10.7, 8000 13.5 / 11.8, 131072 46 / 68; 24 sequences of 3000
  // 34 / 40, 8 trees of 8 behind 2000 17.0 / 18.6; 40 rows behind 4000 14.7 / 11.5, behind 30000 21.1 / 25.8.
  const bool few = R <= AT_FEW && (keys <= 3 * AT_NW * 4096 / d.dim || (int64_t)d.b * d.groups * keys * d.dim >= 6 << 20);
  return attn_plan_of(d, keys, few);
}
AttnArgs attn_args(const fl_attn_desc& d, const uint16_t* q, const uint16_t* k, const uint16_t* v, const int32_t* pos,
                   const uint8_t* mask) {
  AttnArgs a{};
  a.q = q, a.k = k, a.v = v, a.pos = pos, a.mask = mask;
  a.b = d.b, a.m = d.m, a.heads = d.heads, a.groups = d.groups, a.rep = d.heads / d.groups, a.slots = d.slots;
  a.pos0 = d.pos0, a.R = d.m * a.rep;
  a.blocks = a.parts = 1, a.kpp = INT32_MAX;
  a.sc = d.scale * 1.4426950408889634f;
  a.q_b = d.q_b, a.q_m = d.q_m, a.q_h = d.q_h, a.k_b = d.k_b, a.k_g = d.k_g, a.k_s = d.k_s;
  a.v_b = d.v_b, a.v_g = d.v_g, a.v_s = d.v_s, a.mask_b = d.mask_b;
  return a;
}

// one launch holds fewer than 2^32 threads
bool launchable(int64_t wgs, int threads) { return wgs * threads <= (int64_t)UINT32_MAX; }

template <bool H, int D>
int attn_launch(AttnArgs a, const AttnPlan& p, hipStream_t s) {
  const int64_t wgs = (int64_t)a.b * a.groups * p.blocks * p.parts;
  if (!launchable(wgs, p.few ? 64 * AT_NW : 256)) return FL_E_ARG;
  const dim3 grid((uint32_t)wgs);
  if (!p.few) hipLaunchKernelGGL((k_attn_many<H, D>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_attn_few<H, D, AT_NW>), grid, dim3(64 * AT_NW), 0, s, a);
  if (p.parts > 1) {
    hipLaunchKernelGGL((k_attn_merge<H, D>), dim3((a.R + 3) / 4, a.b * a.groups), dim3(256), 0, s, a);
  }
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}
template <bool H, int D>
int weights_launch(AttnArgs a, float* w, int add, hipStream_t s) {
  const bool split = a.R > 32;
  const int tiles = (a.slots + 63) / 64, per = split ? tiles : (tiles + 3) / 4;
  const int64_t wgs = (int64_t)a.b * a.groups * per;
  if (!launchable(wgs, 256)) return FL_E_ARG;
  if (split) hipLaunchKernelGGL((k_attn_weights<H, D, true>), dim3((uint32_t)wgs), dim3(256), 0, s, a, w, add);
  else hipLaunchKernelGGL((k_attn_weights<H, D, false>), dim3((uint32_t)wgs), dim3(256), 0, s, a, w, add);
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}

}  // namespace

int64_t fl_attn_work_bound(const fl_attn_desc& d) {
  if (!desc_ok(&d)) return -1;
  const int64_t few = d.m * (d.heads / d.groups) <= AT_FEW ? attn_plan_of(d, d.slots, true).bytes : 0;
  return std::max(few, attn_plan_of(d, d.slots, false).bytes);
}

extern "C" {

int fl_tree_attention_workspace(const fl_attn_desc* d, int32_t pos_known, int64_t* bytes) {
  if (!desc_ok(d) || !bytes) return FL_E_ARG;
  if (pos_known && (d->pos0 < 0 || d->pos0 > d->slots - d->m)) return FL_E_POS;
  *bytes = attn_plan(*d, pos_known != 0).bytes;
  return FL_OK;
}

int fl_tree_attention(const fl_attn_desc* d, const uint16_t* q, const uint16_t* k, const uint16_t* v, const int32_t* pos,
                      const uint8_t* mask, uint16_t* out, float* lse, void* work, void* stream) {
  if (!desc_ok(d) || !on16(q) || !on16(k) || !on16(v) || !on16(out)) return FL_E_ARG;
  if (!pos && (d->pos0 < 0 || d->pos0 > d->slots - d->m)) return FL_E_POS;
  const AttnPlan p = attn_plan(*d, pos == nullptr);
  if (p.bytes && !on16(work)) return FL_E_ARG;
  AttnArgs a = attn_args(*d, q, k, v, pos, mask);
  a.out = out, a.lse = lse, a.part = static_cast<float*>(work), a.blocks = p.blocks, a.parts = p.parts, a.kpp = p.kpp;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (d->dim == 64) return d->fp16 ? attn_launch<true, 64>(a, p, s) : attn_launch<false, 64>(a, p, s);
  return d->fp16 ? attn_launch<true, 128>(a, p, s) : attn_launch<false, 128>(a, p, s);
}

int fl_attention_weights(const fl_attn_desc* d, const uint16_t* q, const uint16_t* k, const float* lse, const int32_t* pos,
                         const uint8_t* mask, float* weights, int32_t add, void* stream) {
  if (!desc_ok(d) || !on16(q) || !on16(k) || !lse || !weights) return FL_E_ARG;
  if (!pos && (d->pos0 < 0 || d->pos0 > d->slots - d->m)) return FL_E_POS;
  AttnArgs a = attn_args(*d, q, k, nullptr, pos, mask);
  a.lse = const_cast<float*>(lse);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (d->dim == 64) return d->fp16 ? weights_launch<true, 64>(a, weights, add, s) : weights_launch<false, 64>(a, weights, add, s);
  return d->fp16 ? weights_launch<true, 128>(a, weights, add, s) : weights_launch<false, 128>(a, weights, add, s);
}

}  // extern "C"
