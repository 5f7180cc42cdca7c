// Eviction from a K/V cache by the weight that its keys have gathered: which slots of each head stay (k_evict_select)
// and the move of their rows (k_evict_gather into another cache, k_evict_move in place).
#include <algorithm>
#include "fl_common.h"

namespace {

struct EvictArgs {
  unsigned char *k, *v;          // source (and destination in place)
  float* w;
  unsigned char *ko, *vo;        // destination of k_evict_gather
  float* wo;
  int32_t* kept;                 // [heads][keep]
  int n0, n1;                    // heads = n0 * n1
  int slots, slots_out, n, keep, recent, sink, rb;  // rb: bytes of a row
  // bytes between heads (outer, inner) and rows; w and wo are [heads][slots]
  int64_t k0, k1, ks, v0, v1, vs, ko0, ko1, kos, vo0, vo1, vos;
};

constexpr int ES_NT = 1024, ES_NW = ES_NT / FL_WAVE;

// ordered key of a weight: larger weight <-> larger key, a NaN above all, -0 as 0. Keys 0 (no slot) and 2^32 - 1 (a
// slot that always stays) are free.
__device__ __forceinline__ uint32_t w_key(float w) {
  if (w != w) return 0xFFFFFFFEu;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One workgroup per head. The `keep` largest keys by a radix select over 32 bits (four counts of 256 bins), ties to the
// lower slot, the first `sink` and the last `recent` slots above all others; then the kept slots in order: each wave has
// a contiguous piece of the slots, whose counts above the border it has from its own histograms, and places by ballots.
// The counts end where a bin's keys all stay. A lane holds its E keys in registers; E = 0: more slots, read again for
// every walk, eight loads in flight. Bound by the walks, two to four counts and the places, at some 24 clocks of the CU
// for 64 keys (with four counts and a walk for the sums above: 8192 slots of 8 heads 11.9 us with the move of 1024
// rows, now 10.8; 131072 of 2 heads 145, now 99).
template <int E>
__global__ __launch_bounds__(ES_NT) void k_evict_select(EvictArgs a) {
  constexpr int U = 8;
  __shared__ __align__(16) int hist[ES_NW][256];
  __shared__ int sum[256], sel[2], above_w[ES_NW], equal_w[ES_NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, head = blockIdx.x;
  const float* w = a.w + (int64_t)head * a.slots;
  int32_t* kept = a.kept + (int64_t)head * a.keep;
  const int piece = ((a.n + ES_NW - 1) / ES_NW + 63) / 64 * 64, p0 = min(a.n, wave * piece), p1 = min(a.n, p0 + piece);
  auto key_of = [&](int i, float x) -> uint32_t {
    return i >= p1 ? 0u : i < a.sink || i >= a.n - a.recent ? 0xFFFFFFFFu : w_key(x);
  };
  uint32_t held[E ? E : 1];
  if constexpr (E > 0) {
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = p0 + e * 64 + lane < p1 ? w[p0 + e * 64 + lane] : 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) held[e] = key_of(p0 + e * 64 + lane, x[e]);
  }
  // f(slot, key): every lane of the wave, for every slot of its piece, in order
  auto walk = [&](auto f) {
    if constexpr (E > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) f(p0 + e * 64 + lane, held[e]);
    } else {
      for (int i0 = p0; i0 < p1; i0 += 64 * U) {
        float x[U];
#pragma unroll
        for (int e = 0; e < U; ++e) x[e] = i0 + e * 64 + lane < p1 ? w[i0 + e * 64 + lane] : 0.0f;
#pragma unroll
        for (int e = 0; e < U; ++e) f(i0 + e * 64 + lane, key_of(i0 + e * 64 + lane, x[e]));
      }
    }
  };
  uint32_t prefix = 0;
  int need = a.keep;  // of those with the prefix so far (no slot's key 0 lies below all: never reached)
  int above = 0;      // this lane's part of the wave's keys above the prefix, from the wave's own counts
  int shift = 32;
  bool all = false;  // the rest of the bits do not matter: every key with the prefix stays
  while (shift > 0 && !all) {
    shift -= 8;
    // a wave's counts are its own until they are summed: no barrier between these and those
    *reinterpret_cast<int4*>(&hist[wave][4 * lane]) = make_int4(0, 0, 0, 0);
    __builtin_amdgcn_wave_barrier();
    if (shift == 24)
      walk([&](int, uint32_t key) {
        if (key) atomicAdd(&hist[wave][key >> 24], 1);  // no slot: 64 lanes at one address take 64 turns
      });
    else
      walk([&](int, uint32_t key) {
        if ((key >> (shift + 8)) == prefix) atomicAdd(&hist[wave][(key >> shift) & 255], 1);
      });
    __syncthreads();
    if (tid < 256) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < ES_NW; ++i) n += hist[i][tid];
      sum[tid] = n;
    }
    __syncthreads();
    int higher = 0;
    const int bin = select_bin(sum, need, &higher, sel);
    prefix = (prefix << 8) | (uint32_t)bin;
    need -= higher;
    all = sum[bin] == need && prefix != 0;  // a prefix of 0 is also that of no slot
    const int4 c = *reinterpret_cast<const int4*>(&hist[wave][4 * lane]);
    above += (4 * lane > bin ? c.x : 0) + (4 * lane + 1 > bin ? c.y : 0) + (4 * lane + 2 > bin ? c.z : 0) + (4 * lane + 3 > bin ? c.w : 0);
    if (lane == 0) equal_w[wave] = hist[wave][bin];  // of the last turn
  }
  if constexpr (E > 0) {
    above = (int)wave_sum((float)above);  // at most 64 E
  } else {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) above += __shfl_xor(above, o, 64);
  }
  if (lane == 0) above_w[wave] = above;
  __syncthreads();
  int eq = 0, at = 0;  // equal ones before this wave, and the kept ones
  for (int i = 0; i < wave; ++i) {
    at += above_w[i] + min(equal_w[i], max(0, need - eq));
    eq += equal_w[i];
  }
  // slots that always stay are no more than `keep`: a border among them is all of them, and no key is above it
  const uint32_t least = prefix + (all ? 0u : 1u);
  auto before = [](unsigned long long m) { return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u)); };
  walk([&](int i, uint32_t key) {
    const uint32_t top = key >> shift;
    unsigned long long s = __ballot(top >= least);
    if (!all) {
      const unsigned long long e = __ballot(top == prefix);
      if (e) {
        s |= e & __ballot(eq + before(e) < need);
        eq += __popcll(e);
      }
    }
    if ((s >> lane) & 1) kept[at + before(s)] = i;
    at += __popcll(s);
  });
}

__device__ __forceinline__ int64_t head_at(int head, int n1, int64_t s0, int64_t s1) {
  return (int64_t)(head / n1) * s0 + (int64_t)(head % n1) * s1;
}

// Rows into another cache: 16 bytes a thread, K and V of a row by the same thread.
__global__ __launch_bounds__(256) void k_evict_gather(EvictArgs a) {
  const int per = a.rb / 16, head = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.keep * per) return;
  const int j = (int)(i / per), c = (int)(i % per) * 16;
  const int64_t src = a.kept[(int64_t)head * a.keep + j];
  const uint4 x = *reinterpret_cast<const uint4*>(a.k + head_at(head, a.n1, a.k0, a.k1) + src * a.ks + c);
  const uint4 y = *reinterpret_cast<const uint4*>(a.v + head_at(head, a.n1, a.v0, a.v1) + src * a.vs + c);
  *reinterpret_cast<uint4*>(a.ko + head_at(head, a.n1, a.ko0, a.ko1) + (int64_t)j * a.kos + c) = x;
  *reinterpret_cast<uint4*>(a.vo + head_at(head, a.n1, a.vo0, a.vo1) + (int64_t)j * a.vos + c) = y;
  if (c == 0 && a.wo) a.wo[(int64_t)head * a.slots_out + j] = a.w[(int64_t)head * a.slots + src];
}

// In place: a workgroup takes a head's K rows, its V rows or its weights, in order, a batch at a time. A kept row never
// moves up (kept[j] >= j), so what a later batch reads lies above all that the earlier ones write: the only wait is
// for a batch's own reads before its writes.
__global__ __launch_bounds__(256) void k_evict_move(EvictArgs a) {
  constexpr int U = 8;
  const int tid = threadIdx.x, head = blockIdx.x, kind = blockIdx.y;  // 0: K, 1: V, 2: weights
  const int32_t* kept = a.kept + (int64_t)head * a.keep;
  if (kind == 2) {
    float* w = a.w + (int64_t)head * a.slots;
    for (int j0 = 0; j0 < a.keep; j0 += 256 * U) {
      float x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * 256 + tid;
        x[u] = j < a.keep ? w[kept[j]] : 0.0f;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * 256 + tid;
        if (j < a.keep) w[j] = x[u];
      }
    }
    __syncthreads();
    for (int j = a.keep + tid; j < a.n; j += 256) w[j] = 0.0f;
    return;
  }
  unsigned char* base = kind == 0 ? a.k + head_at(head, a.n1, a.k0, a.k1) : a.v + head_at(head, a.n1, a.v0, a.v1);
  const int64_t stride = kind == 0 ? a.ks : a.vs;
  const int per = a.rb / 16, rows = 256 / per;  // rows of a sweep of the workgroup
  const int c = tid % per * 16, r = tid / per;
  for (int j0 = 0; j0 < a.keep; j0 += rows * U) {
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * rows + r;
      x[u] = r < rows && j < a.keep ? *reinterpret_cast<const uint4*>(base + (int64_t)kept[j] * stride + c) : make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * rows + r;
      if (r < rows && j < a.keep) *reinterpret_cast<uint4*>(base + (int64_t)j * stride + c) = x[u];
    }
  }
}

bool strides_ok(const fl_rows* r, int32_t rb) {
  if (!r || !r->data || (reinterpret_cast<uintptr_t>(r->data) & 15)) return false;
  return r->outer >= 0 && r->inner >= 0 && r->row >= rb && !(r->outer % 16) && !(r->inner % 16) && !(r->row % 16);
}

}  // namespace

extern "C" {

int fl_evict(const fl_rows* k, const fl_rows* v, float* weights, int32_t n_outer, int32_t n_inner, int32_t slots,
             int32_t row_bytes, int32_t n, int32_t keep, int32_t recent, int32_t sink, int32_t* kept, const fl_rows* k_out,
             const fl_rows* v_out, float* weights_out, int32_t slots_out, void* stream) {
  if (!weights || !kept || n_outer < 1 || n_inner < 1 || (int64_t)n_outer * n_inner > 65535) return FL_E_ARG;
  if (row_bytes < 16 || row_bytes > 4096 || row_bytes % 16 || !strides_ok(k, row_bytes) || !strides_ok(v, row_bytes)) return FL_E_ARG;
  if (n < 1 || slots < n || slots > 1 << 30 || keep < 1 || keep > n || recent < 0 || sink < 0 || (int64_t)recent + sink > keep) return FL_E_ARG;
  if (!k_out != !v_out || (weights_out && !k_out)) return FL_E_ARG;
  // heads that share their rows can be read, not written
  auto apart = [&](const fl_rows* r) { return (n_outer == 1 || r->outer != 0) && (n_inner == 1 || r->inner != 0); };
  const fl_rows *kd = k_out ? k_out : k, *vd = v_out ? v_out : v;
  if (!apart(kd) || !apart(vd) || kd->data == vd->data) return FL_E_ARG;
  if (k_out && (!strides_ok(k_out, row_bytes) || !strides_ok(v_out, row_bytes) || slots_out < keep)) return FL_E_ARG;
  if (k_out && (int64_t)keep * (row_bytes / 16) > (int64_t)UINT32_MAX - 255) return FL_E_ARG;  // threads of a launch
  const int heads = n_outer * n_inner;
  EvictArgs a{};
  a.k = static_cast<unsigned char*>(k->data), a.v = static_cast<unsigned char*>(v->data), a.w = weights, a.kept = kept;
  a.n0 = n_outer, a.n1 = n_inner, a.slots = slots, a.slots_out = slots_out, a.n = n, a.keep = keep, a.recent = recent, a.sink = sink;
  a.rb = row_bytes;
  a.k0 = k->outer, a.k1 = k->inner, a.ks = k->row, a.v0 = v->outer, a.v1 = v->inner, a.vs = v->row;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int per = ((n + ES_NW - 1) / ES_NW + 63) / 64;  // slots of a lane
  if (per <= 2) hipLaunchKernelGGL(k_evict_select<2>, dim3(heads), dim3(ES_NT), 0, s, a);
  else if (per <= 8) hipLaunchKernelGGL(k_evict_select<8>, dim3(heads), dim3(ES_NT), 0, s, a);
  else if (per <= 16) hipLaunchKernelGGL(k_evict_select<16>, dim3(heads), dim3(ES_NT), 0, s, a);
  else if (per <= 32) hipLaunchKernelGGL(k_evict_select<32>, dim3(heads), dim3(ES_NT), 0, s, a);
  // held, a lane's 48 keys leave room for one workgroup a CU: 40000 slots of 2 heads 27 us, read again 37; of 320 heads 191
  // and 187 (64 keys spill)
  else if (per <= 48 && heads <= 256) hipLaunchKernelGGL(k_evict_select<48>, dim3(heads), dim3(ES_NT), 0, s, a);
  else hipLaunchKernelGGL(k_evict_select<0>, dim3(heads), dim3(ES_NT), 0, s, a);
  if (k_out) {
    a.ko = static_cast<unsigned char*>(k_out->data), a.vo = static_cast<unsigned char*>(v_out->data), a.wo = weights_out;
    a.ko0 = k_out->outer, a.ko1 = k_out->inner, a.kos = k_out->row, a.vo0 = v_out->outer, a.vo1 = v_out->inner, a.vos = v_out->row;
    const int64_t threads = (int64_t)keep * (row_bytes / 16);
    hipLaunchKernelGGL(k_evict_gather, dim3((uint32_t)((threads + 255) / 256), heads), dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL(k_evict_move, dim3(heads, 3), dim3(256), 0, s, a);
  }
  return hipGetLastError() == hipSuccess ? FL_OK : FL_E_LAUNCH;
}

}  // extern "C"
