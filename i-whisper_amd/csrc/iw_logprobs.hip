// Token scores of rows of logits: the log-probability of a given token, the
// entropy and the most probable alternatives.
//
// With m the row's largest logit and the sums over every token but one that holds it,
//   Z' = sum exp((x - m) s),  U' = sum (m - x) s exp((x - m) s),
//   lse = m s + log1p(Z'),  entropy = log1p(Z') + U' / (1 + Z'):
// both terms are positive and keep their digits where one token holds nearly
// all of the probability. Alternatives are ordered by value, then by index.
//
// A block of 1024 threads holds its part of a row in registers: the logits
// are read once. The maxima of 64 groups of its threads meet in LDS, which
// gives every wave m and a bound that at least `top` logits reach; the sums
// and the few logits that reach the bound follow, and each of those finds
// its place by counting the larger ones.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

#include "iw_common.hpp"
#include "iw_tree.hpp"

namespace iw {

namespace {

constexpr int NT = 1024, NW = NT / 64;
constexpr int kPieces = 4096;  // 16-byte pieces of a block's part
constexpr int kCand = 1024;    // candidates that the bound may leave
constexpr int kMaxParts = 1024;  // parts of a row

// One block's part of a row: its largest logit, Z' and U' (in units of s)
struct Part {
  float m, z, u, pad;
};

// A logit and its column as one whole number: larger logits first, then lower
// columns; both zeros are one value and a NaN is the largest.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  if (v != v) return 0xffffffffu;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float v, int col) {
  return ((uint64_t)ordered(v) << 32) | (uint32_t)~col;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int key_col(uint64_t k) { return (int)~(uint32_t)k; }

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = max64(v, __shfl_xor(v, o));
  return v;
}

// Sum over the wave, in every lane (DPP moves within 16 lanes, then their four sums)
__device__ __forceinline__ float wave_sum_f32(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __uint_as_float(
        (uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});
  v += dpp(v, std::integral_constant<int, 0x4E>{});
  v += dpp(v, std::integral_constant<int, 0x141>{});
  v += dpp(v, std::integral_constant<int, 0x140>{});
  const int b = (int)__float_as_uint(v);
  auto at = [&](int l) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane(b, l)); };
  return (at(0) + at(16)) + (at(32) + at(48));
}

__device__ __forceinline__ bool suppressed(const uint32_t *words, int col) {
  return words && ((words[col >> 5] >> (col & 31)) & 1u);
}

// The types. A piece is 16 bytes of logits; `off` has the bits of its
// suppressed ones. Threshold values are 32-bit numbers in the order of the
// logits, of which `rank_bits` from the top are looked at.
template <typename T>
struct Logit;

template <>
struct Logit<int8_t> {
  static constexpr int E = 16;
  static __device__ __forceinline__ float one(const int8_t *p) { return (float)*p; }
  static __device__ __forceinline__ float get(const uint4 &w, int i) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    return (float)(int8_t)(v[i >> 2] >> (8 * (i & 3)));
  }
};
template <>
struct Logit<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ float one(const float *p) { return *p; }
  static __device__ __forceinline__ float get(const uint4 &w, int i) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    return __uint_as_float(v[i]);
  }
  static __device__ __forceinline__ void mask(uint4 &w, uint32_t off) {
    uint32_t *v = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((off >> i) & 1u) v[i] = 0xff800000u;
  }
};
template <uint32_t INF>
struct Half {
  static constexpr int E = 8;
  static __device__ __forceinline__ void mask(uint4 &w, uint32_t off) {
    uint32_t *v = &w.x;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((off >> i) & 1u) v[i >> 1] = (i & 1) ? (v[i >> 1] & 0xffffu) | INF << 16 : (v[i >> 1] & 0xffff0000u) | INF;
  }
};
template <>
struct Logit<__hip_bfloat16> : Half<0xff80u> {
  static __device__ __forceinline__ float one(const __hip_bfloat16 *p) {
    return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(p) << 16);
  }
  static __device__ __forceinline__ float get(const uint4 &w, int i) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    return __uint_as_float((i & 1) ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
  }
};
template <>
struct Logit<__half> : Half<0xfc00u> {
  static __device__ __forceinline__ float one(const __half *p) { return __half2float(*p); }
  static __device__ __forceinline__ float get(const uint4 &w, int i) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    return __half2float(__ushort_as_half((uint16_t)(v[i >> 1] >> (16 * (i & 1)))));
  }
};

// The k-th largest of the 64 lanes' numbers, of which the top `bits` are
// looked at: a bound that at least k of them reach.
template <int BITS>
__device__ __forceinline__ uint32_t kth_largest(uint32_t v, int k) {
  uint32_t p = 0;
#pragma unroll
  for (int b = 31; b > 31 - BITS; --b) {
    const uint32_t c = p | (1u << b);
    if (__popcll(__ballot(v >= c)) >= k) p = c;
  }
  return p;
}

struct Shared {
  uint32_t group[64];
  float z[NW], u[NW], n[NW];
  float e[256];  // int8: exp(-y s) of the distances y from m
  int cands;
  uint64_t best[NW];
  uint64_t cand[kCand];
  uint64_t top[kScoreMaxTop];
};

// The top alternatives of a block's part one after the other, each the largest
// key below the last: for rows whose bound leaves too many candidates (whole
// rows of ties) or too few (suppressed tokens among the alternatives, NaN).
template <typename T>
__device__ __noinline__ void top_by_rounds(const T *x, int c0, int n, const uint32_t *suppress, int top, Shared &s) {
  uint64_t prev = ~0ull;
  for (int i = 0; i < top; ++i) {
    uint64_t k = 0;
    for (int c = threadIdx.x; c < n; c += NT) {
      const uint64_t q = key_of(suppressed(suppress, c0 + c) ? -INFINITY : Logit<T>::one(x + c), c0 + c);
      if (q < prev) k = max64(k, q);
    }
    k = wave_max64(k);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.best[threadIdx.x >> 6] = k;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) k = max64(k, s.best[w]);
    if (threadIdx.x == 0) s.top[i] = k;  // 0: the part has no more logits
    prev = k;
  }
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ void write_row(const ScoreArgs &a, int64_t row, float m, float l, float z, float u) {
  if (a.logprob) {
    const int64_t at = a.targets[row];
    float lp = __uint_as_float(0x7fc00000u);  // a token outside the vocabulary has none
    if (at >= 0 && at < a.cols) {
      const float v = suppressed(a.suppress, (int)at) ? -INFINITY
                                                      : Logit<T>::one(reinterpret_cast<const T *>(a.x) + row * a.ld + at);
      lp = (v - m) * a.scale - l;
    }
    a.logprob[row] = lp;
  }
  if (a.entropy) a.entropy[row] = l + u * a.scale / (1.f + z);
}

// log1p(Z'), NaN where the row has no finite maximum (all suppressed, an infinity, a NaN)
__device__ __forceinline__ float row_log(float m, float z) { return log1pf(z) + (m - m); }

template <typename T>
__global__ __launch_bounds__(NT) void token_scores_kernel(ScoreArgs a, int chunks, int span) {
  using L = Logit<T>;
  constexpr bool I8 = std::is_same<T, int8_t>::value;
  constexpr int E = L::E, P = kPieces / NT;
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / chunks;
  const int chunk = blockIdx.x % chunks;
  const int c0 = chunk * span, n = min(a.cols - c0, span);  // this block's columns
  const T *x = reinterpret_cast<const T *>(a.x) + row * a.ld + c0;
  // whole 16-byte pieces, and up to 2 (E - 1) logits before and behind them
  const int head = min((int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)), n);
  const int pieces = (n - head) / E, tail0 = head + pieces * E;
  const uint4 *xa = reinterpret_cast<const uint4 *>(x + head);
  uint4 w[P];
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (p * NT + tid < pieces) w[p] = xa[p * NT + tid];
  const int extra = tid < head ? tid : tail0 + tid - head;  // this thread's single logit
  bool has_extra = extra < n;
  float xe = has_extra ? L::one(x + extra) : -INFINITY;
  if (has_extra && suppressed(a.suppress, c0 + extra)) {
    xe = -INFINITY;
    if (I8) has_extra = false;
  }
  uint32_t off[I8 ? P : 1];  // int8 has no -inf: its suppressed logits stay bits
#pragma unroll
  for (int p = 0; p < (I8 ? P : 1); ++p) off[p] = 0;
  if (a.suppress) {
    const int last = (a.cols - 1) >> 5;
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (p * NT + tid < pieces) {
        const int col0 = c0 + head + (p * NT + tid) * E;
        const uint64_t two = (uint64_t)a.suppress[min((col0 >> 5) + 1, last)] << 32 | a.suppress[col0 >> 5];
        const uint32_t bits = (uint32_t)(two >> (col0 & 31)) & ((1u << E) - 1u);
        if constexpr (I8)
          off[p] = bits;
        else
          L::mask(w[p], bits);
      }
  }

  // ---- the thread's largest logit (int8: -129 for none) ----
  float tmax = -INFINITY;
  if constexpr (I8) {
    typedef int16_t v2s __attribute__((ext_vector_type(2)));
    v2s hi{-32768, -32768}, lo{-32768, -32768};
    bool any = has_extra;
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (p * NT + tid < pieces) {
        uint32_t v[4] = {w[p].x, w[p].y, w[p].z, w[p].w};
        any = any || off[p] != 0xffffu;
        if (off[p]) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if ((off[p] >> i) & 1u) v[i >> 2] = (v[i >> 2] & ~(0xffu << (8 * (i & 3)))) | 0x80u << (8 * (i & 3));
        }
        // the odd bytes lead their 16-bit halves, the even ones once shifted up
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          hi = __builtin_elementwise_max(hi, __builtin_bit_cast(v2s, v[q]));
          lo = __builtin_elementwise_max(lo, __builtin_bit_cast(v2s, v[q]) << (int16_t)8);
        }
      }
    int32_t t = max(max(hi.x >> 8, hi.y >> 8), max(lo.x >> 8, lo.y >> 8));
    if (has_extra) t = max(t, (int32_t)xe);
    tmax = any ? (float)t : -129.f;
  } else {
    tmax = xe;
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (p * NT + tid < pieces) {
#pragma unroll
        for (int e = 0; e < E; ++e) tmax = fmaxf(tmax, L::get(w[p], e));
      }
  }
  // numbers in the logits' order, the largest of each 16 threads
  uint32_t g = I8 ? (uint32_t)(int32_t)(tmax + 129.f) << 23 : ordered(tmax);
  g = max(g, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)g, 0xB1, 0xf, 0xf, true));
  g = max(g, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)g, 0x4E, 0xf, 0xf, true));
  g = max(g, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)g, 0x141, 0xf, 0xf, true));
  g = max(g, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)g, 0x140, 0xf, 0xf, true));
  if ((lane & 15) == 0) s.group[tid >> 4] = g;
  if (tid == 0) s.cands = 0;
  __syncthreads();
  g = s.group[lane];
  const uint32_t bound = a.top > 0 ? kth_largest<I8 ? 9 : 16>(g, a.top) : 0u;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) g = max(g, (uint32_t)__shfl_xor((int)g, o));
  const float m = I8 ? (g == 0 ? -INFINITY : (float)((int)(g >> 23) - 129)) : key_value((uint64_t)g << 32);
  const float ms = m == -INFINITY ? 0.f : m;  // a part without finite logits sums to 0

  // ---- Z', U' / s and the number of logits that equal m ----
  float z = 0.f, u = 0.f, eq = 0.f;
  const bool mine = tmax == m;  // few threads hold it and look for it
  if constexpr (I8) {
    // exp by a table over the distances y = m - x; 255 stands for a suppressed
    // logit (below m = 127 no other has it)
    if (tid < 256) s.e[tid] = tid == 0 || (tid == 255 && m < 127.f) ? 0.f : expf(-(float)tid * a.scale);
    __syncthreads();
    const uint32_t m4 = (uint32_t)((int)ms + 128) * 0x01010101u;
    const bool clash = a.suppress && m == 127.f;
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (p * NT + tid < pieces) {
        const uint32_t v[4] = {w[p].x, w[p].y, w[p].z, w[p].w};
        if (!clash) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t y = m4 - (v[q] ^ 0x80808080u);
            if (off[p]) {
              const uint32_t o4 = ((((off[p] >> (4 * q)) & 15u) * 0x00204081u) & 0x01010101u) * 0xffu;
              // bytes of suppressed logits may lie above m: without borrows
              y = (m4 - ((v[q] ^ 0x80808080u) & ~o4)) | o4;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t d = (y >> (8 * i)) & 0xffu;
              const float e = s.e[d];
              z += e;
              u += e * (float)d;
              if (mine && d == 0) eq += 1.f;
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!((off[p] >> i) & 1u)) {
              const int d = 127 - (int)(int8_t)(v[i >> 2] >> (8 * (i & 3)));
              const float e = s.e[d];
              z += e;
              u += e * (float)d;
              if (d == 0) eq += 1.f;
            }
        }
      }
    if (has_extra) {
      const int d = (int)ms - (int)xe;
      const float e = s.e[d];
      z += e;
      u += e * (float)d;
      if (d == 0) eq += 1.f;
    }
  } else {
    // d * log2(e) s in two parts, as the product's rounding would be the same for all
    const double cd = (double)a.scale * 1.4426950408889634;
    const float ch = (float)cd, cl = (float)(cd - (double)ch);
    auto add = [&](float v, bool all) {
      const float d = v - ms;
      const float e = __builtin_amdgcn_exp2f(fmaf(d, ch, d * cl));
      if (all || d != 0.f) {
        z += e;
        u -= e > 0.f ? d * e : 0.f;
      } else {
        eq += 1.f;
      }
    };
    if (has_extra) add(xe, false);
    if (mine) {
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (p * NT + tid < pieces)
#pragma unroll
          for (int e = 0; e < E; ++e) add(L::get(w[p], e), false);
    } else {
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (p * NT + tid < pieces)
#pragma unroll
          for (int e = 0; e < E; ++e) add(L::get(w[p], e), true);
    }
  }

  // ---- the logits that reach the bound ----
  float reach = I8 ? (float)((int)(bound >> 23) - 129) : key_value((uint64_t)bound << 32);
  if (reach != reach) reach = -INFINITY;  // below every number: all logits
  if (a.top > 0 && tmax >= reach) {
    auto put = [&](float v, int col) {
      if (v >= reach) {
        const int at = atomicAdd(&s.cands, 1);
        if (at < kCand) s.cand[at] = key_of(v, col);
      }
    };
    if (has_extra) put(xe, c0 + extra);
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (p * NT + tid < pieces)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!I8 || !((off[I8 ? p : 0] >> e) & 1u)) put(L::get(w[p], e), c0 + head + (p * NT + tid) * E + e);
  }
  z = wave_sum_f32(z);
  u = wave_sum_f32(u);
  eq = wave_sum_f32(eq);
  if (lane == 0) s.z[wave] = z, s.u[wave] = u, s.n[wave] = eq;
  __syncthreads();
  z = u = eq = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) z += s.z[i], u += s.u[i], eq += s.n[i];
  if (eq > 0.f) z += eq - 1.f;
  const float l = row_log(m, z);

  const int cands = s.cands;
  const bool rounds = a.top > 0 && (cands > kCand || cands < min(a.top, n) || z != z || m - m != 0.f);
  if (rounds) top_by_rounds<T>(x, c0, n, a.suppress, a.top, s);
  uint64_t *tops = nullptr;
  if (chunks > 1)
    tops = reinterpret_cast<uint64_t *>(reinterpret_cast<Part *>(a.workspace) + a.rows * chunks) + (int64_t)blockIdx.x * a.top;
  auto place = [&](int at, uint64_t k) {
    if (tops) {
      tops[at] = k;
    } else {
      a.top_ids[row * a.top + at] = key_col(k);
      a.top_lp[row * a.top + at] = (key_value(k) - m) * a.scale - l;
    }
  };
  if (rounds) {
    if (tid < a.top) place(tid, s.top[tid]);
  } else if (tid < cands) {
    const uint64_t k = s.cand[tid];
    int larger = 0;
    for (int i = 0; i < cands; ++i) larger += s.cand[i] > k;
    if (larger < a.top) place(larger, k);
  } else if (tops && tid >= NT - 64 && cands + tid - (NT - 64) < a.top) {
    tops[cands + tid - (NT - 64)] = 0;  // a part of fewer logits than alternatives
  }
  if (tid != 0) return;
  if (tops)
    reinterpret_cast<Part *>(a.workspace)[blockIdx.x] = Part{m, z, u, 0.f};
  else
    write_row<T>(a, row, m, l, z, u);
}

// Joins a row's parts, one wave per row.
template <typename T>
__global__ __launch_bounds__(64) void token_scores_join_kernel(ScoreArgs a, int chunks) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const Part *parts = reinterpret_cast<const Part *>(a.workspace) + row * chunks;
  const uint64_t *tops =
      reinterpret_cast<const uint64_t *>(reinterpret_cast<const Part *>(a.workspace) + a.rows * chunks) +
      row * chunks * a.top;
  // the first part that holds the largest logit keeps it out of Z'
  uint64_t best = 0;
  for (int c = lane; c < chunks; c += 64) best = max64(best, key_of(parts[c].m, c));
  best = wave_max64(best);
  const float m = key_value(best), ms = m == -INFINITY ? 0.f : m;
  float z = 0.f, u = 0.f;
  for (int c = lane; c < chunks; c += 64) {
    const Part p = parts[c];
    const float d = p.m - ms, e = expf(d * a.scale);
    // the part's sums are over m_c - x: exp and distance move on to m
    const float all = p.z + (c == key_col(best) ? 0.f : 1.f);
    z += p.z != p.z ? p.z : e > 0.f ? e * all : 0.f;
    u += e > 0.f ? e * (p.u - d * all) : 0.f;
  }
  z = wave_sum_f32(z);
  u = wave_sum_f32(u);
  const float l = row_log(m, z);
  if (a.top > 0) {
    // the parts' lists are in order: the largest of their heads, one after the other
    __shared__ uint8_t head[kMaxParts];
    for (int c = lane; c < chunks; c += 64) head[c] = 0;
    for (int i = 0; i < a.top; ++i) {
      uint64_t k = 0;
      for (int c = lane; c < chunks; c += 64)
        if (head[c] < a.top) k = max64(k, tops[(int64_t)c * a.top + head[c]]);
      const uint64_t b = wave_max64(k);
      for (int c = lane; c < chunks; c += 64)
        if (head[c] < a.top && tops[(int64_t)c * a.top + head[c]] == b) ++head[c];
      if (lane == 0) {
        a.top_ids[row * a.top + i] = key_col(b);
        a.top_lp[row * a.top + i] = (key_value(b) - m) * a.scale - l;
      }
    }
  }
  if (lane == 0) write_row<T>(a, row, m, l, z, u);
}

// Parts of a row and their columns: at most what a block holds.
void split(int item, int64_t rows, int64_t cols, int *chunks, int *span) {
  const int64_t most = (int64_t)(kPieces - 1) * 16 / item;
  *chunks = (int)((cols + most - 1) / most);
  *span = (int)((cols + *chunks - 1) / *chunks + 63) / 64 * 64;
  *chunks = (int)((cols + *span - 1) / *span);
}

template <typename T>
int launch_scores(const ScoreArgs &a, hipStream_t s) {
  int chunks, span;
  split((int)sizeof(T), a.rows, a.cols, &chunks, &span);
  if (chunks > kMaxParts || a.rows * chunks > (1LL << 32) / NT - 1) return fail("too many logits for one call");
  hipLaunchKernelGGL((token_scores_kernel<T>), dim3((unsigned)(a.rows * chunks)), dim3(NT), 0, s, a, chunks, span);
  if (chunks > 1)
    hipLaunchKernelGGL((token_scores_join_kernel<T>), dim3((unsigned)a.rows), dim3(64), 0, s, a, chunks);
  return check_launch("token_scores_kernel");
}

}  // namespace

int64_t score_workspace(int type, int64_t rows, int64_t cols, int64_t top) {
  int chunks, span;
  split(type == LOGIT_I8 ? 1 : type == LOGIT_F32 ? 4 : 2, rows, cols, &chunks, &span);
  return chunks > 1 ? rows * chunks * ((int64_t)sizeof(Part) + 8 * top) : 0;
}

int launch_token_scores(const ScoreArgs &a, hipStream_t s) {
  switch (a.type) {
    case LOGIT_I8: return launch_scores<int8_t>(a, s);
    case LOGIT_F32: return launch_scores<float>(a, s);
    case LOGIT_BF16: return launch_scores<__hip_bfloat16>(a, s);
    default: return launch_scores<__half>(a, s);
  }
}

}  // namespace iw
