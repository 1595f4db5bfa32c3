// Token scores of rows of logits: the log-probability of a given token, the
// entropy and the most probable alternatives.
//
// With m the row's largest logit and the sums over every token but one that holds it,
//   Z' = sum exp((x - m) s),  U' = sum (m - x) s exp((x - m) s),
//   lse = m s + log1p(Z'),  entropy = log1p(Z') + U' / (1 + Z'):
// both terms are positive and keep their digits where one token holds nearly
// all of the probability. Alternatives are ordered by value, then by index.
//
// A block holds its part of a row in registers: the logits are read once. The
// largest of 64 groups of its threads meet in LDS, which gives every wave m
// and a bound that at least `top` logits reach; the sums and the few logits
// that reach the bound follow, and each of those finds its place by counting
// the larger ones. int8 logits are counted instead, one LDS add each: m, the
// sums and the exact bound come from the 256 counts, without an exp per logit
// and in any order the same.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "iw_common.hpp"
#include "iw_tree.hpp"

namespace iw {

namespace {

constexpr int kCand = 1024;      // candidates that the bound may leave
constexpr int kCopies = 4;       // of the int8 counts, for neighbouring lanes
constexpr int kMaxParts = 1024;  // parts of a row
constexpr int kPartBytes = 65536;  // of a block, in its registers
constexpr int kFewBlocks = 256;  // up to here: 1024 threads a block

// One block's part of a row: its largest logit, Z' and U' (in units of s)
struct Part {
  float m, z, u, pad;
};

// A logit and its column as one whole number: larger logits first, then lower
// columns; both zeros are one value and a NaN is the largest. Every key is above 0 and
// below ~0, also a NaN's in column 0.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  if (v != v) return 0xfffffffeu;
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

__device__ __forceinline__ uint32_t wave_max_u32_dpp(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
  return max(max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16)),
             max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}

// Sum over the wave, in every lane (DPP moves within 16 lanes, then their four sums)
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum_f32(float v) {
  v += dpp_f32<0xB1>(v);
  v += dpp_f32<0x4E>(v);
  v += dpp_f32<0x141>(v);
  v += dpp_f32<0x140>(v);
  const int b = (int)__float_as_uint(v);
  auto at = [&](int l) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane(b, l)); };
  return (at(0) + at(16)) + (at(32) + at(48));
}

__device__ __forceinline__ bool suppressed(const uint32_t *words, int col) {
  return words && ((words[col >> 5] >> (col & 31)) & 1u);
}

// The types. A piece is 16 bytes of logits; `off` has the bits of its
// suppressed ones.
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
  // the largest in the upper bytes of two 16-bit halves: the odd bytes lead
  // theirs, the even ones once shifted up
  typedef int16_t v2s __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ v2s halves(const uint4 &w) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    v2s t{-32768, -32768};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const v2s b = __builtin_bit_cast(v2s, v[q]);
      t = __builtin_elementwise_max(t, __builtin_elementwise_max(b, (v2s)(b << (int16_t)8)));
    }
    return t;
  }
  // bit 8 i + q for each byte i of word q that is v or more (v from -128 on)
  static __device__ __forceinline__ uint32_t reaching(const uint4 &w, int v) {
    constexpr uint32_t H = 0x80808080u;
    const uint32_t x[4] = {w.x, w.y, w.z, w.w}, low = (uint32_t)(v & 0x7f) * 0x01010101u;
    uint32_t bits = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // the bytes' lower seven bits are those of v or more; a byte's own sign decides if v has the other
      const uint32_t ge = (x[q] | H) - low;
      bits |= ((v < 0 ? ~x[q] | ge : ~x[q] & ge) & H) >> (7 - q);
    }
    return bits;
  }
};
template <typename D, int N>
struct FloatMax {
  static __device__ __forceinline__ float max(const uint4 &w) {
    float t = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; ++e) t = fmaxf(t, D::get(w, e));
    return t;
  }
};
template <>
struct Logit<float> : FloatMax<Logit<float>, 4> {
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
struct Logit<__hip_bfloat16> : Half<0xff80u>, FloatMax<Logit<__hip_bfloat16>, 8> {
  static __device__ __forceinline__ float one(const __hip_bfloat16 *p) {
    return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(p) << 16);
  }
  static __device__ __forceinline__ float get(const uint4 &w, int i) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    return __uint_as_float((i & 1) ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
  }
};
template <>
struct Logit<__half> : Half<0xfc00u>, FloatMax<Logit<__half>, 8> {
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

template <int NT>
struct Shared {
  uint32_t group[64];
  float z[NT / 64], u[NT / 64], n[NT / 64];
  uint32_t count[256 * kCopies];  // int8: logits of each value
  int cands;
  uint64_t best[NT / 64];
  uint64_t cand[kCand];
  uint64_t top[kScoreMaxTop];
};

// The top alternatives of a block's part one after the other, each the largest
// key below the last: for rows whose bound leaves too many candidates (whole
// rows of ties) or too few (suppressed tokens among the alternatives, NaN). Also for
// short rows of floats that fill fewer of the 64 groups of threads than there are
// alternatives (a group has up to 64 float32 or 128 16-bit columns) and have more
// than kCand logits: 64 rows of float16 with 32 alternatives take 61.5 us at 3000 columns,
// 9.8 at 4100, with 16 alternatives 6.4 and 6.2.
template <typename T, int NT>
__device__ __noinline__ void top_by_rounds(const T *x, int c0, int n, const uint32_t *suppress, int top,
                                           Shared<NT> &s) {
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
    for (int w = 0; w < NT / 64; ++w) k = max64(k, s.best[w]);
    if (threadIdx.x == 0) s.top[i] = k;  // 0: the part has no more logits
    prev = k;
  }
  __syncthreads();
}

// (v - m) * scale. Where v - m passes float32 the product need not: half of it and twice the scale.
__device__ __forceinline__ float scaled_distance(float v, float m, float scale) {
  const float d = v - m;
  return d == -INFINITY && v != -INFINITY ? (0.5f * v - 0.5f * m) * (2.f * scale) : d * scale;
}

template <typename T>
__device__ __forceinline__ void write_row(const ScoreArgs &a, int64_t row, float m, float l, float z, float u) {
  if (a.logprob) {
    const int64_t at = a.targets[row];
    float lp = __uint_as_float(0x7fc00000u);  // a token outside the vocabulary has none
    if (at >= 0 && at < a.cols) {
      const float v = suppressed(a.suppress, (int)at) ? -INFINITY
                                                      : Logit<T>::one(reinterpret_cast<const T *>(a.x) + row * a.ld + at);
      lp = scaled_distance(v, m, a.scale) - l;
    }
    a.logprob[row] = lp;
  }
  if (a.entropy) a.entropy[row] = l + u * a.scale / (1.f + z);
}

// log1p(Z'), NaN where the row has no finite maximum (all suppressed, an infinity, a NaN)
__device__ __forceinline__ float row_log(float m, float z) { return log1pf(z) + (m - m); }

// What a block works on at a time: the columns c0 .. c0 + n - 1 of a row, as
// whole 16-byte pieces and up to 2 (E - 1) single logits before and behind them.
template <typename T>
struct Item {
  const T *x;
  int64_t row;
  int c0, n, head, pieces;
  __device__ __forceinline__ Item(const ScoreArgs &a, int chunks, int span, int64_t i) {
    row = (uint32_t)i / (uint32_t)chunks;
    c0 = (int)((uint32_t)i % (uint32_t)chunks) * span;
    n = min(a.cols - c0, span);
    x = reinterpret_cast<const T *>(a.x) + row * a.ld + c0;
    head = min((int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)), n);
    pieces = (n - head) / Logit<T>::E;
  }
};

// In the place of pieces and words that there are none of; a choice between it and an argument is
// known to be device memory only as a number
__device__ __attribute__((aligned(16))) const uint32_t kNothing[4] = {};
template <typename V>
__device__ __forceinline__ const V __attribute__((address_space(1))) *in_global(const void *p) {
  return reinterpret_cast<const V __attribute__((address_space(1))) *>(reinterpret_cast<uintptr_t>(p));
}

// P: 16-byte pieces of a thread
template <typename T, int NT, int P>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(NT == 1024 ? 8 : 4))) void token_scores_kernel(
    ScoreArgs a, int chunks, int span) {
  using L = Logit<T>;
  constexpr bool I8 = std::is_same<T, int8_t>::value;
  constexpr int E = L::E, NW = NT / 64;
  __shared__ Shared<NT> s;
  constexpr int S = I8 ? 0 : (P * E + 31) / 32;  // a thread's words of the part's suppressed tokens; span is a multiple of 32
  __shared__ uint32_t sWords[S * NT + 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t item = blockIdx.x;
  const Item<T> it(a, chunks, span, item);
  uint4 w[P];
  // no branch between the loads, so that the first pieces are used while the others are on the way
  uint32_t sw[S + 1];
  {
    const auto *from = in_global<uint32_t>(a.suppress ? a.suppress + it.c0 / 32 : &kNothing[0]);
    const int last = a.suppress ? (it.n - 1) / 32 : 0;
#pragma unroll
    for (int i = 0; i < S; ++i) sw[i] = from[min(i * NT + tid, last)];
  }
  const int extra = tid < it.head ? tid : it.head + it.pieces * E + tid - it.head;
  const bool has_extra = extra < it.n;
  const T xr = it.x[min(extra, it.n - 1)];
  {
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    const auto *xa = in_global<v4u>(it.pieces > 0 ? static_cast<const void *>(it.x + it.head) : kNothing);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const v4u x = xa[min(p * NT + tid, max(it.pieces - 1, 0))];
      w[p] = make_uint4(x.x, x.y, x.z, x.w);
    }
  }
#pragma unroll
  for (int i = 0; i < S; ++i) sWords[i * NT + tid] = sw[i];
  if (tid == 0) s.cands = 0;
  if constexpr (I8)
    for (int i = tid; i < 256 * kCopies; i += NT) s.count[i] = 0;
  lds_barrier();

  const int c0 = it.c0, n = it.n;
  auto held = [&](int p) { return p * NT + tid < it.pieces; };
  auto column = [&](int p) { return c0 + it.head + (p * NT + tid) * E; };
  // the bits of a piece's suppressed logits (a piece may reach into the next word)
  auto hidden = [&](int p) -> uint32_t {
    const int at = column(p) - c0, i = at >> 5;
    const uint32_t *words = I8 ? a.suppress + c0 / 32 : sWords;
    const uint64_t two = (uint64_t)words[I8 ? min(i + 1, (n - 1) >> 5) : i + 1] << 32 | words[i];
    return (uint32_t)(two >> (at & 31)) & ((1u << E) - 1u);
  };
  float xe = has_extra ? L::one(&xr) : -INFINITY;
  if (!I8 && a.suppress && has_extra && ((sWords[extra >> 5] >> (extra & 31)) & 1u)) xe = -INFINITY;

  float m, reach, tmax, z = 0.f, u = 0.f, eq = 0.f;
  if constexpr (I8) {
    uint32_t *const mine = s.count + (lane & (kCopies - 1));
    // value v at 128 + v, that is the byte with its sign bit turned
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (held(p)) {
        const uint32_t v[4] = {w[p].x ^ 0x80808080u, w[p].y ^ 0x80808080u, w[p].z ^ 0x80808080u,
                               w[p].w ^ 0x80808080u};
#pragma unroll
        for (int i = 0; i < 16; ++i) atomicAdd(mine + kCopies * ((v[i >> 2] >> (8 * (i & 3))) & 0xffu), 1u);
      }
    if (has_extra) atomicAdd(mine + kCopies * ((int)xe + 128), 1u);
    // the suppressed ones are few: looked up and taken off
    if (a.suppress)
      for (int i = tid; i < (n + 31) / 32; i += NT) {
        uint32_t o = a.suppress[c0 / 32 + i];
        if (n - 32 * i < 32) o &= (1u << (n - 32 * i)) - 1u;
        for (; o; o &= o - 1) atomicSub(mine + kCopies * ((int)it.x[32 * i + __ffs((int)o) - 1] + 128), 1u);
      }
    lds_barrier();
    // every wave: lane l has the values 4 l .. 4 l + 3 (above -128)
    uint32_t c[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = 0;
#pragma unroll
      for (int j = 0; j < kCopies; ++j) c[i] += s.count[(4 * lane + i) * kCopies + j];
      sum += c[i];
    }
    const uint64_t any = __ballot(sum != 0);
    const int high = c[3] ? 3 : c[2] ? 2 : c[1] ? 1 : 0;
    const int hl = any ? 63 - __clzll((long long)any) : 0;
    const int mi = 4 * hl + __shfl(high, hl) - 128;
    m = any ? (float)mi : -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = mi + 128 - (4 * lane + i);
      if (d > 0 && c[i]) {
        const float e = (float)c[i] * expf(-(float)d * a.scale);
        z += e;
        u += e * (float)d;
      }
      if (d == 0) eq = (float)c[i];
    }
    z = wave_sum_f32(z);
    u = wave_sum_f32(u);
    eq = wave_sum_f32(eq);
    reach = -129.f;
    if (a.top > 0) {
      // the largest value that `top` logits reach: lanes from the top, then values
      uint32_t above = sum;  // logits of this lane's values and the larger ones
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t t = __shfl_down(above, o);
        if (lane + o < 64) above += t;
      }
      const uint64_t full = __ballot(above >= (uint32_t)a.top);
      if (full) {
        const int at = 63 - __clzll((long long)full);
        uint32_t have = __shfl(above - sum, at);
        int i = 3;
#pragma unroll
        for (int j = 3; j > 0; --j) {
          have += __shfl(c[j], at);
          if (i == j && have < (uint32_t)a.top) i = j - 1;
        }
        reach = (float)(4 * at + i - 128);
      }
    }
  } else {
    if (a.suppress) {
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (held(p)) {
          const uint32_t o = hidden(p);
          if (o) L::mask(w[p], o);
        }
    }
    tmax = xe;
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (held(p)) {
#pragma unroll
        for (int e = 0; e < E; ++e) tmax = fmaxf(tmax, L::get(w[p], e));
      }
    // the largest of each of 64 groups of threads
    float g = tmax;
    g = fmaxf(g, dpp_f32<0xB1>(g));
    g = fmaxf(g, dpp_f32<0x4E>(g));
    if (NT >= 512) g = fmaxf(g, dpp_f32<0x141>(g));
    if (NT >= 1024) g = fmaxf(g, dpp_f32<0x140>(g));
    if (tid % NW == 0) s.group[tid / NW] = ordered(g);
    lds_barrier();
    const uint32_t go = s.group[lane];
    reach = a.top > 0 ? key_value((uint64_t)kth_largest<16>(go, a.top) << 32) : 0.f;
    if (reach != reach) reach = -INFINITY;  // below every number: all logits
    m = key_value((uint64_t)wave_max_u32_dpp(go) << 32);
    const float ms = m == -INFINITY ? 0.f : m;  // a part without finite logits sums to 0
    auto add = [&](float v, bool all) {
      // beyond log2_far exp2 is 0, and near stays where its product with any log2_lo is small
      const float d = v - ms, near = fmaxf(d, a.log2_far);
      // log2(e) * scale in two parts, as the rounding of one would be the same for every logit
      const float e = __builtin_amdgcn_exp2f(fmaf(d, a.log2_hi, near * a.log2_lo));
      if (all || d != 0.f) {
        z += e;
        u -= near * e;  // -inf times its exp of 0 is 0
      } else {
        eq += 1.f;
      }
    };
    if (has_extra) add(xe, false);
    if (tmax == m) {  // few threads hold it and look for it
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (held(p)) {
#pragma unroll
          for (int e = 0; e < E; ++e) add(L::get(w[p], e), false);
        }
    } else {
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (held(p)) {
#pragma unroll
          for (int e = 0; e < E; ++e) add(L::get(w[p], e), true);
        }
    }
    z = wave_sum_f32(z);
    u = wave_sum_f32(u);
    eq = wave_sum_f32(eq);
    if (lane == 0) s.z[wave] = z, s.u[wave] = u, s.n[wave] = eq;
  }

  // ---- the logits that reach the bound ----
  auto put = [&](float v, int col) {
    if (v >= reach) {
      const int at = atomicAdd(&s.cands, 1);
      if (at < kCand) s.cand[at] = key_of(v, col);
    }
  };
  if constexpr (I8) {
    if (a.top > 0) {
      const int least = max((int)reach, -128);
      // a piece whose largest byte is below it has none
      using v2s = typename L::v2s;
      const int16_t under = (int16_t)(256 * least - (least > -128));
      const v2s bound{under, under};
      if (has_extra && !suppressed(a.suppress, c0 + extra)) put(xe, c0 + extra);
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (held(p) && (least == -128 || __builtin_bit_cast(uint32_t, __builtin_elementwise_max(L::halves(w[p]), bound)) !=
                                             __builtin_bit_cast(uint32_t, bound))) {
          uint32_t bits = L::reaching(w[p], least);
          const uint32_t o = a.suppress ? hidden(p) : 0u;
          for (; bits; bits &= bits - 1) {
            const int at = __ffs((int)bits) - 1, e = 4 * (at & 7) + (at >> 3);
            if (!((o >> e) & 1u)) put(L::get(w[p], e), column(p) + e);
          }
        }
    }
  } else if (a.top > 0 && tmax >= reach) {
    if (has_extra) put(xe, c0 + extra);
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (held(p) && L::max(w[p]) >= reach) {
        for (int e = 0; e < E; ++e) put(L::get(w[p], e), column(p) + e);
      }
  }
  lds_barrier();
  if constexpr (!I8) {
    z = u = eq = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) z += s.z[i], u += s.u[i], eq += s.n[i];
  }
  if (eq > 0.f) z += eq - 1.f;
  const float l = row_log(m, z);

  const int64_t row = it.row;
  const int cands = s.cands;
  const bool rounds = a.top > 0 && (cands > kCand || cands < min(a.top, n) || z != z || m - m != 0.f);
  if (rounds) top_by_rounds<T, NT>(it.x, c0, n, a.suppress, a.top, s);
  uint64_t *tops = nullptr;
  if (chunks > 1)
    tops = reinterpret_cast<uint64_t *>(reinterpret_cast<Part *>(a.workspace) + a.rows * chunks) + item * a.top;
  auto place = [&](int at, uint64_t k) {
    if (tops) {
      tops[at] = k;
    } else {
      a.top_ids[row * a.top + at] = key_col(k);
      a.top_lp[row * a.top + at] = scaled_distance(key_value(k), m, a.scale) - l;
    }
  };
  if (rounds) {
    if (tid < a.top) place(tid, s.top[tid]);
  } else {
    for (int j = tid; j < cands; j += NT) {
      const uint64_t k = s.cand[j];
      int larger = 0;
      for (int i = 0; i < cands; ++i) larger += s.cand[i] > k;
      if (larger < a.top) place(larger, k);
    }
    // a part of fewer logits than alternatives
    if (tops && cands + tid < a.top) tops[cands + tid] = 0;
  }
  if (tid == 0) {
    if (tops)
      reinterpret_cast<Part *>(a.workspace)[item] = Part{m, z, u, 0.f};
    else
      write_row<T>(a, row, m, l, z, u);
  }
}

// Joins a row's parts, one block per row.
constexpr int JT = 256, kJoinKeys = 2048;
template <typename T>
__global__ __launch_bounds__(JT) void token_scores_join_kernel(ScoreArgs a, int chunks) {
  __shared__ uint64_t sKey[kJoinKeys];
  __shared__ uint16_t sHead[kMaxParts];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const Part *parts = reinterpret_cast<const Part *>(a.workspace) + row * chunks;
  const int keys = chunks * a.top;
  const uint64_t *tops =
      reinterpret_cast<const uint64_t *>(reinterpret_cast<const Part *>(a.workspace) + a.rows * chunks) + row * keys;
  for (int i = tid; i < min(keys, kJoinKeys); i += JT) sKey[i] = tops[i];
  // every wave sums the parts: the first that holds the largest logit keeps it out of Z'
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
  auto place = [&](int at, uint64_t k) {
    a.top_ids[row * a.top + at] = key_col(k);
    a.top_lp[row * a.top + at] = scaled_distance(key_value(k), m, a.scale) - l;
  };
  __syncthreads();
  if (keys <= kJoinKeys) {
    for (int i = tid; i < keys; i += JT) {  // a key's place is the number of larger ones
      const uint64_t k = sKey[i];
      int larger = 0;
      for (int j = 0; j < keys; ++j) larger += sKey[j] > k;
      if (larger < a.top && k != 0) place(larger, k);
    }
  } else if (tid < 64) {  // the largest of the parts' heads, one after the other
    for (int c = lane; c < chunks; c += 64) sHead[c] = 0;
    for (int i = 0; i < a.top; ++i) {
      uint64_t k = 0;
      for (int c = lane; c < chunks; c += 64)
        if (sHead[c] < a.top) k = max64(k, tops[(int64_t)c * a.top + sHead[c]]);
      const uint64_t b = wave_max64(k);
      for (int c = lane; c < chunks; c += 64)
        if (sHead[c] < a.top && tops[(int64_t)c * a.top + sHead[c]] == b) ++sHead[c];
      if (lane == 0) place(i, b);
    }
  }
  if (tid == 0) write_row<T>(a, row, m, l, z, u);
}

// Parts of a row and their columns, and the kernel's form. us of 256 threads of 16
// pieces, 512 of 8 and 1024 of 4 (all a part of 64 KB):
//   2048 rows of 51865 int8 logits 36.0 / 38.5 / 45.1, 512 rows of float32 33.7 / 33.3 / 33.9,
//   512 rows of float16 33.2 / 28.3 / 29.3: fewer threads do less beside the logits, and int8
//   has next to nothing to do for one;
//   one row of int8 12 / 11 / 10.1, 91 of float32 15.0 / 12.8 / 12.8: few blocks wait for
//   themselves, and more threads are a shorter chain.
// Parts of 16 KB were slower for all (int8 50, float32 34.9, float16 32.7), and so were blocks that
// stay and request their next part early (int8 48, float32 44): their registers cost more waves
// than the reads gained. With pieces used as they arrive and alternatives found by words, 2048
// rows of int8 take 34.0 us, 41.7 with four alternatives, targets and suppressed tokens (42.9 where a
// block waited for all of its pieces), 512 of float32 32.6, 2048 of float32 77 (5.5 TB/s). What is
// left above a read of the bytes (106 MB 19 us): int8 is bound by LDS adds (8.6 cycles per 64
// of them), the others by issuing ~9 instructions a logit at 2 GHz.
struct Split {
  int chunks, span;
  bool few;
};
Split split(int type, int64_t rows, int64_t cols) {
  const int item = type == LOGIT_I8 ? 1 : type == LOGIT_F32 ? 4 : 2;
  const int64_t most = kPartBytes / item - 16;
  Split s;
  s.chunks = (int)((cols + most - 1) / most);
  s.few = rows * s.chunks <= kFewBlocks;
  s.span = (int)((cols + s.chunks - 1) / s.chunks + 63) / 64 * 64;
  s.chunks = (int)((cols + s.span - 1) / s.span);
  return s;
}

template <typename T, int NT, int P>
int launch_scores_p(const ScoreArgs &a, const Split &sp, hipStream_t s) {
  hipLaunchKernelGGL((token_scores_kernel<T, NT, P>), dim3((unsigned)(a.rows * sp.chunks)), dim3(NT), 0, s, a,
                     sp.chunks, sp.span);
  if (sp.chunks > 1)
    hipLaunchKernelGGL((token_scores_join_kernel<T>), dim3((unsigned)a.rows), dim3(JT), 0, s, a, sp.chunks);
  return check_launch("token_scores_kernel");
}

template <typename T>
int launch_scores(ScoreArgs a, hipStream_t s) {
  const Split sp = split(a.type, a.rows, a.cols);
  // blocks of 512 threads at most where they are many, fewer than 2^32 threads
  if (sp.chunks > kMaxParts || a.rows * sp.chunks > (1LL << 32) / 512 - 1) return fail("too many logits for one call");
  const double c = (double)a.scale * 1.4426950408889634;
  a.log2_hi = (float)std::min(c, 3.4e38);
  a.log2_lo = (float)(c - (double)a.log2_hi);
  a.log2_far = (float)(-200.0 / (double)a.log2_hi);
  if (sp.few) return launch_scores_p<T, 1024, 4>(a, sp, s);
  return launch_scores_p<T, sizeof(T) == 1 ? 256 : 512, sizeof(T) == 1 ? 16 : 8>(a, sp, s);
}

}  // namespace

int64_t score_workspace(int type, int64_t rows, int64_t cols, int64_t top) {
  const int chunks = split(type, rows, cols).chunks;
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
