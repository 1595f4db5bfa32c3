// Token scores of rows of logits: the log-probability of a given token, the
// entropy and the most probable alternatives.
//
// With m the row's largest logit and the sums over every other token,
//   Z' = sum exp((x - m) s),  U' = sum (m - x) s exp((x - m) s),
//   lse = m s + log1p(Z'),  entropy = log1p(Z') + U' / (1 + Z'):
// both terms are positive and keep their digits where one token holds nearly
// all of the probability. Alternatives are ordered by value, then by index.
//
// A block takes up to 65536 logits of a row; longer rows are split over blocks
// whose results a second kernel joins.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "iw_common.hpp"
#include "iw_tree.hpp"

namespace iw {

namespace {

constexpr int NT = 1024, NW = NT / 64;
constexpr int kChunk = 65536;  // logits of a block

// One block's part of a row (m and best: its largest logit and its key)
struct Part {
  uint64_t best;
  float z, u;
};

template <typename T>
struct Logit;
template <>
struct Logit<int8_t> {
  static constexpr int E = 16;
  static __device__ __forceinline__ float get(const uint4 &w, int i) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    return (float)(int8_t)(v[i >> 2] >> (8 * (i & 3)));
  }
  static __device__ __forceinline__ float one(const int8_t *p) { return (float)*p; }
};
template <>
struct Logit<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ float get(const uint4 &w, int i) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    return __uint_as_float(v[i]);
  }
  static __device__ __forceinline__ float one(const float *p) { return *p; }
};
template <>
struct Logit<__hip_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ float get(const uint4 &w, int i) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    return __uint_as_float((i & 1) ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
  }
  static __device__ __forceinline__ float one(const __hip_bfloat16 *p) {
    return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(p) << 16);
  }
};
template <>
struct Logit<__half> {
  static constexpr int E = 8;
  static __device__ __forceinline__ float get(const uint4 &w, int i) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    return __half2float(__ushort_as_half((uint16_t)(v[i >> 1] >> (16 * (i & 1)))));
  }
  static __device__ __forceinline__ float one(const __half *p) { return __half2float(*p); }
};

// A logit and its column as one whole number: larger logits first, then lower
// columns; both zeros are one value and a NaN is the largest.
__device__ __forceinline__ uint64_t key_of(float v, int col) {
  uint32_t b = __float_as_uint(v + 0.0f);
  b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  if (v != v) b = 0xffffffffu;
  return ((uint64_t)b << 32) | (uint32_t)~col;
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
__device__ __forceinline__ uint64_t block_max64(uint64_t v, uint64_t *sh) {
  v = wave_max64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) v = max64(v, sh[w]);
  return v;
}
__device__ __forceinline__ float block_sum(float v, float *sh) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) v += sh[w];
  return v;
}

__device__ __forceinline__ bool suppressed(const uint32_t *words, int col) {
  return words && ((words[col >> 5] >> (col & 31)) & 1u);
}

// A row's results from its best key, Z' and U' over the others, and the alternatives' keys.
template <typename T>
__device__ __forceinline__ void write_row(const ScoreArgs &a, int64_t row, uint64_t best, float z, float u,
                                          const uint64_t *top) {
  const float m = key_value(best);
  // no finite maximum (all suppressed, an infinity or a NaN): no probabilities
  const float bad = (m - m);
  const float l = log1pf(z) + bad;
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
  if (a.entropy) a.entropy[row] = l + u / (1.f + z);
  for (int i = 0; i < a.top; ++i) {
    a.top_ids[row * a.top + i] = key_col(top[i]);
    a.top_lp[row * a.top + i] = (key_value(top[i]) - m) * a.scale - l;
  }
}

template <typename T>
__global__ __launch_bounds__(NT) void token_scores_kernel(ScoreArgs a, int chunks) {
  using L = Logit<T>;
  constexpr int E = L::E;
  __shared__ uint64_t sKey[NW];
  __shared__ float sSum[NW];
  __shared__ uint64_t sTop[kScoreMaxTop];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / chunks;
  const int chunk = blockIdx.x % chunks;
  const int c0 = chunk * kChunk, n = min(a.cols - c0, kChunk);  // this block's columns
  const T *x = reinterpret_cast<const T *>(a.x) + row * a.ld + c0;
  // whole 16-byte pieces, and up to 2 (E - 1) logits before and behind them
  const int head = min((int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)), n);
  const int pieces = (n - head) / E, tail0 = head + pieces * E;
  const uint4 *xa = reinterpret_cast<const uint4 *>(x + head);
  const int extra = tid < head ? tid : tail0 + tid - head;  // this thread's single logit
  const bool has_extra = extra < n;
  float xe = has_extra ? L::one(x + extra) : 0.f;
  if (has_extra && suppressed(a.suppress, c0 + extra)) xe = -INFINITY;

  auto each = [&](auto &&f) {
    if (has_extra) f(xe, c0 + extra);
    for (int i0 = tid; i0 < pieces; i0 += NT) {
      const uint4 w = xa[i0];
      const int col0 = c0 + head + i0 * E;
      uint32_t off = 0;
      if (a.suppress) {
        const int last = (a.cols - 1) >> 5;
        const uint64_t two = (uint64_t)a.suppress[min((col0 >> 5) + 1, last)] << 32 | a.suppress[col0 >> 5];
        off = (uint32_t)(two >> (col0 & 31));
      }
#pragma unroll
      for (int e = 0; e < E; ++e) f((off >> e) & 1u ? -INFINITY : L::get(w, e), col0 + e);
    }
  };

  uint64_t best = 0;
  each([&](float v, int col) { best = max64(best, key_of(v, col)); });
  best = block_max64(best, sKey);
  const float m = key_value(best);
  const int bcol = key_col(best);
  float z = 0.f, u = 0.f;
  each([&](float v, int col) {
    const float d = (v - m) * a.scale;
    const float e = __expf(d);
    if (col != bcol) {
      z += e;
      u += e > 0.f ? -d * e : 0.f;
    }
  });
  z = block_sum(z, sSum);
  u = block_sum(u, sSum);
  if (a.top) {
    uint64_t prev = best;
    if (tid == 0) sTop[0] = best;
    for (int i = 1; i < min(a.top, n); ++i) {
      uint64_t k = 0;
      each([&](float v, int col) {
        const uint64_t q = key_of(v, col);
        if (q < prev) k = max64(k, q);
      });
      prev = block_max64(k, sKey);
      if (tid == 0) sTop[i] = prev;
    }
    if (tid == 0)
      for (int i = n; i < a.top; ++i) sTop[i] = 0;
  }
  if (tid != 0) return;
  if (chunks == 1) {
    write_row<T>(a, row, best, z, u, sTop);
    return;
  }
  Part *parts = reinterpret_cast<Part *>(a.workspace);
  uint64_t *tops = reinterpret_cast<uint64_t *>(parts + a.rows * chunks) + (int64_t)blockIdx.x * a.top;
  parts[blockIdx.x] = Part{best, z, u};
  for (int i = 0; i < a.top; ++i) tops[i] = sTop[i];
}

// Joins a row's parts: one thread per row.
template <typename T>
__global__ __launch_bounds__(64) void token_scores_join_kernel(ScoreArgs a, int chunks) {
  const int64_t row = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (row >= a.rows) return;
  const Part *parts = reinterpret_cast<const Part *>(a.workspace) + row * chunks;
  const uint64_t *tops =
      reinterpret_cast<const uint64_t *>(reinterpret_cast<const Part *>(a.workspace) + a.rows * chunks) +
      row * chunks * a.top;
  uint64_t best = 0;
  for (int c = 0; c < chunks; ++c) best = max64(best, parts[c].best);
  const float m = key_value(best);
  float z = 0.f, u = 0.f;
  for (int c = 0; c < chunks; ++c) {
    const Part p = parts[c];
    if (p.best == best) {
      z += p.z;
      u += p.u;
    } else {  // the part's sums are over (x - m_c): exp and the distance move to m
      const float d = (key_value(p.best) - m) * a.scale, e = __expf(d);
      if (e > 0.f) {
        z += e * (1.f + p.z);
        u += e * (p.u - d * (1.f + p.z));
      }
    }
  }
  uint64_t top[kScoreMaxTop];
  uint64_t prev = ~0ull;
  for (int i = 0; i < a.top; ++i) {
    uint64_t k = 0;
    for (int c = 0; c < chunks * a.top; ++c)
      if (tops[c] < prev) k = max64(k, tops[c]);
    top[i] = prev = k;
  }
  write_row<T>(a, row, best, z, u, top);
}

template <typename T>
int launch_scores(const ScoreArgs &a, hipStream_t s) {
  const int chunks = (a.cols + kChunk - 1) / kChunk;
  hipLaunchKernelGGL((token_scores_kernel<T>), dim3((unsigned)(a.rows * chunks)), dim3(NT), 0, s, a, chunks);
  if (chunks > 1)
    hipLaunchKernelGGL((token_scores_join_kernel<T>), dim3((unsigned)((a.rows + 63) / 64)), dim3(64), 0, s, a, chunks);
  return check_launch("token_scores_kernel");
}

}  // namespace

int64_t score_workspace(int64_t rows, int64_t cols, int64_t top) {
  const int64_t chunks = (cols + kChunk - 1) / kChunk;
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
