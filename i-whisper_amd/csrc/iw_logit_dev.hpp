// Device helpers of the kernels that read rows of logits (iw_logprobs.hip,
// iw_sample.hip): the types, pieces of 16 bytes, ordered keys.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "iw_common.hpp"

namespace iw {

namespace {

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
  // the bits spread over the halves are opaque to the compiler, which makes a compare and a select of each otherwise
  static __device__ __forceinline__ void mask(uint4 &w, uint32_t off) {
    uint32_t *v = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t lo, hi;
      asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(lo) : "v"(off), "n"(2 * i));
      asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(hi) : "v"(off), "n"(2 * i + 1));
      const uint32_t no = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
      v[i] = (v[i] & ~no) | (INF * 0x10001u & no);
    }
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

}  // namespace

}  // namespace iw
