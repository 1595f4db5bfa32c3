// Device helpers of the attention kernels whose blocks hold the values of the shift
// exponential up to where it is 0 (iw_attn_tree.hip, iw_attn_window.hip): the tables,
// byte moves, and the four output columns of a lane.
#pragma once

#include "iw_attn_dev.hpp"
#include "iw_common.hpp"
#include "iw_kernels.hpp"

namespace iw {

namespace {

constexpr int kTableBits = 10, kTableBytes = 4992;

// First distance from which every value is 0: 2^-(t / 2^f) in f (at most 7)
// fractional bits is 0 once t > min(f, 7) 2^f, and t >= 23/16 n - 1.
__host__ __device__ constexpr int shift_exp_zero(int f) { return (((f < 7 ? f : 7) << f) + 2) * 16 / 23 + 1; }
// The tables lie one after the other, each in whole 16 bytes.
__host__ __device__ constexpr int table_at(int f) {
  int at = 0;
  for (int i = 1; i < f; ++i) at += (shift_exp_zero(i) + 16) / 16 * 16;
  return at;
}
static_assert(table_at(kTableBits + 1) - table_at(kTableBits) == kTableBytes, "the largest table fills the block's copy");

// The shift exponential of -n (n the score's distance from the row maximum
// plus one, 0 .. 32767): with t = n + ceil(n/2) - ceil(n/16) (n log2 e in
// 16-bit steps), 2^-(t / 2^f) as a linear fraction and a shift. Distances
// whose t passes 2^15 wrap there and give 0.
__host__ __device__ constexpr uint32_t shift_exp(int32_t n, int32_t f) {
  const int32_t t = n + ((n + 1) >> 1) - ((n + 15) >> 4);
  const int32_t m = (1 << f) - 1;
  const int32_t sh = ((t + m) >> f) + (f > 7 ? f - 7 : 0);
  const uint32_t num = (1u << f) | ((uint32_t)(-t & m) >> 1);
  return t > 32768 ? 0u : num >> (sh < 31 ? sh : 31);
}

struct ShiftExpTables {
  uint8_t v[table_at(kTableBits + 1)];
  constexpr ShiftExpTables() : v() {
    for (int f = 1; f <= kTableBits; ++f)
      for (int i = 0; i < table_at(f + 1) - table_at(f); ++i) v[table_at(f) + i] = (uint8_t)shift_exp(i, f);
  }
};
__device__ __attribute__((aligned(16))) constexpr ShiftExpTables kTables{};

// 0xff in the bytes of a 4-bit mask's set bits
__device__ __forceinline__ uint32_t byte_mask(uint32_t four) {
  const uint32_t ones = __umul24(four, 0x00204081u) & 0x01010101u;
  return (ones << 8) - ones;
}

// four words of four bytes to their transpose
__device__ __forceinline__ void transpose4(const uint32_t (&in)[4], uint32_t (&out)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u);  // in0.0 in1.0 in0.1 in1.1
  const uint32_t b = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);
  const uint32_t d = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
  out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// Four columns of a row's output from their sums and the row's inverse square root.
__device__ __forceinline__ uint32_t output_word(const AttnArgs &a, const uint32_t *sums, int32_t inv) {
  uint32_t w = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    int32_t y = rshift((int32_t)(sums[c] * (uint32_t)inv), a.rsqrt_off);
    y = rshift((int32_t)((uint32_t)y * (uint32_t)inv), a.rsqrt_off);
    y = rshift((int32_t)((uint32_t)y * a.av_m), a.av_s);
    w |= ((uint32_t)clampi(y, -127, 127) & 0xffu) << (8 * c);
  }
  return w;
}

}  // namespace

}  // namespace iw
