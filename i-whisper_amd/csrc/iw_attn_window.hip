// Integer attention of each query over the keys of a window around its position and
// the first keys of its row. Query i of row b at position p sees key j where
//   j < len[b],  j <= p + after,  and  j >= p - before or j < sinks:
// a decoder's causal window (after = 0), an encoder's local one, or the frames around
// where a row is. The arithmetic per (query, key) is that of the other integer attention
// kernels: the requantized scores' row maximum first, then P = E(S - rowmax - 1), sum P
// and P.V, exact modulo 2^32 in any order, so the keys can be split over waves.
//
// A block has 16 * QT queries of a (batch, head) and goes through the 64-key chunks that any of
// them sees: those of the first keys, then those of the windows. In a chunk's four 16x16x64
// score products, row 4g + r of product t is key 16g + 4t + r: lane group g then holds the scores
// of the 16 consecutive keys that its bytes of the P.V operand stand for, and no lane
// exchange is needed. V's columns go to the products as d = 4n + c (lane n, product c): a lane
// reads whole words, and its four sums are one word of the output. A query's window is
// an interval of a lane group's 16 keys: its mask is three shifts.
#include <algorithm>

#include "iw_attn_sexp.hpp"
#include "iw_common.hpp"
#include "iw_drafts.hpp"

namespace iw {

namespace {

// The keys that a query sees: [start, end) and [0, first)
struct Seen {
  int start, end, first;
};
__device__ __forceinline__ Seen seen_from(const WindowArgs &t, int len, int64_t p) {
  Seen s;
  s.end = (int)max((int64_t)0, min((int64_t)len, p + t.after + 1));
  s.start = (int)max((int64_t)0, min((int64_t)s.end, p - t.before));
  s.first = min(t.sinks, s.end);
  return s;
}

// the lowest n bits of 16, n clamped to [0, 16]
__device__ __forceinline__ uint32_t low_bits(int n) { return (1u << clampi(n, 0, 16)) - 1u; }

__device__ __forceinline__ uint32_t low4(int n) { return (1u << clampi(n, 0, 4)) - 1u; }

// Minimum and maximum over the 16 lanes of a DPP row, in every lane of it
__device__ __forceinline__ int row16_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(INT32_MIN, v, 0xB1, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(INT32_MIN, v, 0x4E, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(INT32_MIN, v, 0x141, 0xf, 0xf, false));
  return max(v, __builtin_amdgcn_update_dpp(INT32_MIN, v, 0x140, 0xf, 0xf, false));
}
__device__ __forceinline__ int row16_min(int v) { return ~row16_max(~v); }

// The score where bit i of `hidden` is 0, else INT32_MIN. The bit spread over the word is opaque to the compiler,
// which makes a compare and a select of each otherwise (the score comes from a matrix instruction, so that the
// instruction which reads it has to be the compiler's).
__device__ __forceinline__ int32_t hide(int32_t score, uint32_t hidden, int i) {
  int32_t no;
  asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(no) : "v"(hidden), "n"(i));
  return (no & INT32_MIN) | (~no & score);
}

// The bytes of w whose bit of the four is set, 0 in the others: a byte permute gives 0 for a selector of 12, 0xff
// for 13
__device__ __forceinline__ uint32_t keep_bytes(uint32_t w, uint32_t four) {
  const uint32_t sel = (__umul24(four, 0x00204081u) & 0x01010101u) | 0x0c0c0c0cu;
  return w & __builtin_amdgcn_perm(w, w, sel);
}

// Four bytes as a word
__device__ __forceinline__ uint32_t pack4(uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b3, b2, 0x0c0c0400u), __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u),
                               0x05040100u);
}

// The last steps of a row: sums * inv, twice, and the output's scale, each rounded. Products of 24-bit numbers take
// a quarter of a 32-bit one's time: the first shift leaves 24 bits where it is 8 or more, and the second 24 - 8.
struct Finish {
  bool brief;  // the shifts allow it
  int32_t off, av_s, av_m, off_half, av_half;
  __device__ __forceinline__ explicit Finish(const AttnArgs &a)
      : brief(a.rsqrt_off >= 8 && a.av_s >= 1 && a.av_s <= 31), off((int32_t)a.rsqrt_off), av_s((int32_t)a.av_s),
        av_m((int32_t)a.av_m), off_half(a.rsqrt_off ? 1 << (a.rsqrt_off - 1) : 0), av_half(a.av_s >= 1 && a.av_s <= 31 ? 1 << (a.av_s - 1) : 0) {}
  static __device__ __forceinline__ int32_t shift(int32_t x, int32_t half, int32_t s) {
    return (int32_t)((uint32_t)x + (uint32_t)half + (uint32_t)(x >> 31)) >> s;
  }
  __device__ __forceinline__ uint32_t word(const AttnArgs &a, const uint32_t *sums, int32_t inv, bool fast) const {
    if (!fast) return output_word(a, sums, inv);
    uint32_t b[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      int32_t y = shift((int32_t)(sums[c] * (uint32_t)inv), off_half, off);
      y = shift(__mul24(y, inv), off_half, off);
      y = shift(__mul24(y, av_m), av_half, av_s);
      b[c] = (uint32_t)clampi(y, -127, 127);
    }
    return pack4(b[0], b[1], b[2], b[3]);
  }
};

// Row q from element r of a lane's products, four columns of each
template <int KS>
__device__ __forceinline__ void finish_row(const WindowArgs &t, const Finish &fin, int8_t *obase, int q, int cnt,
                                           const v4i (&o)[KS][4], int r, int32_t inv, bool fast, int n) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const uint32_t sums[4] = {(uint32_t)o[ks][0][r], (uint32_t)o[ks][1][r], (uint32_t)o[ks][2][r], (uint32_t)o[ks][3][r]};
    const uint32_t w = fin.word(t.a, sums, inv, fast);
    const int d = 64 * ks + 4 * n;
    if (q < t.a.Tq && d < t.a.D) *reinterpret_cast<uint32_t *>(obase + (int64_t)q * t.a.o_st + d) = q < cnt ? w : 0u;
  }
}

// waves a SIMD: registers allow four with 64 columns a head; two blocks of 128 columns fill a CU's LDS (70 528 bytes each)
constexpr int rows_waves(int ks) { return ks == 1 ? 4 : 2; }

// The chunks of 64 keys that any of the 16 queries of a tile sees: the first ns hold first keys, the others follow
// one another from w0 on. And the keys that all of them see.
struct Tile {
  int ns, w0, nch, start, end, first, all_from, all_to;
  __device__ __forceinline__ int at(int c) const { return c < ns ? c : w0 + c - ns; }
  __device__ __forceinline__ bool whole(int kc) const { return 64 * kc >= all_from && 64 * kc + 64 <= all_to; }
  // The first and last key of the chunk at kc that any of them sees: no others are read (2560 heads of 64, one query a
  // tile: 128 keys and four first ones 16.3 us with whole chunks, 15.6 so; 257 frames 35.8 and 31.4).
  __device__ __forceinline__ int low(int kc) const { return 64 * kc < first ? 0 : max(start - 64 * kc, 0); }
  __device__ __forceinline__ int high(int kc) const { return min((kc < w0 ? first : end) - 64 * kc, 64) - 1; }
};
// the tile at q0 < cnt, lane n & 15 has query q0 + n (queries past the count repeat the last one)
__device__ __forceinline__ Tile tile_of(const WindowArgs &t, int64_t b, int len, int cnt, int q, int sinks, Seen &seen) {
  const int64_t p = t.positions ? (int64_t)t.positions[b * t.pos_sb + q] : (int64_t)len - cnt + q;
  seen = seen_from(t, len, p);
  const int start = __builtin_amdgcn_readfirstlane(row16_min(seen.start));
  const int end = __builtin_amdgcn_readfirstlane(row16_max(seen.end));
  Tile x;
  x.start = start, x.end = end, x.first = min(sinks, end);
  x.all_from = __builtin_amdgcn_readfirstlane(row16_max(seen.start));
  x.all_to = __builtin_amdgcn_readfirstlane(row16_min(seen.end));
  x.w0 = min(start, end) / 64;
  x.ns = min((min(sinks, end) + 63) / 64, x.w0);
  x.nch = x.ns + max(0, (end + 63) / 64 - x.w0);
  return x;
}

// Where several blocks share the chunks of a tile: a part's words in the workspace are the sums of P.V of its rows,
// those of P, the row maxima. Every part but the last has as many chunks, the last ones may have none.
constexpr int part_words(int ks) { return 16 * (64 * ks + 2); }
template <int KS>
__device__ __forceinline__ uint32_t *part_of(const WindowArgs &t, int64_t block, int part, int parts) {
  return t.workspace + (block * parts + part) * part_words(KS);
}
__device__ __forceinline__ int part_share(int nch, int parts) { return max(1, (nch + parts - 1) / parts); }

// Of all keys, or of blockIdx.y's part of them: the row maxima, or with every part's maxima the sums
enum { ALL, PART_MAX, PART_SUM };

// Few queries, or positions in any order: a block has one tile, its waves take the chunks in turn. KS: 64-column parts
// of the head; QUADS: V in key quads; NW waves; NC > 0: a wave has at most NC chunks, whose K and V are all requested at the
// start and kept.
constexpr int window_waves(int ks, int nc) { return ks * (nc > 0 ? nc : 1) == 1 ? 4 : ks * nc <= 2 ? 3 : 2; }
template <int KS, bool QUADS, int NW, int NC, int MODE>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(window_waves(KS, NC)))) void attn_window_kernel(
    WindowArgs t, int qblocks, int blocks, int per_xcd, int per_word, int table_off) {
  constexpr int QR = 16, OLD = 64 * KS + 4, HC = NC > 0 ? NC : 1;
  static_assert(MODE == ALL || NC == 0, "parts loop over their chunks");
  __shared__ __attribute__((aligned(16))) uint8_t sTable[kTableBytes];
  __shared__ int32_t sMax[NW][QR];
  __shared__ uint32_t sSum[NW][QR];
  __shared__ int32_t sInv[QR];
  __shared__ __attribute__((aligned(16))) uint32_t sO[NW][QR * OLD];

  // the blocks of a (batch, head) are neighbours on one XCD (blockIdx % 8) and share its L2
  const int block = (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8);
  if (block >= blocks) return;
  const AttnArgs &a = t.a;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int q0 = block % qblocks * QR, bh = block / qblocks;
  const int h = bh % a.H;
  const int64_t b = bh / a.H;
  const int D = a.D, N = a.Tq;
  const int len = t.lengths ? clampi(t.lengths[b], 0, a.Tk) : a.Tk;
  const int cnt = t.counts ? clampi(t.counts[b], 0, N) : N;
  const int8_t *const kbase = a.k + b * a.k_sb + (int64_t)h * a.k_sh;
  const int8_t *const vbase = a.vt + b * a.v_sb + (int64_t)h * a.v_sh;
  int8_t *const obase = a.out + b * a.o_sb + (int64_t)h * D;
  const int words = D / 4, rows = min(N - q0, QR);
  // i / words for the i < 2^9 of the output
  const auto by_words = [&](int i) { return (int)__umul24(i, per_word) >> 16; };

  if (q0 >= cnt) {  // no query of these is in use
    if (MODE != ALL) return;
    for (int i = tid; i < rows * words; i += 64 * NW) {
      const int q = by_words(i);
      *reinterpret_cast<uint32_t *>(obase + (int64_t)(q0 + q) * a.o_st + 4 * (i - q * words)) = 0u;
    }
    return;
  }
  const int q = min(q0 + n, cnt - 1);
  Seen seen;
  const Tile tile = tile_of(t, b, len, cnt, q, t.sinks, seen);
  const int parts = MODE == ALL ? 1 : (int)gridDim.y, part = MODE == ALL ? 0 : (int)blockIdx.y;
  const int share = MODE == ALL ? tile.nch : part_share(tile.nch, parts);
  const int c_lo = part * share, c_hi = min(c_lo + share, tile.nch);  // this block's chunks
  if (MODE != ALL && part > 0 && c_lo >= tile.nch) return;

  // The K operands of the chunk at kc: keys that no query sees repeat the next one that any does, head dims past D the
  // last ones (the query is zero there). A chunk's base is uniform, its lanes' offsets fit 32 bits and are the same
  // for every chunk of which all keys are read.
  const int kcol = 16 * g, key0 = 16 * (n >> 2) + (n & 3);
  uint32_t koff[KS], voff[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    koff[ks] = (uint32_t)key0 * (uint32_t)a.k_st + (uint32_t)min(64 * ks + kcol, D - 16);
    const uint32_t d0 = (uint32_t)min(64 * ks + 4 * n, D - 4);
    voff[ks] = QUADS ? (uint32_t)(4 * g) * (uint32_t)a.v_sq + 4 * d0 : d0 * (uint32_t)a.v_sd + (uint32_t)(16 * g);
  }
  auto load_k = [&](int kc, v4i (&f)[4][KS]) {
    const int8_t *base = kbase + (int64_t)(64 * kc) * a.k_st;
    const int low = tile.low(kc), high = tile.high(kc);
    if (low == 0 && high == 63) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          f[i][ks] = *reinterpret_cast<const v4i *>(base + (int64_t)(4 * i) * a.k_st + koff[ks]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          f[i][ks] = *reinterpret_cast<const v4i *>(base + ((uint32_t)clampi(key0 + 4 * i, low, high) * (uint32_t)a.k_st +
                                                            (uint32_t)min(64 * ks + kcol, D - 16)));
    }
  };
  // Quads and transposed rows hold words of four keys of one column. Columns past D
  // repeat the last ones; their sums are not stored.
  auto load_v = [&](int kc, v4i (&f)[KS][4]) {
    const int8_t *base = vbase + (QUADS ? (int64_t)(16 * kc) * a.v_sq : (int64_t)(64 * kc));
    const int low = tile.low(kc), high = tile.high(kc);
    if (low == 0 && high == 63) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          f[ks][i] = *reinterpret_cast<const v4i *>(base + (int64_t)i * (QUADS ? a.v_sq : a.v_sd) + voff[ks]);
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint32_t d0 = (uint32_t)min(64 * ks + 4 * n, D - 4);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          f[ks][i] = *reinterpret_cast<const v4i *>(
              base + (QUADS ? (uint32_t)clampi(4 * g + i, low >> 2, high >> 2) * (uint32_t)a.v_sq + 4 * d0
                            : (d0 + i) * (uint32_t)a.v_sd + (uint32_t)clampi(16 * g, low & ~15, high & ~15)));
      }
    }
  };

  // ---- everything that the start can ask for ----
  v4i kf[HC][4][KS], vf[HC][KS][4], qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int d0 = 64 * ks + 16 * g;
    qf[ks] = v4i{0, 0, 0, 0};
    if (d0 < D) qf[ks] = *reinterpret_cast<const v4i *>(a.q + b * a.q_sb + (int64_t)q * a.q_st + (int64_t)h * D + d0);
  }
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (wave + NW * i < tile.nch) load_k(tile.at(wave + NW * i), kf[i]);
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (wave + NW * i < tile.nch) load_v(tile.at(wave + NW * i), vf[i]);
    __builtin_amdgcn_sched_barrier(0);
  }
  const bool table = table_off >= 0;
  const int zero = table ? shift_exp_zero(a.frac_bits) : IW_SEXP_LUT - 1;
  if (MODE != PART_MAX && table)
    for (int i = 16 * tid; i <= zero; i += 16 * 64 * NW)
      *reinterpret_cast<uint4 *>(sTable + i) = *reinterpret_cast<const uint4 *>(kTables.v + table_off + i);

  auto scores = [&](const v4i (&f)[KS]) {
    v4i s{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[ks], qf[ks], s, 0, 0, 0);
    return s;
  };
  // which of the lane group's 16 keys of the chunk at kc this lane's query sees
  auto counted = [&](int kc) -> uint32_t {
    const int k0 = 64 * kc + 16 * g;
    return (low_bits(seen.end - k0) & ~low_bits(seen.start - k0)) | low_bits(seen.first - k0);
  };

  // ---- pass 1: row maximum of the raw scores ----
  int32_t mx = INT32_MIN;
  auto chunk_max = [&](int kc, const v4i (&f)[4][KS]) {
    v4i s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = scores(f[i]);
    if (!tile.whole(kc)) {
      const uint32_t off = ~counted(kc);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] = hide(s[i][r], off, 4 * i + r);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = max(max(max(mx, s[i][0]), s[i][1]), max(s[i][2], s[i][3]));
  };
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (wave + NW * i < tile.nch) chunk_max(tile.at(wave + NW * i), kf[i]);
  } else if constexpr (MODE != PART_SUM) {
    v4i kn[4][KS];
#pragma unroll 1
    for (int c = c_lo + wave; c < c_hi; c += 2 * NW) {
      load_k(tile.at(c), kf[0]);
      if (c + NW < c_hi) load_k(tile.at(c + NW), kn);
      chunk_max(tile.at(c), kf[0]);
      if (c + NW < c_hi) chunk_max(tile.at(c + NW), kn);
    }
  }
  if (MODE == PART_SUM)  // the maxima of the parts that have chunks, shared out to the waves' lane groups
    for (int p = NW * g + wave; p == 0 || p * share < tile.nch; p += 4 * NW)
      mx = max(mx, (int32_t)part_of<KS>(t, block, p, parts)[QR * (64 * KS + 1) + n]);
  mx = max(mx, __shfl_xor(mx, 16));
  mx = max(mx, __shfl_xor(mx, 32));
  if (lane < 16) sMax[wave][lane] = mx;
  lds_barrier();  // the table too
#pragma unroll
  for (int w = 0; w < NW; ++w) mx = max(mx, sMax[w][n]);
  if constexpr (MODE == PART_MAX) {
    if (tid < 16) part_of<KS>(t, block, part, parts)[QR * (64 * KS + 1) + tid] = (uint32_t)mx;
    return;
  }
  // requantization keeps the order, so the maximum's is the maximum; a query without keys may have any
  const int32_t rowmax = mx == INT32_MIN ? 0 : qk_requant16(mx, a.qk_m, a.qk_s);
  // The short index where no row maximum wraps and none is so low that saturated scores are near it: the keys that
  // count lie at a distance of 1 at least, the others are taken for such.
  const bool brief = table && a.qk_s >= 1 && a.qk_s < 30 && !__any(rowmax >= 32767 || rowmax < zero - 32768);

  // ---- pass 2: P and P.V over this wave's keys ----
  v4i o[KS][4];
  uint32_t psum = 0u;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[ks][i] = v4i{0, 0, 0, 0};
  // operand i of the products with V: column 64 ks + 4 n + i of the lane group's 16 keys
  auto add_pv = [&](const v4i (&f)[KS][4], const v4i &x) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v4i v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = QUADS ? f[ks][j][i] : f[ks][i][j];
        o[ks][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, v, o[ks][i], 0, 0, 0);
      }
  };
  ScoreIndex ix(a, rowmax, zero);
  ix.flo = 1, ix.fhi = zero;
  auto chunk_brief = [&](int kc, const v4i (&f)[4][KS], const v4i (&v)[KS][4]) {
    v4i s[4], p;
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = scores(f[i]);
    if (tile.whole(kc)) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[i] = (int)pack4(sTable[ix.seen(s[i][0])], sTable[ix.seen(s[i][1])], sTable[ix.seen(s[i][2])], sTable[ix.seen(s[i][3])]);
    } else {
      const uint32_t ok = counted(kc);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[i] = (int)keep_bytes(pack4(sTable[ix.bounded(s[i][0])], sTable[ix.bounded(s[i][1])], sTable[ix.bounded(s[i][2])],
                                     sTable[ix.bounded(s[i][3])]), (ok >> (4 * i)) & 15u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) psum = __builtin_amdgcn_udot4((uint32_t)p[i], 0x01010101u, psum, false);
    add_pv(v, p);
  };
  // Any row maximum, any precision. A P of 128 (a row maximum of 32767 wraps) is too much for the signed product: the
  // rest of it goes in twice.
  auto chunk_any = [&](int kc, const v4i (&f)[4][KS], const v4i (&v)[KS][4]) {
    const uint32_t ok = counted(kc);
    v4i p, rest;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const v4i s = scores(f[i]);
      uint32_t w = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t d = ix.any(s[r]);
        const uint32_t e = table ? (uint32_t)sTable[d] : shift_exp((int32_t)d, a.frac_bits);
        w |= ((ok >> (4 * i + r)) & 1u ? e & 0xffu : 0u) << (8 * r);
      }
      psum = __builtin_amdgcn_udot4(w, 0x01010101u, psum, false);
      p[i] = (int)(w & 0x7f7f7f7fu), rest[i] = (int)((w >> 1) & 0x40404040u);
    }
    add_pv(v, p);
    add_pv(v, rest);
    add_pv(v, rest);
  };
  auto all_chunks = [&](auto chunk) {
    if constexpr (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (wave + NW * i < tile.nch) chunk(tile.at(wave + NW * i), kf[i], vf[i]);
    } else {
#pragma unroll 1
      for (int c = c_lo + wave; c < c_hi; c += NW) {
        load_k(tile.at(c), kf[0]);
        load_v(tile.at(c), vf[0]);
        chunk(tile.at(c), kf[0], vf[0]);
      }
    }
  };
  if (brief)
    all_chunks(chunk_brief);
  else
    all_chunks(chunk_any);

  // ---- the waves' sums meet in LDS: a lane's four products are four columns of a row ----
  psum += (uint32_t)__shfl_xor((int)psum, 16);
  psum += (uint32_t)__shfl_xor((int)psum, 32);
  if (lane < 16) sSum[wave][lane] = psum;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<v4i *>(&sO[wave][(4 * g + r) * OLD + 64 * ks + 4 * n]) =
          v4i{o[ks][0][r], o[ks][1][r], o[ks][2][r], o[ks][3][r]};
  lds_barrier();
  auto sum_of = [&](int at) {
    v4i v = *reinterpret_cast<const v4i *>(&sO[0][at]);
#pragma unroll
    for (int w = 1; w < NW; ++w) v += *reinterpret_cast<const v4i *>(&sO[w][at]);
    return v;
  };
  uint32_t sum = 0;
  if (tid < QR) {
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += sSum[w][tid];
  }
  if constexpr (MODE == PART_SUM) {
    uint32_t *mine = part_of<KS>(t, block, part, parts);
    for (int i = 4 * tid; i < QR * 64 * KS; i += 4 * 64 * NW)
      *reinterpret_cast<v4i *>(mine + i) = sum_of(i / (64 * KS) * OLD + i % (64 * KS));
    if (tid < QR) mine[QR * 64 * KS + tid] = sum;
    return;
  }
  if (tid < QR) sInv[tid] = fisr((int32_t)sum, a.rsqrt_off);
  lds_barrier();
  for (int i = tid; i < rows * words; i += 64 * NW) {
    const int r = by_words(i), d = 4 * (i - r * words);
    uint32_t w = 0;
    if (q0 + r < cnt) {
      const v4i v = sum_of(r * OLD + d);
      const uint32_t sums[4] = {(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3]};
      w = output_word(a, sums, sInv[r]);
    }
    *reinterpret_cast<uint32_t *>(obase + (int64_t)(q0 + r) * a.o_st + d) = w;
  }
}

// Adds the parts of a tile's row and finishes it, a wave a row: lane l has word l % W of parts l / W, l / W + 64 / W, ...,
// four of them on the way at once.
template <int KS>
__global__ __launch_bounds__(256) void attn_window_join_kernel(WindowArgs t, int qblocks, int parts) {
  constexpr int QR = 16, W = 16 * KS, AT_ONCE = 64 / W;
  const AttnArgs &a = t.a;
  const int lane = threadIdx.x & 63, w = lane % W;
  const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), block = blockIdx.y;
  const int q0 = block % qblocks * QR, q = q0 + row, bh = block / qblocks, h = bh % a.H;
  const int64_t b = bh / a.H;
  if (q >= a.Tq) return;
  const int len = t.lengths ? clampi(t.lengths[b], 0, a.Tk) : a.Tk;
  const int cnt = t.counts ? clampi(t.counts[b], 0, a.Tq) : a.Tq;
  uint32_t sums[4] = {0u, 0u, 0u, 0u}, psum = 0u;
  if (q < cnt) {
    Seen seen;
    const Tile tile = tile_of(t, b, len, cnt, min(q0 + (lane & 15), cnt - 1), t.sinks, seen);
    const int share = part_share(tile.nch, parts);
    const int used = max(1, (tile.nch + share - 1) / share);  // parts that have chunks, or the first
    for (int p0 = lane / W; p0 < used; p0 += 4 * AT_ONCE) {
      v4i x[4];
      uint32_t y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t *from = part_of<KS>(t, block, min(p0 + j * AT_ONCE, used - 1), parts);
        x[j] = *reinterpret_cast<const v4i *>(from + row * 64 * KS + 4 * w);
        y[j] = from[QR * 64 * KS + row];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (p0 + j * AT_ONCE < used) {
#pragma unroll
          for (int c = 0; c < 4; ++c) sums[c] += (uint32_t)x[j][c];
          psum += y[j];
        }
    }
#pragma unroll
    for (int m = W; m < 64; m *= 2) {
#pragma unroll
      for (int c = 0; c < 4; ++c) sums[c] += (uint32_t)__shfl_xor((int)sums[c], m);
      psum += (uint32_t)__shfl_xor((int)psum, m);
    }
  }
  if (lane < a.D / 4)
    *reinterpret_cast<uint32_t *>(a.out + b * a.o_sb + (int64_t)q * a.o_st + (int64_t)h * a.D + 4 * lane) =
        q < cnt ? output_word(a, sums, fisr((int32_t)psum, a.rsqrt_off)) : 0u;
}

// One value a lane that is the sum over the 4 * KS lanes of a group: lane c of it gets that of x[c]
template <int CTRL>
__device__ __forceinline__ int32_t swap_add(bool upper, int32_t lower_one, int32_t upper_one) {
  return (upper ? upper_one : lower_one) +
         __builtin_amdgcn_update_dpp(0, upper ? lower_one : upper_one, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ int32_t sums_of_4(const int32_t *x, int lane) {
  const int32_t a = swap_add<0xB1>(lane & 1, x[0], x[1]), b = swap_add<0xB1>(lane & 1, x[2], x[3]);
  return swap_add<0x4E>(lane & 2, a, b);
}
__device__ __forceinline__ int32_t sums_of_8(const int32_t *x, int lane) {
  int32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = swap_add<0x141>(lane & 4, x[i], x[i + 4]);  // lane 7 - c has the other halves
  return sums_of_4(y, lane);
}
__device__ __forceinline__ int32_t lanes_max(int32_t v) {
  v = row16_max(v);
  return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ __forceinline__ int32_t dpp_sum(int32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true);
  return (__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16)) +
         (__builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48));
}
__device__ __forceinline__ int32_t dot16(const v4i &x, const v4i &y, int32_t sum) {
#pragma unroll
  for (int j = 0; j < 4; ++j) sum = __builtin_amdgcn_sdot4(x[j], y[j], sum, false);
  return sum;
}

// Where several blocks share the chunks of a head: the workspace has `chunks` times 64 scores a head, then each part's
// sums of P.V, those of P and the row maximum, in words
constexpr int token_words(int ks) { return 64 * ks + 4; }
__device__ __forceinline__ uint32_t *token_part(const WindowArgs &t, int ks, int blocks, int block, int part, int parts) {
  return t.workspace + t.scores + ((int64_t)block * parts + part) * token_words(ks);
}

// One query a row. Matrix products would have the same 16 rows: here 16 / KS keys are a load of 16 bytes a lane, the
// lanes of a key add up their dot products so that every lane is left with the score of one key of 64, and P is a byte in
// LDS that the lanes of its value find there. Keys are taken in units of 16, those of the first keys and then the
// window's as one list, four units a chunk, the chunks by NW waves in turn. NC > 0: at most NC chunks a wave, whose K and V
// are all requested at the start; else scores wait in LDS for the row maximum. Either way K and V are read once, and that
// is what bounds it: 2560 heads of 64 columns and 2048 keys take 124 us in quads, 5.4 TB/s, and 1024 keys 65.
template <int KS, bool QUADS, int NW, int NC, int MODE>
__global__ __launch_bounds__(64 * NW) void attn_window_token_kernel(WindowArgs t, int blocks, int per_xcd, int chunks) {
  static_assert(MODE == ALL || NC == 0, "parts loop over their chunks");
  constexpr int LOADS = 4 * KS, LPQ = 16 * KS, ACCS = QUADS ? 4 : LOADS, HC = NC > 0 ? NC : 1;
  extern __shared__ int32_t sScores[];
  __shared__ __attribute__((aligned(16))) uint8_t sP[NW][HC][64];
  __shared__ int32_t sMax[NW];
  __shared__ uint32_t sSum[NW];
  __shared__ __attribute__((aligned(16))) uint32_t sO[NW][64 * KS];

  const int block = (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8);
  if (block >= blocks) return;
  const AttnArgs &a = t.a;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = block % a.H, D = a.D;
  const int64_t b = block / a.H;
  const int len = t.lengths ? clampi(t.lengths[b], 0, a.Tk) : a.Tk;
  const int cnt = t.counts ? clampi(t.counts[b], 0, 1) : 1;
  const int8_t *const kbase = a.k + b * a.k_sb + (int64_t)h * a.k_sh;
  const int8_t *const vbase = a.vt + b * a.v_sb + (int64_t)h * a.v_sh;
  const Seen seen = seen_from(t, len, t.positions ? (int64_t)t.positions[b * t.pos_sb] : (int64_t)len - 1);
  const int w0 = seen.start / 16, ns = min((seen.first + 15) / 16, w0);
  const int nu = cnt ? ns + max(0, (seen.end + 15) / 16 - w0) : 0;
  // this block's chunks
  const int parts = MODE == ALL ? 1 : (int)gridDim.y, share = part_share((nu + 3) / 4, parts);
  const int c_lo = MODE == ALL ? 0 : (int)blockIdx.y * share, nch = MODE == ALL ? (nu + 3) / 4 : min(c_lo + share, (nu + 3) / 4);
  uint32_t *const record = MODE == ALL ? nullptr : token_part(t, KS, blocks, block, blockIdx.y, parts);
  int32_t *const scores = MODE == ALL ? sScores : reinterpret_cast<int32_t *>(t.workspace) + (int64_t)block * chunks * 64;
  // the first key of unit u (those past the last repeat it)
  auto unit_at = [&](int u) { return 16 * (u < ns ? u : w0 + u - ns); };
  // the first and last key of the unit from key k0 on that the query sees: no others are read
  auto low = [&](int k0) { return k0 < seen.first ? 0 : max(seen.start - k0, 0); };
  auto high = [&](int k0) { return min((k0 < 16 * w0 ? seen.first : seen.end) - k0, 16) - 1; };

  const int c = lane % LOADS, kk = lane / LOADS, part = lane & 3, n = lane % LPQ, qd = lane / LPQ;
  const uint32_t kcol = (uint32_t)min(16 * c, D - 16), k_st16 = (uint32_t)a.k_st >> 4, v_sq16 = (uint32_t)a.v_sq >> 4;
  auto load_k = [&](int ch, v4i (&f)[LOADS]) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int k0 = unit_at(min(4 * ch + i / KS, nu - 1));
      const int key = clampi(i % KS * 8 + kk, low(k0), high(k0));
      f[i] = *reinterpret_cast<const v4i *>(kbase + k0 * a.k_st + (__umul24(key, k_st16) * 16 + kcol));
    }
  };
  // quads: load i has 4 / KS of them, whole; transposed rows: 16 columns, four units of each
  auto load_v = [&](int ch, v4i (&f)[LOADS]) {
    if constexpr (QUADS) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int k0 = unit_at(min(4 * ch + i / KS, nu - 1));
        const int quad = clampi(i % KS * 2 + qd, low(k0) >> 2, high(k0) >> 2);
        f[i] = *reinterpret_cast<const v4i *>(vbase + (k0 >> 2) * a.v_sq + (__umul24(quad, v_sq16) * 16 + 4 * min(4 * n, D - 4)));
      }
    } else {
      const uint32_t at = (uint32_t)(lane >> 2) * (uint32_t)a.v_sd + (uint32_t)unit_at(min(4 * ch + part, nu - 1));
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        f[i] = *reinterpret_cast<const v4i *>(vbase + 16 * min(i, D / 16 - 1) * a.v_sd + at);
    }
  };

  v4i kf[HC][LOADS], vf[HC][LOADS], qf{0, 0, 0, 0};
  if (16 * c < D) qf = *reinterpret_cast<const v4i *>(a.q + b * a.q_sb + (int64_t)h * D + 16 * c);
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (wave + NW * i < nch) load_k(wave + NW * i, kf[i]);
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (wave + NW * i < nch) load_v(wave + NW * i, vf[i]);
    __builtin_amdgcn_sched_barrier(0);
  }

  // this lane's key of a chunk: its score, INT32_MIN where the query does not see it
  auto score = [&](int ch, const v4i (&f)[LOADS]) {
    int32_t x[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) x[i] = dot16(f[i], qf, 0);
    const int32_t s = KS == 1 ? sums_of_4(x, lane) : sums_of_8(x, lane);
    const int u = 4 * ch + c / KS, key = unit_at(u) + c % KS * 8 + kk;
    return u < nu && ((key >= seen.start && key < seen.end) || key < seen.first) ? s : INT32_MIN;
  };
  int32_t mx = INT32_MIN, held[HC];
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      held[i] = INT32_MIN;
      if (wave + NW * i < nch) held[i] = score(wave + NW * i, kf[i]);
      mx = max(mx, held[i]);
    }
  } else {
    auto one = [&](int ch, const v4i (&f)[LOADS]) {
      const int32_t s = score(ch, f);
      scores[64 * ch + lane] = s;
      mx = max(mx, s);
    };
    if (MODE != PART_SUM) {
      v4i kn[LOADS];
      if (c_lo + wave < nch) load_k(c_lo + wave, kf[0]);
#pragma unroll 1
      for (int ch = c_lo + wave; ch < nch; ch += 2 * NW) {
        if (ch + NW < nch) load_k(ch + NW, kn);
        one(ch, kf[0]);
        if (ch + 2 * NW < nch) load_k(ch + 2 * NW, kf[0]);
        if (ch + NW < nch) one(ch + NW, kn);
      }
    }
    if (MODE != PART_MAX && c_lo + wave < nch) load_v(c_lo + wave, vf[0]);
    if (MODE == PART_SUM)
      for (int p = lane; p < parts; p += 64) mx = max(mx, (int32_t)token_part(t, KS, blocks, block, p, parts)[64 * KS + 1]);
  }
  mx = lanes_max(mx);
  if constexpr (MODE != PART_SUM) {
    if (lane == 0) sMax[wave] = mx;
    lds_barrier();
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = max(mx, sMax[w]);
  }
  if constexpr (MODE == PART_MAX) {
    if (tid == 0) record[64 * KS + 1] = (uint32_t)mx;
    return;
  }
  // requantization keeps the order, so the maximum's is the maximum; a query without keys may have any
  const int32_t rowmax = mx == INT32_MIN ? 0 : qk_requant16(mx, a.qk_m, a.qk_s);
  const bool wraps = rowmax >= 32767;  // a P of 128 is too much for the signed product: the rest of it goes in twice
  const ScoreIndex ix(a, rowmax);

  int32_t acc[ACCS];
  uint32_t psum = 0u;
#pragma unroll
  for (int i = 0; i < ACCS; ++i) acc[i] = 0;
  auto add = [&](int32_t s, const v4i (&f)[LOADS], uint8_t *at) {
    const uint32_t p = s == INT32_MIN ? 0u : shift_exp((int32_t)ix.any(s), a.frac_bits) & 0xffu;
    psum += p;
    at[16 / KS * c + kk] = (uint8_t)p;
    __builtin_amdgcn_wave_barrier();
    auto products = [&](auto of) {
      if constexpr (QUADS) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int32_t w = of(*reinterpret_cast<const int32_t *>(at + 16 / KS * i + 4 * qd));
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_sdot4(f[i][j], w, acc[j], false);
        }
      } else {
        v4i w = *reinterpret_cast<const v4i *>(at + 16 * part);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = of(w[j]);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) acc[i] = dot16(f[i], w, acc[i]);
      }
    };
    products([](int32_t w) { return w & 0x7f7f7f7f; });
    if (wraps) {
      products([](int32_t w) { return (w >> 1) & 0x40404040; });
      products([](int32_t w) { return (w >> 1) & 0x40404040; });
    }
    __builtin_amdgcn_wave_barrier();
  };
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (wave + NW * i < nch) add(held[i], vf[i], sP[wave][i]);
  } else {
    v4i vn[LOADS];
    const int first = c_lo + wave;
    int32_t s0 = first < nch ? scores[64 * first + lane] : 0, s1 = 0;
#pragma unroll 1
    for (int ch = first; ch < nch; ch += 2 * NW) {
      if (ch + NW < nch) load_v(ch + NW, vn), s1 = scores[64 * (ch + NW) + lane];
      add(s0, vf[0], sP[wave][0]);
      if (ch + 2 * NW < nch) load_v(ch + 2 * NW, vf[0]), s0 = scores[64 * (ch + 2 * NW) + lane];
      if (ch + NW < nch) add(s1, vn, sP[wave][0]);
    }
  }

  // the lanes' and then the waves' sums
  psum = (uint32_t)dpp_sum((int32_t)psum);
  if (lane == 0) sSum[wave] = psum;
  if constexpr (QUADS) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (KS == 1) acc[j] += __shfl_xor(acc[j], 16);
      acc[j] += __shfl_xor(acc[j], 32);
    }
    if (lane < LPQ) *reinterpret_cast<v4i *>(&sO[wave][4 * n]) = v4i{acc[0], acc[1], acc[2], acc[3]};
  } else {
#pragma unroll
    for (int i = 0; i < KS; ++i) sO[wave][64 * i + 16 * part + (lane >> 2)] = (uint32_t)sums_of_4(acc + 4 * i, lane);
  }
  lds_barrier();
  if (4 * tid < D) {
    v4i v = *reinterpret_cast<const v4i *>(&sO[0][4 * tid]);
    uint32_t sum = sSum[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += *reinterpret_cast<const v4i *>(&sO[w][4 * tid]), sum += sSum[w];
    if constexpr (MODE == PART_SUM) {
      *reinterpret_cast<v4i *>(record + 4 * tid) = v;
      if (tid == 0) record[64 * KS] = sum;
      return;
    }
    const uint32_t sums[4] = {(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3]};
    *reinterpret_cast<uint32_t *>(a.out + b * a.o_sb + (int64_t)h * D + 4 * tid) =
        output_word(a, sums, fisr((int32_t)sum, a.rsqrt_off));
  }
}

// Adds a head's parts and finishes them (added in memory by the parts and finished by the last of them, the fences
// between dies that this takes made it 47 us in the place of 16 for 32 heads of 4096 keys): a wave a head, lane l has
// word l % W of parts l / W, l / W + 64 / W, ...
template <int KS>
__global__ __launch_bounds__(64) void attn_window_token_join_kernel(WindowArgs t, int parts) {
  constexpr int W = 16 * KS, AT_ONCE = 64 / W;
  const AttnArgs &a = t.a;
  const int lane = threadIdx.x, w = lane % W, block = blockIdx.x, blocks = gridDim.x;
  v4i sum{0, 0, 0, 0};
  uint32_t psum = 0u;
#pragma unroll 4
  for (int p = lane / W; p < parts; p += AT_ONCE) {
    const uint32_t *from = token_part(t, KS, blocks, block, p, parts);
    sum += *reinterpret_cast<const v4i *>(from + 4 * min(w, a.D / 4 - 1));
    psum += from[64 * KS];
  }
#pragma unroll
  for (int m = W; m < 64; m *= 2) {
#pragma unroll
    for (int c = 0; c < 4; ++c) sum[c] += __shfl_xor(sum[c], m);
    psum += (uint32_t)__shfl_xor((int)psum, m);
  }
  const uint32_t sums[4] = {(uint32_t)sum[0], (uint32_t)sum[1], (uint32_t)sum[2], (uint32_t)sum[3]};
  if (lane < a.D / 4)
    *reinterpret_cast<uint32_t *>(a.out + block / a.H * a.o_sb + (int64_t)(block % a.H) * a.D + 4 * lane) =
        output_word(a, sums, fisr((int32_t)psum, a.rsqrt_off));
}

// Word j of lane group g (16 lanes) becomes word g of lane group j
__device__ __forceinline__ void transpose_groups(v4i &p) {
  const auto a = __builtin_amdgcn_permlane32_swap((uint32_t)p[0], (uint32_t)p[2], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)p[1], (uint32_t)p[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  p = v4i{(int)c[0], (int)c[1], (int)d[0], (int)d[1]};
}

// Many queries at the row's last positions: a block has 16 * QT queries of each of its NW waves, whose windows
// follow one another, and every wave goes through the chunks that any of them sees. A chunk is copied to LDS once a
// block, as the register images of the products' operands (1 KB each, a lane's 16 bytes at 16 * lane, so reads have no
// conflicts), a step ahead and without registers. First every chunk's K passes for the maxima, four chunks a step, then K
// and V, two chunks a step (steps of one chunk, three of them in LDS: 143 us in the place of 136 for the case below).
// Row 4g + r of score product i is key 16i + 4g + r: a product is 16 keys in a row, and at a window's borders those
// that no query sees are left out and those that all see need no mask. Byte 4i + r of lane group g's P.V operand is
// that key too, and V in quads has words of four keys. Transposed rows have 16 keys in a row, for which the lane groups
// exchange their words of P.
// A score takes an instruction for the maximum, a multiplication, three simple ones and a byte from the table for its
// value, and P.V next to nothing: the vector units and the ways between them and LDS bound it. 16 rows of 20 heads of 1500
// frames that see 511 and 16 others take 133 us, two thirds of them the vector units' own; its matrix products would
// take 29. It needs its four waves a SIMD: with three and no spilled registers (8 now, 10 with
// quads, between the passes) it takes 167. 128 columns a head have two, as two blocks fill a CU's LDS.
template <int KS, bool QUADS, int QT, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(rows_waves(KS)))) void attn_window_rows_kernel(
    WindowArgs t, int qblocks, int blocks, int per_xcd, int table_off) {
  constexpr int QW = 16 * QT, QR = QW * NW, IMAGES = 4 * KS, IMAGE = 1024, CHUNK = IMAGES * IMAGE, PLACE = 4 * CHUNK;
  static_assert(NW == 4, "each wave copies KS images of K and of V");
  __shared__ __attribute__((aligned(1024))) int8_t sChunk[2 * PLACE];
  __shared__ __attribute__((aligned(16))) uint8_t sTable[kTableBytes];

  const int block = (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8);
  if (block >= blocks) return;
  const AttnArgs &a = t.a;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int q0 = block % qblocks * QR, bh = block / qblocks;
  const int h = bh % a.H;
  const int64_t b = bh / a.H;
  const int D = a.D, N = a.Tq;
  const int len = t.lengths ? clampi(t.lengths[b], 0, a.Tk) : a.Tk;
  const int cnt = t.counts ? clampi(t.counts[b], 0, N) : N;
  const int8_t *const kbase = a.k + b * a.k_sb + (int64_t)h * a.k_sh;
  const int8_t *const vbase = a.vt + b * a.v_sb + (int64_t)h * a.v_sh;
  int8_t *const obase = a.out + b * a.o_sb + (int64_t)h * D;
  // positions rise by one: what the first query sees begins and ends first
  auto seen_by = [&](int q) { return seen_from(t, len, (int64_t)len - cnt + q); };
  const int used = min(q0 + QR, cnt);  // queries of the block that are in use end here
  int nch = 0, ns = 0, w0 = 0;
  if (q0 < used) {
    const Seen first = seen_by(q0), last = seen_by(used - 1);
    w0 = min(first.start, last.end) / 64;
    ns = min((min(t.sinks, last.end) + 63) / 64, w0);
    nch = ns + max(0, (last.end + 63) / 64 - w0);
  }
  auto chunk_at = [&](int c) { return c < ns ? c : w0 + c - ns; };

  // ---- copies to LDS: image j of a chunk's K (keys past the last repeat it, head dims past D the last ones), of its V ----
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>(sChunk));
  // A lane's offsets from a chunk's base are the same in every chunk that ends before the row does.
  const auto k_at = [&](int w, int last) {
    const int j = wave + NW * w, i = j / KS, ks = j % KS;
    return (uint32_t)min(16 * i + n, last) * (uint32_t)a.k_st + (uint32_t)min(64 * ks + 16 * g, D - 16);
  };
  const auto v_at = [&](int w, int last) {  // the chunk's last key
    const int j = wave + NW * w, ks = j / 4, i = j % 4;
    const uint32_t d0 = (uint32_t)min(64 * ks + 4 * n, D - 4);
    return QUADS ? (uint32_t)min(4 * i + g, last >> 2) * (uint32_t)a.v_sq + 4 * d0
                 : (d0 + i) * (uint32_t)a.v_sd + (uint32_t)min(16 * g, last & ~15);
  };
  uint32_t koff[KS], voff[KS];
#pragma unroll
  for (int w = 0; w < KS; ++w) koff[w] = k_at(w, 63), voff[w] = v_at(w, 63);
  auto copy_k = [&](int kc, uint32_t to) {
    const int8_t *base = kbase + (int64_t)(64 * kc) * a.k_st;
    const int last = len - 1 - 64 * kc;
#pragma unroll
    for (int w = 0; w < KS; ++w) dma16_lds(base, last >= 63 ? koff[w] : k_at(w, last), to + IMAGE * (wave + NW * w));
  };
  auto copy_v = [&](int kc, uint32_t to) {
    const int8_t *base = vbase + (QUADS ? (int64_t)(16 * kc) * a.v_sq : (int64_t)(64 * kc));
    const int last = len - 1 - 64 * kc;
#pragma unroll
    for (int w = 0; w < KS; ++w) dma16_lds(base, last >= 63 ? voff[w] : v_at(w, last), to + IMAGE * (wave + NW * w));
  };
  // The first steps have K of four chunks each, the others K and V of two. A barrier says that the copies of its step are
  // there and that every wave is done with the one before, whose place those of the next take.
  const int steps = (nch + 3) / 4, all_steps = steps + (nch + 1) / 2;
  auto copy = [&](int s) {
    const uint32_t to = lds0 + (s & 1) * PLACE;
    if (s < steps) {
#pragma unroll 1
      for (int c = 4 * s; c < min(4 * s + 4, nch); ++c) copy_k(chunk_at(c), to + CHUNK * (c & 3));
    } else {
      const int c0 = 2 * (s - steps);
#pragma unroll 1
      for (int c = c0; c < min(c0 + 2, nch); ++c) {
        copy_k(chunk_at(c), to + 2 * CHUNK * (c & 1));
        copy_v(chunk_at(c), to + 2 * CHUNK * (c & 1) + CHUNK);
      }
    }
  };
  uint32_t from = 0;
  auto arrive = [&](int s) {
    wait_vm<0>();
    lds_barrier();
    if (s + 1 < all_steps) copy(s + 1);
  };

  // ---- queries, and what they see ----
  const int qw = q0 + wave * QW;
  v4i qf[QT][KS];
  Seen seen[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    const int q = max(0, min(qw + 16 * u + n, cnt - 1));  // queries past the count repeat the last one
    seen[u] = seen_by(q);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d0 = 64 * ks + 16 * g;
      qf[u][ks] = v4i{0, 0, 0, 0};
      if (d0 < D) qf[u][ks] = *reinterpret_cast<const v4i *>(a.q + b * a.q_sb + (int64_t)q * a.q_st + (int64_t)h * D + d0);
    }
  }
  const bool table = table_off >= 0;
  const int zero = table ? shift_exp_zero(a.frac_bits) : IW_SEXP_LUT - 1;
  if (table)
    for (int i = 16 * tid; i <= zero; i += 16 * 64 * NW)
      *reinterpret_cast<uint4 *>(sTable + i) = *reinterpret_cast<const uint4 *>(kTables.v + table_off + i);
  if (nch > 0) copy(0);
  // In products of 16 keys: those that any of this wave's queries sees a key of ([p_from, p_to) and below p_first), and
  // those that all see all of ([p_all, p_end))
  const int qe = min(qw + QW, cnt) - 1;
  Seen wf{0, 0, 0}, wl{0, 0, 0};
  if (qw <= qe) wf = seen_by(qw), wl = seen_by(qe);
  const int p_from = wf.start / 16, p_to = (wl.end + 15) / 16, p_first = (wl.first + 15) / 16;
  const int p_all = (wl.start + 15) / 16, p_end = wf.end / 16;
  auto some = [&](int p0, int m) { return (p0 < p_to && p0 + m > p_from) || p0 < p_first; };
  auto whole = [&](int p0, int m) { return p0 >= p_all && p0 + m <= p_end; };
  // which of the four keys from k0 + 4 g on this lane's query of tile u sees; borders that lie elsewhere cost nothing
  auto counted = [&](int p0, int u) -> uint32_t {
    const int k = 16 * p0 + 4 * g;
    uint32_t ok = 15u;
    if (p0 >= p_end) ok = low4(seen[u].end - k);
    if (p0 < p_all) ok &= ~low4(seen[u].start - k);
    if (p0 < p_first) ok |= low4(seen[u].first - k);
    return ok;
  };
  auto image = [&](int j) { return *reinterpret_cast<const v4i *>(&sChunk[from + IMAGE * j + 16 * lane]); };
  auto scores = [&](int i, v4i (&out)[QT]) {
#pragma unroll
    for (int u = 0; u < QT; ++u) out[u] = v4i{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const v4i f = image(i * KS + ks);
#pragma unroll
      for (int u = 0; u < QT; ++u) out[u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, qf[u][ks], out[u], 0, 0, 0);
    }
  };

  // ---- pass 1: row maximum of the raw scores ----
  int32_t mx[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) mx[u] = INT32_MIN;
  auto more = [&](const v4i (&x)[QT]) {
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      mx[u] = max(max(mx[u], x[u][0]), x[u][1]);
      mx[u] = max(max(mx[u], x[u][2]), x[u][3]);
    }
  };
#pragma unroll 1
  for (int s = 0; s < nch; ++s) {
    if ((s & 3) == 0) arrive(s / 4);
    from = (s / 4 & 1) * PLACE + CHUNK * (s & 3);
    const int p0 = 4 * chunk_at(s);
    if (!some(p0, 4)) continue;
    if (whole(p0, 4)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v4i x[QT];
        scores(i, x);
        more(x);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (some(p0 + i, 1)) {
          v4i x[QT];
          scores(i, x);
          if (!whole(p0 + i, 1)) {
#pragma unroll
            for (int u = 0; u < QT; ++u) {
              const uint32_t off = ~counted(p0 + i, u);
#pragma unroll
              for (int r = 0; r < 4; ++r) x[u][r] = hide(x[u][r], off, r);
            }
          }
          more(x);
        }
    }
  }
  int32_t rowmax[QT];
  bool sat = false;
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    mx[u] = max(mx[u], __shfl_xor(mx[u], 16));
    mx[u] = max(mx[u], __shfl_xor(mx[u], 32));
    // requantization keeps the order, so the maximum's is the maximum; a query without keys may have any
    rowmax[u] = mx[u] == INT32_MIN ? 0 : qk_requant16(mx[u], a.qk_m, a.qk_s);
    sat = sat || rowmax[u] >= 32767 || rowmax[u] < zero - 32768;
  }
  // The short index where no row maximum wraps and none is so low that saturated scores are near it: the keys that
  // count lie at a distance of 1 at least, the others are taken for such.
  const bool brief = table && a.qk_s >= 1 && a.qk_s < 30 && !__any(sat);

  // ---- pass 2: P and P.V ----
  v4i o[QT][KS][4];
  uint32_t psum[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    psum[u] = 0u;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[u][ks][i] = v4i{0, 0, 0, 0};
  }
  // operand c of the products with V: columns 64 ks + 4 n + c
  auto v_operands = [&](int ks, v4i (&v)[4]) {
    v4i f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = image(IMAGES + 4 * ks + i);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[c][i] = QUADS ? f[i][c] : f[c][i];
  };
  auto add_pv = [&](v4i (&x)[QT]) {
#pragma unroll
    for (int u = 0; u < QT; ++u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) psum[u] = __builtin_amdgcn_udot4((uint32_t)x[u][i], 0x01010101u, psum[u], false);
      if (!QUADS) transpose_groups(x[u]);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      v4i v[4];
      v_operands(ks, v);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int u = 0; u < QT; ++u)
          o[u][ks][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[u], v[c], o[u][ks][c], 0, 0, 0);
    }
  };
  ScoreIndex ix(a, 0, zero);
  ix.flo = 1, ix.fhi = zero;
  int32_t K[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) K[u] = ScoreIndex(a, rowmax[u], zero).fK;
  auto values = [&](const v4i &x, int u) {
    ix.fK = K[u];
    return pack4(sTable[ix.seen(x[0])], sTable[ix.seen(x[1])], sTable[ix.seen(x[2])], sTable[ix.seen(x[3])]);
  };
  auto some_values = [&](const v4i &x, int u) {
    ix.fK = K[u];
    return pack4(sTable[ix.bounded(x[0])], sTable[ix.bounded(x[1])], sTable[ix.bounded(x[2])], sTable[ix.bounded(x[3])]);
  };
#pragma unroll 1
  for (int s = 0; s < nch; ++s) {
    if ((s & 1) == 0) arrive(steps + s / 2);
    from = (steps + s / 2 & 1) * PLACE + 2 * CHUNK * (s & 1);
    const int p0 = 4 * chunk_at(s);
    if (!some(p0, 4)) continue;
    v4i p[QT];
    if (brief) {
      if (whole(p0, 4)) {
        v4i x[2][QT];
        scores(0, x[0]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i < 3) scores(i + 1, x[(i + 1) & 1]);
#pragma unroll
          for (int u = 0; u < QT; ++u) p[u][i] = (int)values(x[i & 1][u], u);
        }
      } else {
#pragma unroll
        for (int u = 0; u < QT; ++u) p[u] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (some(p0 + i, 1)) {
            v4i x[QT];
            scores(i, x);
#pragma unroll
            for (int u = 0; u < QT; ++u) p[u][i] = (int)keep_bytes(some_values(x[u], u), counted(p0 + i, u));
          }
      }
      add_pv(p);
    } else {
      // Any row maximum, any precision, a tile at a time. A P of 128 (a row maximum of 32767 wraps) is too much for
      // the signed product: the rest of it goes in twice.
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        const ScoreIndex at(a, rowmax[u], zero);
        v4i p1, rest;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v4i x{0, 0, 0, 0};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            x = __builtin_amdgcn_mfma_i32_16x16x64_i8(image(i * KS + ks), qf[u][ks], x, 0, 0, 0);
          const uint32_t ok = counted(p0 + i, u);
          uint32_t w = 0;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t d = at.any(x[r]);
            const uint32_t e = table ? (uint32_t)sTable[d] : shift_exp((int32_t)d, a.frac_bits);
            w |= ((ok >> r) & 1u ? e & 0xffu : 0u) << (8 * r);
          }
          psum[u] = __builtin_amdgcn_udot4(w, 0x01010101u, psum[u], false);
          p1[i] = (int)(w & 0x7f7f7f7fu), rest[i] = (int)((w >> 1) & 0x40404040u);
        }
        if (!QUADS) transpose_groups(p1), transpose_groups(rest);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          v4i v[4];
          v_operands(ks, v);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            v4i &to = o[u][ks][c];
            to = __builtin_amdgcn_mfma_i32_16x16x64_i8(p1, v[c], to, 0, 0, 0);
            to = __builtin_amdgcn_mfma_i32_16x16x64_i8(rest, v[c], to, 0, 0, 0);
            to = __builtin_amdgcn_mfma_i32_16x16x64_i8(rest, v[c], to, 0, 0, 0);
          }
        }
      }
    }
  }

  // a lane group finds the roots of one tile's queries: group u those of tile u
  const Finish fin(a);
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    psum[u] += (uint32_t)__shfl_xor((int)psum[u], 16);
    psum[u] += (uint32_t)__shfl_xor((int)psum[u], 32);
  }
  uint32_t mine = psum[0];
#pragma unroll
  for (int u = 1; u < QT; ++u) mine = g == u ? psum[u] : mine;
  const int32_t inv = fisr((int32_t)mine, a.rsqrt_off);
  const bool fast = fin.brief && !__any((inv << 8) >> 8 != inv);
#pragma unroll
  for (int u = 0; u < QT; ++u)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      finish_row<KS>(t, fin, obase, qw + 16 * u + 4 * g + r, cnt, o[u], r, __shfl(inv, 16 * u + 4 * g + r), fast, n);
}

template <int KS, bool QUADS, int QT>
int launch_window_rows(const WindowArgs &t, hipStream_t s) {
  constexpr int NW = 4;
  const int64_t qblocks = (t.a.Tq + 16 * QT * NW - 1) / (16 * QT * NW), blocks = qblocks * t.a.B * t.a.H;
  const int64_t per_xcd = (blocks + 7) / 8;
  const int table = t.a.frac_bits <= kTableBits ? table_at(t.a.frac_bits) : -1;
  if (8 * per_xcd * 64 * NW >= 1LL << 32) return fail("too many heads and queries for one call");
  hipLaunchKernelGGL((attn_window_rows_kernel<KS, QUADS, QT, NW>), dim3((unsigned)(8 * per_xcd)), dim3(64 * NW), 0, s, t,
                     (int)qblocks, (int)blocks, (int)per_xcd, table);
  return check_launch("attn_window_rows_kernel");
}

template <int KS, bool QUADS, int NW, int NC, int MODE = ALL>
int launch_window(const WindowArgs &t, hipStream_t s, int parts = 1) {
  const int64_t qblocks = (t.a.Tq + 15) / 16, blocks = qblocks * t.a.B * t.a.H;
  const int64_t per_xcd = (blocks + 7) / 8;
  const int words = t.a.D / 4, per_word = (65536 + words - 1) / words;
  const int table = t.a.frac_bits <= kTableBits ? table_at(t.a.frac_bits) : -1;
  // a grid has fewer than 2^32 threads
  if (8 * per_xcd * 64 * NW >= 1LL << 32) return fail("too many heads and queries for one call");
  hipLaunchKernelGGL((attn_window_kernel<KS, QUADS, NW, NC, MODE>), dim3((unsigned)(8 * per_xcd), (unsigned)parts),
                     dim3(64 * NW), 0, s, t, (int)qblocks, (int)blocks, (int)per_xcd, per_word, table);
  return check_launch("attn_window_kernel");
}

template <int KS, bool QUADS, int NW, int NC, int MODE = ALL>
int launch_window_token(const WindowArgs &t, int64_t chunks, hipStream_t s, int parts = 1) {
  const int64_t blocks = (int64_t)t.a.B * t.a.H, per_xcd = (blocks + 7) / 8;
  if (8 * per_xcd * 64 * NW >= 1LL << 32) return fail("too many heads and queries for one call");
  hipLaunchKernelGGL((attn_window_token_kernel<KS, QUADS, NW, NC, MODE>), dim3((unsigned)(8 * per_xcd), (unsigned)parts),
                     dim3(64 * NW), NC > 0 || MODE != ALL ? 0 : (unsigned)(256 * chunks), s, t, (int)blocks, (int)per_xcd, (int)chunks);
  return check_launch("attn_window_token_kernel");
}

template <int KS, bool QUADS>
int launch_token_parts(WindowArgs t, int64_t chunks, int parts, hipStream_t s) {
  const int64_t blocks = (int64_t)t.a.B * t.a.H;
  t.scores = blocks * chunks * 64;
  int rc = launch_window_token<KS, true, 8, 0, PART_MAX>(t, chunks, s, parts);  // reads K only
  if (rc == 0) rc = launch_window_token<KS, QUADS, 8, 0, PART_SUM>(t, chunks, s, parts);
  if (rc) return rc;
  hipLaunchKernelGGL((attn_window_token_join_kernel<KS>), dim3((unsigned)blocks), dim3(64), 0, s, t, parts);
  return check_launch("attn_window_token_join_kernel");
}

template <int KS, bool QUADS>
int launch_window_parts(const WindowArgs &t, int parts, hipStream_t s) {
  int rc = launch_window<KS, true, 8, 0, PART_MAX>(t, s, parts);  // reads K only
  if (rc == 0) rc = launch_window<KS, QUADS, 8, 0, PART_SUM>(t, s, parts);
  if (rc) return rc;
  const int qblocks = (t.a.Tq + 15) / 16;
  hipLaunchKernelGGL((attn_window_join_kernel<KS>), dim3(4, (unsigned)(qblocks * t.a.B * t.a.H)), dim3(256), 0, s, t,
                     qblocks, parts);
  return check_launch("attn_window_join_kernel");
}

// The most chunks that a tile of queries has, whatever the lengths: its windows (16 queries at positions that
// follow one another, or one at any) from any key on, and the first keys.
int64_t most_chunks(int64_t queries, int64_t cap, int64_t before, int64_t after, int64_t sinks) {
  const int64_t keys = std::min(cap, before + after + std::min<int64_t>(queries, 16));
  return std::min((cap + 63) / 64, (keys + 62) / 64 + 1 + (std::min(sinks, cap) + 63) / 64);
}

// Blocks that share the chunks of a tile. Three launches and the sums' way through memory are worth it where each
// block is left with much less. 20 queries of heads of 64 columns, us in a block of 8 waves a tile and in parts:
//   tiles x parts    4096 keys      8192 keys      16384 keys
//   16 x 8 to 16     14.6, 12.2     23.8, 12.8     45.0, 15.9
//   64 x 4           16.7, 15.8     27.7, 19.6     49.6, 27.2
//   128 x 2          17.8, 20.0     29.8, 27.6     59.1, 43.6
// and of 128 columns 2048 keys: 26.5 and 15.6 for 16 tiles, 27.4 and 19.5 for 64, 27.8 and 25.0 for 128 (1024 keys: 16.4
// in one).
constexpr int kCus = 256;
int window_parts(int64_t heads, int64_t queries, int64_t head_dim, int64_t cap, int64_t before, int64_t after, int64_t sinks) {
  if (cap < 1024) return 1;
  const int64_t blocks = heads * ((queries + 15) / 16), chunks = most_chunks(queries, cap, before, after, sinks);
  const int64_t parts = std::min(kCus / blocks, (chunks + 7) / 8);
  return parts > 1 && parts * chunks > (head_dim <= 64 ? 256 : 64) ? (int)parts : 1;
}

// Chunks of one query: of keys in units of 16
int64_t token_chunks(int64_t cap, int64_t before, int64_t after, int64_t sinks) {
  const int64_t units = (std::min(cap, before + after + 1) + 14) / 16 + 1 + (std::min(sinks, cap) + 15) / 16;
  return (std::min((cap + 15) / 16, units) + 3) / 4;
}
constexpr int64_t kTokenScores = 224;  // chunks whose scores fit a block's LDS
// Blocks that share the chunks of one query's head, us in one block of 8 waves and so, 64 columns a head:
//   heads x parts    2048 keys      4096 keys      8192 keys
//   8 x 5 to 17      7.9, 9.6       11.4, 10.0     18.4, 9.9
//   32 x 8           7.9, 10.1      14.9, 11.7     26.0, 15.2
//   64 x 4           9.5, 11.8      15.3, 15.2     25.7, 19.9
//   120 x 2          10.8, 15.0     16.7, 20.7     37.6, 36.0
// (128 columns, 32 heads: 12.4 and 12.9, 21.3 and 16.1, 37.6 and 20.5)
int token_parts(int64_t heads, int64_t chunks) {
  const int64_t parts = std::min(kCus / heads, (chunks + 7) / 8);
  return parts > 1 && parts * chunks > 256 ? (int)parts : 1;
}

// Which of the kernels, with the same results. Queries at the last positions share chunks in LDS where 64 of them a block
// fill the device: heads of 128 columns from a block a CU on, of 64 columns from one and a half (us of a block a 16-query
// tile and so, windows of 512 keys, with 64 and 128 columns: 20 heads of 1500 queries, 480 blocks, 29 and 19, 54 and
// 26; 64 of 300, 320 blocks, 11.5 and 12.9, 22 and 16; 64 of 128, 128 blocks, 9.5 and 15.7, 18 and 23), but not
// for 32 queries or fewer (1280 heads of 32: 40 and 41, 81 and 79; of 64: 63 and 43, 139 and 81).
// Two tiles a wave pay where windows are longer and their 128 queries a block fill the device too (320 heads of 1500
// queries with 64 and 128 columns, one tile and two: 256 keys 107 and 92, 223 and 179; 512 keys 150 and 122, 324 and 245;
// 1280 of 300 with 128 keys 66 and 68, 131 and 124; of 64 with 512 keys, half of a block, 43 and 51, 81 and 102). Blocks of
// 128 columns are two to a CU with either, whose LDS they fill.
// One query has its own kernel, a wave a chunk where there are few (quads, 64 columns, us with this and with the next: 20
// heads of 128 keys, 4.5 and 5.3, of 384 keys, 5.3 and 5.9; 2560 heads of them 12.0 and 15.9, 23.0 and 26.8), else eight
// waves (1024 keys, 20 heads 7.0 and 7.8, 2560 heads 65 and 85; four waves 8.4 and 68, sixteen 7.5 and 74).
// Else a wave holds its chunks where they are few: 8 queries of 20 heads of 64, 128 keys, 5.5 us in a loop and 5.5 so, 2560
// heads of 16 keys 14.2 and 12.5; 256 keys, two chunks a wave, 6.4 and 6.1. Eight waves take long windows
// faster if there are few tiles: 1024 keys, 20 heads 9.1 and 7.8, 256 heads 12.1 and 11.1, 640 heads 22.7 and 25.4.
template <int KS, bool QUADS>
int launch_form(const WindowArgs &t, hipStream_t s) {
  const int64_t heads = (int64_t)t.a.B * t.a.H, tiles = (t.a.Tq + 15) / 16;
  if (!t.positions && t.a.Tq > 32) {
    if (std::min<int64_t>(t.before + t.after, t.a.Tk) >= 3 * 64 && t.a.Tq > 96 && heads * ((tiles + 7) / 8) >= kCus)
      return launch_window_rows<KS, QUADS, 2>(t, s);
    if (2 * heads * ((tiles + 3) / 4) >= (KS == 1 ? 3 : 2) * kCus) return launch_window_rows<KS, QUADS, 1>(t, s);
  }
  if (t.a.Tq == 1) {
    const int64_t chunks = token_chunks(t.a.Tk, t.before, t.after, t.sinks);
    const int parts = token_parts(heads, chunks);
    if (parts > 1) return launch_token_parts<KS, QUADS>(t, chunks, parts, s);
    if (chunks <= 1) return launch_window_token<KS, QUADS, 1, 1>(t, chunks, s);
    if (chunks <= 4) return launch_window_token<KS, QUADS, 4, 1>(t, chunks, s);
    if (chunks <= 8) return launch_window_token<KS, QUADS, 8, 1>(t, chunks, s);
    if (chunks <= kTokenScores) return launch_window_token<KS, QUADS, 8, 0>(t, chunks, s);
  }
  const int parts = window_parts(heads, t.a.Tq, t.a.D, t.a.Tk, t.before, t.after, t.sinks);
  if (parts > 1) return launch_window_parts<KS, QUADS>(t, parts, s);
  const int64_t any = (t.a.Tk + 63) / 64;  // queries at positions that need not follow one another
  const int64_t most = t.positions && t.a.Tq > 1 ? any : most_chunks(t.a.Tq, t.a.Tk, t.before, t.after, t.sinks);
  if (most <= 4) return launch_window<KS, QUADS, 4, 1>(t, s);
  if (most <= 8) return launch_window<KS, QUADS, 4, 2>(t, s);
  return heads * tiles <= kCus ? launch_window<KS, QUADS, 8, 0>(t, s) : launch_window<KS, QUADS, 4, 0>(t, s);
}

}  // namespace

int64_t attn_window_workspace(int64_t heads, int64_t queries, int64_t head_dim, int64_t cap, int64_t before,
                              int64_t after, int64_t sinks) {
  if (queries == 1) {
    const int64_t chunks = token_chunks(cap, before, after, sinks);
    const int parts = token_parts(heads, chunks);
    if (parts > 1) return 4 * heads * (64 * chunks + parts * token_words(head_dim <= 64 ? 1 : 2));
    if (chunks <= kTokenScores) return 0;
  }
  const int64_t parts = window_parts(heads, queries, head_dim, cap, before, after, sinks);
  return parts == 1 ? 0 : 4 * heads * ((queries + 15) / 16) * parts * part_words(head_dim <= 64 ? 1 : 2);
}

int launch_attn_window(const WindowArgs &t, hipStream_t s) {
  const bool quads = t.a.v_sq != 4;
  if (t.a.D <= 64) return quads ? launch_form<1, true>(t, s) : launch_form<1, false>(t, s);
  return quads ? launch_form<2, true>(t, s) : launch_form<2, false>(t, s);
}

}  // namespace iw
