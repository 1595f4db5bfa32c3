// Attention of a tree of drafted tokens over an int8 KV cache: node i of row b
// attends to the row's cached keys 0 .. lengths[b] - 1 and to the nodes that
// its visibility word names (its ancestors and itself), whose K and V are read
// where the projection left them. The arithmetic per (query, key) is that of
// the other integer attention kernels: the requantized scores' row maximum
// first, then P = E(S - rowmax - 1), sum P and P.V, exact modulo 2^32 in any
// order, so the keys can be split over waves.
//
// One block per (batch, head) and 16 or 32 nodes (one or two 16-query MFMA tiles). The
// block's waves take 64-key chunks in turn, the tree itself is one more chunk; their sums
// meet in LDS as whole words, a copy each (added there one by one, 64 nodes of 2560
// heads took 67 us in the place of 53).
// In a chunk's four 16x16x64 score products, row 4g + r of product t is key
// 16g + 4t + r: lane group g then holds the scores of the 16 consecutive keys
// that its bytes of the P.V operand stand for, and no lane exchange is needed.
// V's columns go to the products as d = 4n + c (lane n, product c): a lane
// reads whole words, and its four sums are one word of the output.
//
// The shift exponential is 0 from a distance of about 4.9 * 2^frac_bits on. Up to
// frac_bits 10 the distances below that are read from a table that the block
// copies to LDS while its K and V are on the way (1249 bytes at 8, 4988 at 10);
// beyond, each score computes its own.
//
// Where a long cache meets few heads, several blocks share the keys of a block's
// nodes: a first launch leaves each part's row maxima in the workspace, a second
// each part's sums, a third adds them.
#include <algorithm>

#include "iw_attn_dev.hpp"
#include "iw_common.hpp"
#include "iw_tree.hpp"

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

// A part in the workspace: the sums of P.V of its rows, those of P, the row maxima
constexpr int64_t part_words(int ks, int qt) { return 16 * qt * (64 * ks + 2); }
template <int KS, int QT>
__device__ __forceinline__ uint32_t *part_of(const TreeArgs &t, int block, int part, int parts) {
  return t.workspace + ((int64_t)block * parts + part) * part_words(KS, QT);
}
// chunks of a part, of the nkc cached ones and the tree's
__device__ __forceinline__ int part_share(int nkc, int parts) { return (nkc + parts) / parts; }

// Of all keys, or of blockIdx.y's part of them: the row maxima, or with every part's maxima the sums
enum { ALL, PART_MAX, PART_SUM };

// KS: 64-column parts of the head; QUADS: V in key quads; QT: 16-query tiles of
// the block; NW waves; NC > 0: a wave has at most NC chunks, whose K and V
// are all requested at the start and kept. Waves per SIMD are asked for where the
// registers allow them: held chunks of 64-wide heads in 128 registers, which the compiler
// exceeds on its own (206, two waves: 16 nodes of 2560 heads 38 us, with four 28).
constexpr int tree_waves(int ks, int qt, int nc, int mode) {
  if (mode == PART_MAX) return 4;
  if (nc == 2) return ks == 1 ? (qt == 1 ? 4 : 3) : 2;
  return nc == 1 || ks * qt == 1 ? 4 : 2;
}
template <int KS, bool QUADS, int QT, int NW, int NC, int MODE>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(tree_waves(KS, QT, NC, MODE)))) void attn_tree_kernel(
    TreeArgs t, int qblocks, int blocks, int per_xcd, int per_word, int table_off) {
  constexpr int QR = 16 * QT, OLD = 64 * KS + 4, HC = NC > 0 ? NC : 1;
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
  const int len = clampi(t.lengths[b], 0, a.Tk);
  const int cnt = t.counts ? clampi(t.counts[b], 0, N) : N;
  const int nkc = (len + 63) / 64;  // cached chunks; chunk nkc is the tree
  const int parts = MODE == ALL ? 1 : (int)gridDim.y, part = MODE == ALL ? 0 : (int)blockIdx.y;
  const int share = part_share(nkc, parts);
  // this block's cached chunks, and whether the tree is its too
  const int c_lo = part * share, c_hi = min(c_lo + share, nkc);
  const bool has_tree = c_lo <= nkc && c_lo + share > nkc;
  const int8_t *const kbase = a.k + b * a.k_sb + (int64_t)h * a.k_sh;
  const int8_t *const vbase = a.vt + b * a.v_sb + (int64_t)h * a.v_sh;
  const int8_t *const knew = t.kn + b * t.kn_sb + (int64_t)h * D;
  const int8_t *const vnew = t.vn + b * t.vn_sb + (int64_t)h * D;
  int8_t *const obase = a.out + b * a.o_sb + (int64_t)h * D;
  const int words = D / 4, rows = min(N - q0, QR);
  // i / words for the i < 2^11 of the output
  const auto by_words = [&](int i) { return (int)__umul24(i, per_word) >> 16; };

  if (MODE != ALL && (q0 >= cnt || c_lo > nkc)) return;
  if (q0 >= cnt) {  // no node of these is in use
    for (int i = tid; i < rows * words; i += 64 * NW) {
      const int q = by_words(i);
      *reinterpret_cast<uint32_t *>(obase + (int64_t)(q0 + q) * a.o_st + 4 * (i - q * words)) = 0u;
    }
    return;
  }

  const int nfk = len / 64;  // chunks in which every key counts

  // The K operands of chunk c: keys past the last repeat it, head dims past D the
  // last ones (the query is zero there). A chunk's base is uniform, its lanes'
  // offsets fit 32 bits.
  const int kcol = 16 * g, key0 = 16 * (n >> 2) + (n & 3);
  auto load_k = [&](int c, bool tree, v4i (&f)[4][KS]) {
    const uint32_t st = (uint32_t)(tree ? t.kn_st : a.k_st);
    const int8_t *base = tree ? knew : kbase + (int64_t)(64 * c) * a.k_st;
    const int last = (tree ? cnt : len - 64 * c) - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        f[i][ks] = *reinterpret_cast<const v4i *>(base + ((uint32_t)min(key0 + 4 * i, last) * st +
                                                          (uint32_t)min(64 * ks + kcol, D - 16)));
  };
  // What the V operands are made of: quads and transposed rows hold words of four
  // keys of one column, the tree's rows (word j of f[i] from node 16 g + 4 j + i) four
  // columns. Columns past D repeat the last ones; their sums are not stored.
  auto load_v = [&](int c, bool tree, int ks, v4i (&f)[4]) {
    const uint32_t d0 = (uint32_t)min(64 * ks + 4 * n, D - 4);
    if (tree) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          f[i][j] = *reinterpret_cast<const int32_t *>(
              vnew + ((uint32_t)min(16 * g + 4 * j + i, cnt - 1) * (uint32_t)t.vn_st + d0));
    } else if (QUADS) {
      const int8_t *base = vbase + (int64_t)(16 * c) * a.v_sq;
      const int last = ((len - 1) >> 2) - 16 * c;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = *reinterpret_cast<const v4i *>(base + ((uint32_t)min(4 * g + j, last) * (uint32_t)a.v_sq + 4 * d0));
    } else {
      const int8_t *base = vbase + 64 * c;
      const uint32_t at = (uint32_t)min(16 * g, (len - 1 - 64 * c) & ~15);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        f[i] = *reinterpret_cast<const v4i *>(base + ((d0 + i) * (uint32_t)a.v_sd + at));
    }
  };
  // the operand of product i: column 64 ks + 4 n + i of the lane group's 16 keys
  auto v_operands = [&](bool tree, const v4i (&f)[4], v4i (&o)[4]) {
    if (tree) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t in[4] = {(uint32_t)f[0][j], (uint32_t)f[1][j], (uint32_t)f[2][j], (uint32_t)f[3][j]};
        uint32_t x[4];
        transpose4(in, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i][j] = (int)x[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = QUADS ? f[j][i] : f[i][j];
    }
  };

  // ---- everything that the start can ask for ----
  v4i kf[HC][4][KS], vf[HC][KS][4];
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = wave + NW * i;
      if (c <= nkc) load_k(c, c == nkc, kf[i]);
    }
  }
  v4i qf[QT][KS];
  uint64_t vis[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    const int q = min(q0 + 16 * u + n, cnt - 1);  // queries past the count repeat the last one
    vis[u] = t.visible[b * t.vis_sb + q];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d0 = 64 * ks + 16 * g;
      qf[u][ks] = v4i{0, 0, 0, 0};
      if (d0 < D) qf[u][ks] = *reinterpret_cast<const v4i *>(a.q + b * a.q_sb + (int64_t)q * a.q_st + (int64_t)h * D + d0);
    }
  }
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = wave + NW * i;
      if (c <= nkc) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) load_v(c, c == nkc, ks, vf[i][ks]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  const bool table = table_off >= 0;
  const int zero = table ? shift_exp_zero(a.frac_bits) : IW_SEXP_LUT - 1;
  if (MODE != PART_MAX && table)
    for (int i = 16 * tid; i <= zero; i += 16 * 64 * NW)
      *reinterpret_cast<uint4 *>(sTable + i) = *reinterpret_cast<const uint4 *>(kTables.v + table_off + i);

  auto scores = [&](const v4i (&f)[KS], int u) {
    v4i s{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[ks], qf[u][ks], s, 0, 0, 0);
    return s;
  };
  // which of the lane group's 16 keys of chunk c count for this lane's query of tile u
  const uint64_t in_use = cnt == 64 ? ~0ull : (1ull << cnt) - 1;
  auto counted = [&](int c, bool tree, int u) -> uint32_t {
    if (tree) return (uint32_t)((vis[u] & in_use) >> (16 * g)) & 0xffffu;
    return (1u << clampi(len - 64 * c - 16 * g, 0, 16)) - 1u;
  };
  // ---- pass 1: row maximum of the raw scores ----
  int32_t mx[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) mx[u] = INT32_MIN;
  auto chunk_max = [&](int c, bool tree, const v4i (&f)[4][KS]) {
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      if (c < nfk) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v4i s = scores(f[i], u);
          mx[u] = max(max(mx[u], s[0]), s[1]);
          mx[u] = max(max(mx[u], s[2]), s[3]);
        }
      } else {
        const uint32_t ok = counted(c, tree, u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v4i s = scores(f[i], u);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if ((ok >> (4 * i + r)) & 1u) mx[u] = max(mx[u], s[r]);
        }
      }
    }
  };
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = wave + NW * i;
      if (c <= nkc) chunk_max(c, c == nkc, kf[i]);
    }
  } else if constexpr (MODE != PART_SUM) {
    v4i kn[4][KS];
#pragma unroll 1
    for (int c = c_lo + wave; c < c_hi; c += 2 * NW) {
      load_k(c, false, kf[0]);
      if (c + NW < c_hi) load_k(c + NW, false, kn);
      chunk_max(c, false, kf[0]);
      if (c + NW < c_hi) chunk_max(c + NW, false, kn);
    }
    if (has_tree && (nkc - c_lo) % NW == wave) {
      load_k(nkc, true, kf[0]);
      chunk_max(nkc, true, kf[0]);
    }
  }
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    if (MODE == PART_SUM)  // the maxima of the parts that have chunks, shared out to the waves' lane groups
      for (int p = NW * g + wave; p * share <= nkc; p += 4 * NW)
        mx[u] = max(mx[u], (int32_t)part_of<KS, QT>(t, block, p, parts)[QR * (64 * KS + 1) + 16 * u + n]);
    mx[u] = max(mx[u], __shfl_xor(mx[u], 16));
    mx[u] = max(mx[u], __shfl_xor(mx[u], 32));
    if (lane < 16) sMax[wave][16 * u + lane] = mx[u];
  }
  lds_barrier();
  int32_t rowmax[QT];
  bool sat = false;
#pragma unroll
  for (int u = 0; u < QT; ++u) {
#pragma unroll
    for (int w = 0; w < NW; ++w) mx[u] = max(mx[u], sMax[w][16 * u + n]);
    if constexpr (MODE == PART_MAX) {
      if (tid < 16) part_of<KS, QT>(t, block, part, parts)[QR * (64 * KS + 1) + 16 * u + tid] = (uint32_t)mx[u];
      continue;
    }
    // requantization keeps the order, so the maximum's is the maximum
    rowmax[u] = mx[u] == INT32_MIN ? -32768 : qk_requant16(mx[u], a.qk_m, a.qk_s);
    sat = sat || rowmax[u] >= 32767;
  }
  if constexpr (MODE == PART_MAX) return;
  // the short index where no row maximum wraps: the keys that count lie at a
  // distance of 1 at least, the others are taken for such
  const bool brief = table && !__any(sat);

  // ---- pass 2: P and P.V over this wave's keys ----
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
  // P of chunk c as the operands of its products; hi where a P of 128 (a row maximum
  // of 32767 wraps) is left out, as the product is signed: it goes in as twice 64
  auto chunk_p = [&](int c, bool tree, const v4i (&f)[4][KS], v4i (&p)[QT], v4i (&hi)[QT]) {
    bool any_hi = false;
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      ScoreIndex ix(a, rowmax[u], zero);
      ix.flo = max(ix.flo, 1);
      if (brief) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v4i s = scores(f[i], u);
          p[u][i] = (int)((uint32_t)sTable[ix.full(s[0])] | (uint32_t)sTable[ix.full(s[1])] << 8 |
                          (uint32_t)sTable[ix.full(s[2])] << 16 | (uint32_t)sTable[ix.full(s[3])] << 24);
        }
        if (c >= nfk) {
          const uint32_t ok = counted(c, tree, u);
#pragma unroll
          for (int i = 0; i < 4; ++i) p[u][i] &= (int)byte_mask((ok >> (4 * i)) & 15u);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) psum[u] = __builtin_amdgcn_udot4((uint32_t)p[u][i], 0x01010101u, psum[u], false);
      } else {
        const uint32_t ok = counted(c, tree, u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v4i s = scores(f[i], u);
          uint32_t w = 0;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t d = ix.any(s[r]);
            const uint32_t e = table ? (uint32_t)sTable[d] : shift_exp((int32_t)d, a.frac_bits);
            w |= ((ok >> (4 * i + r)) & 1u ? e & 0xffu : 0u) << (8 * r);
          }
          psum[u] = __builtin_amdgcn_udot4(w, 0x01010101u, psum[u], false);
          p[u][i] = (int)(w & 0x7f7f7f7fu), hi[u][i] = (int)((w >> 1) & 0x40404040u);
        }
        any_hi = any_hi || (hi[u][0] | hi[u][1] | hi[u][2] | hi[u][3]) != 0;
      }
    }
    return __any(any_hi) != 0;
  };
  auto chunk_pv = [&](bool tree, int ks, const v4i (&vr)[4], const v4i (&p)[QT], const v4i (&hi)[QT], bool any_hi) {
    v4i v[4];
    v_operands(tree, vr, v);
    auto pv = [&](const v4i (&x)[QT]) {
#pragma unroll
      for (int u = 0; u < QT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          o[u][ks][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[u], v[i], o[u][ks][i], 0, 0, 0);
    };
    pv(p);
    if (any_hi) {
      pv(hi);
      pv(hi);
    }
  };
  v4i p[QT], hi[QT];
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = wave + NW * i;
      if (c <= nkc) {
        const bool any_hi = chunk_p(c, c == nkc, kf[i], p, hi);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) chunk_pv(c == nkc, ks, vf[i][ks], p, hi, any_hi);
      }
    }
  } else {
    auto chunk = [&](int c, bool tree) {
      load_k(c, tree, kf[0]);
      load_v(c, tree, 0, vf[0][0]);
      const bool any_hi = chunk_p(c, tree, kf[0], p, hi);
      // the second half of a wide head's V follows where K was
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks > 0) load_v(c, tree, ks, vf[0][0]);
        chunk_pv(tree, ks, vf[0][0], p, hi, any_hi);
      }
    };
#pragma unroll 1
    for (int c = c_lo + wave; c < c_hi; c += NW) chunk(c, false);
    if (has_tree && (nkc - c_lo) % NW == wave) chunk(nkc, true);
  }

  // ---- the waves' sums meet in LDS: a lane's four products are four columns of a row ----
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    psum[u] += (uint32_t)__shfl_xor((int)psum[u], 16);
    psum[u] += (uint32_t)__shfl_xor((int)psum[u], 32);
    if (lane < 16) sSum[wave][16 * u + lane] = psum[u];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<v4i *>(&sO[wave][(16 * u + 4 * g + r) * OLD + 64 * ks + 4 * n]) =
            v4i{o[u][ks][0][r], o[u][ks][1][r], o[u][ks][2][r], o[u][ks][3][r]};
  }
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
    uint32_t *mine = part_of<KS, QT>(t, block, part, parts);
    for (int i = 4 * tid; i < QR * 64 * KS; i += 4 * 64 * NW)
      *reinterpret_cast<v4i *>(mine + i) = sum_of(i / (64 * KS) * OLD + i % (64 * KS));
    if (tid < QR) mine[QR * 64 * KS + tid] = sum;
    return;
  }
  if (tid < QR) sInv[tid] = fisr((int32_t)sum, a.rsqrt_off);
  lds_barrier();
  for (int i = tid; i < rows * words; i += 64 * NW) {
    const int q = by_words(i), d = 4 * (i - q * words);
    uint32_t w = 0;
    if (q0 + q < cnt) {
      const v4i v = sum_of(q * OLD + d);
      const uint32_t sums[4] = {(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3]};
      w = output_word(a, sums, sInv[q]);
    }
    *reinterpret_cast<uint32_t *>(obase + (int64_t)(q0 + q) * a.o_st + d) = w;
  }
}

// Adds the parts of a block's row and finishes it, a wave a row: lane l has word l % W of parts l / W,
// l / W + 64 / W, ..., four of them on the way at once.
template <int KS, int QT>
__global__ __launch_bounds__(256) void attn_tree_join_kernel(TreeArgs t, int qblocks, int parts) {
  constexpr int QR = 16 * QT, W = 16 * KS, AT_ONCE = 64 / W;
  const AttnArgs &a = t.a;
  const int lane = threadIdx.x & 63, w = lane % W;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), block = blockIdx.y;
  const int q = block % qblocks * QR + row, bh = block / qblocks, h = bh % a.H;
  const int64_t b = bh / a.H;
  if (q >= a.Tq) return;
  const int nkc = (clampi(t.lengths[b], 0, a.Tk) + 63) / 64;
  const int cnt = t.counts ? clampi(t.counts[b], 0, a.Tq) : a.Tq;
  const int used = nkc / part_share(nkc, parts) + 1;  // parts that have chunks
  uint32_t sums[4] = {0u, 0u, 0u, 0u}, psum = 0u;
  if (q < cnt) {
    for (int p0 = lane / W; p0 < used; p0 += 4 * AT_ONCE) {
      v4i x[4];
      uint32_t y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t *from = part_of<KS, QT>(t, block, min(p0 + j * AT_ONCE, used - 1), parts);
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

constexpr int kCus = 256;

template <int KS, bool QUADS, int QT, int NW, int NC, int MODE = ALL>
int launch_tree(const TreeArgs &t, hipStream_t s, int parts = 1) {
  const int qblocks = (t.a.Tq + 16 * QT - 1) / (16 * QT), blocks = qblocks * t.a.B * t.a.H, per_xcd = (blocks + 7) / 8;
  const int words = t.a.D / 4, per_word = (65536 + words - 1) / words;
  const int table = t.a.frac_bits <= kTableBits ? table_at(t.a.frac_bits) : -1;
  // a grid has fewer than 2^32 threads
  if (8LL * per_xcd * 64 * NW >= 1LL << 32) return fail("too many heads and nodes for one call");
  hipLaunchKernelGGL((attn_tree_kernel<KS, QUADS, QT, NW, NC, MODE>), dim3((unsigned)(8 * per_xcd), (unsigned)parts),
                     dim3(64 * NW), 0, s, t, qblocks, blocks, per_xcd, per_word, table);
  return check_launch("attn_tree_kernel");
}

template <int KS, bool QUADS, int QT>
int launch_tree_parts(const TreeArgs &t, int parts, hipStream_t s) {
  int rc = launch_tree<KS, true, QT, 8, 0, PART_MAX>(t, s, parts);  // reads K only
  if (rc == 0) rc = launch_tree<KS, QUADS, QT, 8, 0, PART_SUM>(t, s, parts);
  if (rc) return rc;
  const int qblocks = (t.a.Tq + 16 * QT - 1) / (16 * QT);
  hipLaunchKernelGGL((attn_tree_join_kernel<KS, QT>), dim3((unsigned)(4 * QT), (unsigned)(qblocks * t.a.B * t.a.H)),
                     dim3(256), 0, s, t, qblocks, parts);
  return check_launch("attn_tree_join_kernel");
}

// Blocks to the keys of one (batch, head) and its 16 nodes, or 32 where there are more: as many as the CUs hold at
// one each. A CU draws 25 to 40 bytes a ns from beyond L2, which bounds a long cache's blocks where they are
// few, but three launches are about 15 us. us split and not: 40 heads of 128 over up to 4096 keys, 61 nodes 27.1 / 39.6,
// 16 nodes 18.7 / 39.2, over up to 1024 18.8 / 15.6 and 15.5 / 15.5, 120 heads over 1500 21.0 / 20.9, over 2048 24.1 / 27.9.
// Narrow heads, 16 and 61 nodes of 40: over 4096 keys 14.5 / 14.3 and 18.4 / 14.4, 8192 17.0 / 23.1 and 23.1 / 22.7,
// 16384 24.7 / 52.1 and 35.4 / 47.7. Two groups of waves with 32 nodes each on the same keys took 28.9 in the place of
// 27.1, 64 nodes a wave 38.7 (spills), the next keys requested ahead 27.3.
constexpr int kSplitNarrow = 8192, kSplitWide = 1536;  // positions
int tree_parts(int64_t heads, int64_t nodes, int64_t head_dim, int64_t cap) {
  if (cap < (head_dim <= 64 ? kSplitNarrow : kSplitWide)) return 1;
  const int64_t blocks = heads * (nodes <= 16 ? 1 : (nodes + 31) / 32), chunks = (cap + 63) / 64 + 1;
  return (int)std::max<int64_t>(1, std::min(kCus / blocks, (chunks + 7) / 8));
}

// Caches of up to 448 positions are eight chunks with the tree's: a wave each while a block has
// a CU to itself (26 nodes of 20 heads, us with eight waves of one chunk, four of two and eight in a loop over
// both passes: 4.9 / 5.5 / 5.2), else four waves of two, which leave more blocks to a CU (16
// nodes of 2560 heads over 224 keys on average 25.7 / 24.2 / 33.3, one node over 447 31.3 / 30.3 / 38.6).
// Longer ones loop.
template <int KS, bool QUADS, int QT>
int launch_tree_q(const TreeArgs &t, hipStream_t s) {
  const int chunks = (t.a.Tk + 63) / 64 + 1;
  const int64_t blocks = (int64_t)t.a.B * t.a.H * ((t.a.Tq + 16 * QT - 1) / (16 * QT));
  if (chunks > 8) return launch_tree<KS, QUADS, QT, 8, 0>(t, s);
  if constexpr (QT == 1)
    if (blocks <= kCus) return launch_tree<KS, QUADS, QT, 8, 1>(t, s);
  return launch_tree<KS, QUADS, QT, 4, 2>(t, s);
}

// 16 nodes a block, or 32 over one set of K and V fragments, where the blocks of either are many (wide heads
// count twice). us of either: 32 nodes of 20, 320 and 640 heads 5.0 / 7.0, 9.5 / 11.4 and 13.4 / 14.3, of 1040
// 19.7 / 20.0, 1280 23.6 / 22.8, 2560 37.8 / 35.0; 64 nodes of 320 heads 13.0 / 13.3, 480 17.0 / 15.6, 640 20.5 / 19.0, 2560
// 64.3 / 52.9, of 240 96 wide ones 19.3 / 15.2, of 320 128 wide ones over 2300 keys 131 / 86; 48 nodes, whose last
// block has 16, of 1280 heads 29.3 / 31.0.
constexpr int64_t kPairTiles = 7 * kCus;
template <int KS, bool QUADS>
int launch_tree_k(const TreeArgs &t, hipStream_t s) {
  const int parts = tree_parts((int64_t)t.a.B * t.a.H, t.a.Tq, t.a.D, t.a.Tk);
  if (parts > 1)
    return t.a.Tq <= 16 ? launch_tree_parts<KS, QUADS, 1>(t, parts, s) : launch_tree_parts<KS, QUADS, 2>(t, parts, s);
  const int64_t tiles = (int64_t)t.a.B * t.a.H * ((t.a.Tq + 15) / 16);
  if (t.a.Tq > 16 && KS * tiles > kPairTiles) return launch_tree_q<KS, QUADS, 2>(t, s);
  return launch_tree_q<KS, QUADS, 1>(t, s);
}

}  // namespace

int64_t attn_tree_workspace(int64_t heads, int64_t nodes, int64_t head_dim, int64_t cap) {
  const int64_t parts = tree_parts(heads, nodes, head_dim, cap), qt = nodes <= 16 ? 1 : 2;
  if (parts == 1) return 0;
  return 4 * heads * ((nodes + 16 * qt - 1) / (16 * qt)) * parts * part_words(head_dim <= 64 ? 1 : 2, (int)qt);
}

int launch_attn_tree(const TreeArgs &t, hipStream_t s) {
  const bool quads = t.a.v_sq != 4;
  if (t.a.D <= 64) return quads ? launch_tree_k<1, true>(t, s) : launch_tree_k<1, false>(t, s);
  return quads ? launch_tree_k<2, true>(t, s) : launch_tree_k<2, false>(t, s);
}

}  // namespace iw
