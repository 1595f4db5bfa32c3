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

// Minimum and maximum over the 16 lanes of a DPP row, in every lane of it
__device__ __forceinline__ int row16_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(INT32_MIN, v, 0xB1, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(INT32_MIN, v, 0x4E, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(INT32_MIN, v, 0x141, 0xf, 0xf, false));
  return max(v, __builtin_amdgcn_update_dpp(INT32_MIN, v, 0x140, 0xf, 0xf, false));
}
__device__ __forceinline__ int row16_min(int v) { return ~row16_max(~v); }

// KS: 64-column parts of the head; QUADS: V in key quads; QT: 16-query tiles of the block; NW waves.
template <int KS, bool QUADS, int QT, int NW>
__global__ __launch_bounds__(64 * NW) void attn_window_kernel(WindowArgs t, int qblocks, int blocks, int per_xcd,
                                                              int per_word, int table_off) {
  constexpr int QR = 16 * QT, OLD = 64 * KS + 4;
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
  // i / words for the i < 2^11 of the output
  const auto by_words = [&](int i) { return (int)__umul24(i, per_word) >> 16; };

  if (q0 >= cnt) {  // no query of these is in use
    for (int i = tid; i < rows * words; i += 64 * NW) {
      const int q = by_words(i);
      *reinterpret_cast<uint32_t *>(obase + (int64_t)(q0 + q) * a.o_st + 4 * (i - q * words)) = 0u;
    }
    return;
  }

  // ---- queries, what each sees, and what any and all of the block see ----
  v4i qf[QT][KS];
  Seen seen[QT];
  int start = INT32_MAX, end = 0, all_from = 0, all_to = INT32_MAX;
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    const int q = min(q0 + 16 * u + n, cnt - 1);  // queries past the count repeat the last one
    const int64_t p = t.positions ? (int64_t)t.positions[b * t.pos_sb + q] : (int64_t)len - cnt + q;
    seen[u] = seen_from(t, len, p);
    start = min(start, seen[u].start), end = max(end, seen[u].end);
    all_from = max(all_from, seen[u].start), all_to = min(all_to, seen[u].end);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d0 = 64 * ks + 16 * g;
      qf[u][ks] = v4i{0, 0, 0, 0};
      if (d0 < D) qf[u][ks] = *reinterpret_cast<const v4i *>(a.q + b * a.q_sb + (int64_t)q * a.q_st + (int64_t)h * D + d0);
    }
  }
  start = __builtin_amdgcn_readfirstlane(row16_min(start));
  end = __builtin_amdgcn_readfirstlane(row16_max(end));
  all_from = __builtin_amdgcn_readfirstlane(row16_max(all_from));
  all_to = __builtin_amdgcn_readfirstlane(row16_min(all_to));
  // chunk c of the block's list is chunk c of the keys while it holds first keys, then w0 + c - ns
  const int w0 = min(start, end) / 64, w1 = (end + 63) / 64;
  const int ns = min((min(t.sinks, end) + 63) / 64, w0);
  const int nch = ns + max(0, w1 - w0);
  auto chunk_at = [&](int c) { return c < ns ? c : w0 + c - ns; };

  // The K operands of chunk c: keys past the last repeat it, head dims past D the
  // last ones (the query is zero there). A chunk's base is uniform, its lanes'
  // offsets fit 32 bits.
  const int kcol = 16 * g, key0 = 16 * (n >> 2) + (n & 3);
  auto load_k = [&](int c, v4i (&f)[4][KS]) {
    const int8_t *base = kbase + (int64_t)(64 * c) * a.k_st;
    const int last = len - 64 * c - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        f[i][ks] = *reinterpret_cast<const v4i *>(base + ((uint32_t)min(key0 + 4 * i, last) * (uint32_t)a.k_st +
                                                          (uint32_t)min(64 * ks + kcol, D - 16)));
  };
  // Quads and transposed rows hold words of four keys of one column. Columns past D
  // repeat the last ones; their sums are not stored.
  auto load_v = [&](int c, int ks, v4i (&f)[4]) {
    const uint32_t d0 = (uint32_t)min(64 * ks + 4 * n, D - 4);
    if (QUADS) {
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
  auto v_operands = [&](const v4i (&f)[4], v4i (&o)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = QUADS ? f[j][i] : f[i][j];
  };

  const bool table = table_off >= 0;
  const int zero = table ? shift_exp_zero(a.frac_bits) : IW_SEXP_LUT - 1;
  if (table)
    for (int i = 16 * tid; i <= zero; i += 16 * 64 * NW)
      *reinterpret_cast<uint4 *>(sTable + i) = *reinterpret_cast<const uint4 *>(kTables.v + table_off + i);

  auto scores = [&](const v4i (&f)[KS], int u) {
    v4i s{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[ks], qf[u][ks], s, 0, 0, 0);
    return s;
  };
  // every query of the block sees every key of the chunk at kc
  auto whole = [&](int kc) { return 64 * kc >= all_from && 64 * kc + 64 <= all_to; };
  // which of the lane group's 16 keys of the chunk at kc this lane's query of tile u sees
  auto counted = [&](int kc, int u) -> uint32_t {
    const int k0 = 64 * kc + 16 * g;
    return (low_bits(seen[u].end - k0) & ~low_bits(seen[u].start - k0)) | low_bits(seen[u].first - k0);
  };

  // ---- pass 1: row maximum of the raw scores ----
  int32_t mx[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) mx[u] = INT32_MIN;
  v4i kf[4][KS];
#pragma unroll 1
  for (int c = wave; c < nch; c += NW) {
    const int kc = chunk_at(c);
    load_k(kc, kf);
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      if (whole(kc)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v4i s = scores(kf[i], u);
          mx[u] = max(max(mx[u], s[0]), s[1]);
          mx[u] = max(max(mx[u], s[2]), s[3]);
        }
      } else {
        const uint32_t ok = counted(kc, u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v4i s = scores(kf[i], u);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if ((ok >> (4 * i + r)) & 1u) mx[u] = max(mx[u], s[r]);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < QT; ++u) {
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
    // requantization keeps the order, so the maximum's is the maximum
    rowmax[u] = mx[u] == INT32_MIN ? -32768 : qk_requant16(mx[u], a.qk_m, a.qk_s);
    sat = sat || rowmax[u] >= 32767;
  }
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
  // P of the chunk at kc as the operands of its products; hi where a P of 128 (a row maximum
  // of 32767 wraps) is left out, as the product is signed: it goes in as twice 64
  auto chunk_p = [&](int kc, const v4i (&f)[4][KS], v4i (&p)[QT], v4i (&hi)[QT]) {
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
        if (!whole(kc)) {
          const uint32_t ok = counted(kc, u);
#pragma unroll
          for (int i = 0; i < 4; ++i) p[u][i] &= (int)byte_mask((ok >> (4 * i)) & 15u);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) psum[u] = __builtin_amdgcn_udot4((uint32_t)p[u][i], 0x01010101u, psum[u], false);
      } else {
        const uint32_t ok = counted(kc, u);
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
  v4i p[QT], hi[QT];
#pragma unroll 1
  for (int c = wave; c < nch; c += NW) {
    const int kc = chunk_at(c);
    v4i vr[KS][4];
    load_k(kc, kf);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) load_v(kc, ks, vr[ks]);
    const bool any_hi = chunk_p(kc, kf, p, hi);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      v4i v[4];
      v_operands(vr[ks], v);
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
    }
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
  if (tid < QR) {
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += sSum[w][tid];
    sInv[tid] = fisr((int32_t)sum, a.rsqrt_off);
  }
  lds_barrier();
  for (int i = tid; i < rows * words; i += 64 * NW) {
    const int q = by_words(i), d = 4 * (i - q * words);
    uint32_t w = 0;
    if (q0 + q < cnt) {
      v4i v = *reinterpret_cast<const v4i *>(&sO[0][q * OLD + d]);
#pragma unroll
      for (int j = 1; j < NW; ++j) v += *reinterpret_cast<const v4i *>(&sO[j][q * OLD + d]);
      const uint32_t sums[4] = {(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3]};
      w = output_word(a, sums, sInv[q]);
    }
    *reinterpret_cast<uint32_t *>(obase + (int64_t)(q0 + q) * a.o_st + d) = w;
  }
}

template <int KS, bool QUADS, int QT, int NW>
int launch_window(const WindowArgs &t, hipStream_t s) {
  const int64_t qblocks = (t.a.Tq + 16 * QT - 1) / (16 * QT), blocks = qblocks * t.a.B * t.a.H;
  const int64_t per_xcd = (blocks + 7) / 8;
  const int words = t.a.D / 4, per_word = (65536 + words - 1) / words;
  const int table = t.a.frac_bits <= kTableBits ? table_at(t.a.frac_bits) : -1;
  // a grid has fewer than 2^32 threads
  if (8 * per_xcd * 64 * NW >= 1LL << 32) return fail("too many heads and queries for one call");
  hipLaunchKernelGGL((attn_window_kernel<KS, QUADS, QT, NW>), dim3((unsigned)(8 * per_xcd)), dim3(64 * NW), 0, s, t,
                     (int)qblocks, (int)blocks, (int)per_xcd, per_word, table);
  return check_launch("attn_window_kernel");
}

}  // namespace

int64_t attn_window_workspace(int64_t heads, int64_t queries, int64_t head_dim, int64_t cap, int64_t before,
                              int64_t after, int64_t sinks) {
  return 0;
}

int launch_attn_window(const WindowArgs &t, hipStream_t s) {
  const bool quads = t.a.v_sq != 4;
  if (t.a.D <= 64) return quads ? launch_window<1, true, 1, 4>(t, s) : launch_window<1, false, 1, 4>(t, s);
  return quads ? launch_window<2, true, 1, 4>(t, s) : launch_window<2, false, 1, 4>(t, s);
}

}  // namespace iw
