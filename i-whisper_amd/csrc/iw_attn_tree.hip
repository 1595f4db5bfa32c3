// Attention of a tree of drafted tokens over an int8 KV cache: node i of row b
// attends to the row's cached keys 0 .. lengths[b] - 1 and to the nodes that
// its visibility word names (its ancestors and itself), whose K and V are read
// where the projection left them. The arithmetic per (query, key) is that of
// the other integer attention kernels: the requantized scores' row maximum
// first, then P = E(S - rowmax - 1), sum P and P.V, exact modulo 2^32 in any
// order, so the keys can be split over waves.
//
// One block per (batch, head); up to 64 nodes are four 16-query MFMA tiles. The
// block's waves take 64-key chunks in turn, the tree itself is one more chunk.
// In a chunk's four 16x16x64 score products, row 4g + r of product t is key
// 16g + 4t + r: lane group g then holds the scores of the 16 consecutive keys
// that its bytes of the P.V operand stand for, and no lane exchange is needed.
// V's columns go to the products as d = 4n + c (lane n, product c): a lane
// reads whole words, and its four sums are one word of the output.
#include "iw_attn_dev.hpp"
#include "iw_common.hpp"
#include "iw_tree.hpp"

namespace iw {

namespace {

// The shift exponential of -n (n the score's distance from the row maximum
// plus one, 0 .. 32767): with t = n + ceil(n/2) - ceil(n/16) (n log2 e in
// 16-bit steps), 2^-(t / 2^f) as a linear fraction and a shift. Distances
// whose t passes 2^15 wrap there and give 0.
struct ShiftExp {
  int32_t f, down;
  __device__ __forceinline__ explicit ShiftExp(int32_t frac) : f(frac), down(max(frac - 7, 0)) {}
  __device__ __forceinline__ uint32_t operator()(int32_t n) const {
    const int32_t t = n + ((n + 1) >> 1) - ((n + 15) >> 4);
    const int32_t m = (1 << f) - 1;
    const int32_t sh = (t + m) >> f;
    const int32_t num = (1 << f) | ((-t & m) >> 1);
    const uint32_t p = (uint32_t)num >> min(sh + down, 31);
    return t > 32768 ? 0u : p;
  }
};

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

// KS: 64-column parts of the head; QUADS: V in key quads; QT: 16-query tiles.
template <int KS, bool QUADS, int QT, int NW>
__global__ __launch_bounds__(64 * NW) void attn_tree_kernel(TreeArgs t) {
  constexpr int QR = 16 * QT, OLD = 64 * KS + 4;
  __shared__ int32_t sMax[NW][QR];
  __shared__ uint32_t sSum[QR];
  __shared__ int32_t sInv[QR];
  __shared__ __attribute__((aligned(16))) uint32_t sO[QR * OLD];

  const AttnArgs &a = t.a;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int h = blockIdx.x % a.H;
  const int64_t b = blockIdx.x / a.H;
  const int D = a.D, N = a.Tq;
  const int len = clampi(t.lengths[b], 0, a.Tk);
  const int cnt = t.counts ? clampi(t.counts[b], 0, N) : N;
  const int nkc = (len + 63) / 64;  // cached chunks; chunk nkc is the tree
  const int8_t *const kbase = a.k + b * a.k_sb + (int64_t)h * a.k_sh;
  const int8_t *const vbase = a.vt + b * a.v_sb + (int64_t)h * a.v_sh;
  const int8_t *const knew = t.kn + b * t.kn_sb + (int64_t)h * D;
  const int8_t *const vnew = t.vn + b * t.vn_sb + (int64_t)h * D;

  if (cnt == 0) {  // no node of this row is in use
    for (int i = tid; i < N * (D / 4); i += 64 * NW)
      *reinterpret_cast<uint32_t *>(a.out + b * a.o_sb + (int64_t)(i / (D / 4)) * a.o_st + (int64_t)h * D +
                                    4 * (i % (D / 4))) = 0u;
    return;
  }

  v4i qf[QT][KS];
  uint64_t vis[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    const int q = min(16 * u + n, cnt - 1);  // queries past the count repeat the last one
    vis[u] = t.visible[b * t.vis_sb + q];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d0 = 64 * ks + 16 * g;
      qf[u][ks] = v4i{0, 0, 0, 0};
      if (d0 < D) qf[u][ks] = *reinterpret_cast<const v4i *>(a.q + b * a.q_sb + (int64_t)q * a.q_st + (int64_t)h * D + d0);
    }
  }

  // the K operands of chunk c (keys past the last repeat it, head dims past D are zero)
  auto load_k = [&](int c, v4i (&f)[4][KS]) {
    const bool tree = c == nkc;
    const int8_t *base = tree ? knew : kbase;
    const int64_t st = tree ? t.kn_st : a.k_st;
    const int last = (tree ? cnt : len) - 1, k0 = tree ? 0 : 64 * c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = min(k0 + 16 * (n >> 2) + 4 * i + (n & 3), last);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d0 = 64 * ks + 16 * g;
        f[i][ks] = v4i{0, 0, 0, 0};
        if (d0 < D) f[i][ks] = *reinterpret_cast<const v4i *>(base + key * st + d0);
      }
    }
  };
  // the V operands: f[ks][c] holds column 64 ks + 4 n + c of the lane group's 16 keys
  auto load_v = [&](int c, v4i (&f)[KS][4]) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d0 = 64 * ks + 4 * n;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[ks][i] = v4i{0, 0, 0, 0};
      if (d0 >= D) continue;
      if (c == nkc) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t w[4], o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = *reinterpret_cast<const uint32_t *>(vnew + (int64_t)min(16 * g + 4 * j + i, cnt - 1) * t.vn_st + d0);
          transpose4(w, o);
#pragma unroll
          for (int i = 0; i < 4; ++i) f[ks][i][j] = (int)o[i];
        }
      } else if (QUADS) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int quad = min(16 * c + 4 * g + j, (len - 1) >> 2);
          const v4i w = *reinterpret_cast<const v4i *>(vbase + quad * a.v_sq + 4 * d0);
#pragma unroll
          for (int i = 0; i < 4; ++i) f[ks][i][j] = w[i];
        }
      } else {
        const int key0 = min(64 * c + 16 * g, (len - 1) & ~15);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          f[ks][i] = *reinterpret_cast<const v4i *>(vbase + (int64_t)(d0 + i) * a.v_sd + key0);
      }
    }
  };
  auto scores = [&](const v4i (&f)[KS], int u) {
    v4i s{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[ks], qf[u][ks], s, 0, 0, 0);
    return s;
  };
  // which of the lane group's 16 keys of chunk c count for this lane's query of tile u
  const uint64_t in_use = cnt == 64 ? ~0ull : (1ull << cnt) - 1;
  auto counted = [&](int c, int u) -> uint32_t {
    if (c == nkc) return (uint32_t)((vis[u] & in_use) >> (16 * g)) & 0xffffu;
    return (1u << clampi(len - 64 * c - 16 * g, 0, 16)) - 1u;
  };

  // ---- pass 1: row maximum of the raw scores ----
  int32_t mx[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) mx[u] = INT32_MIN;
  v4i kf[4][KS];
  for (int c = wave; c <= nkc; c += NW) {
    load_k(c, kf);
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      const uint32_t ok = counted(c, u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v4i s = scores(kf[i], u);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if ((ok >> (4 * i + r)) & 1u) mx[u] = max(mx[u], s[r]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    mx[u] = max(mx[u], __shfl_xor(mx[u], 16));
    mx[u] = max(mx[u], __shfl_xor(mx[u], 32));
    if (lane < 16) sMax[wave][16 * u + lane] = mx[u];
  }
  for (int i = tid; i < QR; i += 64 * NW) sSum[i] = 0u;
  for (int i = tid; i < QR * OLD; i += 64 * NW) sO[i] = 0u;
  __syncthreads();
  int32_t rowmax[QT];
#pragma unroll
  for (int u = 0; u < QT; ++u) {
#pragma unroll
    for (int w = 0; w < NW; ++w) mx[u] = max(mx[u], sMax[w][16 * u + n]);
    // requantization keeps the order, so the maximum's is the maximum
    rowmax[u] = mx[u] == INT32_MIN ? -32768 : qk_requant16(mx[u], a.qk_m, a.qk_s);
  }

  // ---- pass 2: P and P.V over this wave's keys ----
  const ShiftExp sexp(a.frac_bits);
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
  v4i vf[KS][4];
  for (int c = wave; c <= nkc; c += NW) {
    load_k(c, kf);
    load_v(c, vf);
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      const ScoreIndex ix(a, rowmax[u]);
      const uint32_t ok = counted(c, u);
      v4i p;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v4i s = scores(kf[i], u);
        uint32_t w = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t e = (ok >> (4 * i + r)) & 1u ? sexp((int32_t)ix.any(s[r])) : 0u;
          w |= (e & 0xffu) << (8 * r);
        }
        p[i] = (int)w;
        psum[u] = __builtin_amdgcn_udot4(w, 0x01010101u, psum[u], false);
      }
      // P is unsigned and the product signed: a P of 128 (a row maximum of
      // 32767 wraps) goes in as 0 and twice 64
      v4i lo, hi;
#pragma unroll
      for (int i = 0; i < 4; ++i) lo[i] = p[i] & 0x7f7f7f7f, hi[i] = (int)(((uint32_t)p[i] >> 1) & 0x40404040u);
      const bool any_hi = __any((hi[0] | hi[1] | hi[2] | hi[3]) != 0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[u][ks][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo, vf[ks][i], o[u][ks][i], 0, 0, 0);
          if (any_hi) {
            o[u][ks][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi, vf[ks][i], o[u][ks][i], 0, 0, 0);
            o[u][ks][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi, vf[ks][i], o[u][ks][i], 0, 0, 0);
          }
        }
    }
  }

  // ---- the waves' sums meet in LDS ----
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    psum[u] += (uint32_t)__shfl_xor((int)psum[u], 16);
    psum[u] += (uint32_t)__shfl_xor((int)psum[u], 32);
    if (lane < 16) atomicAdd(&sSum[16 * u + lane], psum[u]);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          atomicAdd(&sO[(16 * u + 4 * g + r) * OLD + 64 * ks + 4 * n + i], (uint32_t)o[u][ks][i][r]);
  }
  __syncthreads();
  if (tid < QR) sInv[tid] = fisr((int32_t)sSum[tid], a.rsqrt_off);
  __syncthreads();
  const int words = D / 4;
  for (int i = tid; i < N * words; i += 64 * NW) {
    const int q = i / words, d = 4 * (i % words);
    uint32_t w = 0;
    if (q < cnt) {
      const int32_t inv = sInv[q];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        int32_t y = rshift((int32_t)(sO[q * OLD + d + c] * (uint32_t)inv), a.rsqrt_off);
        y = rshift((int32_t)((uint32_t)y * (uint32_t)inv), a.rsqrt_off);
        y = rshift((int32_t)((uint32_t)y * a.av_m), a.av_s);
        w |= ((uint32_t)clampi(y, -127, 127) & 0xffu) << (8 * c);
      }
    }
    *reinterpret_cast<uint32_t *>(a.out + b * a.o_sb + (int64_t)q * a.o_st + (int64_t)h * D + d) = w;
  }
}

template <int KS, bool QUADS, int QT>
int launch_tree(const TreeArgs &t, hipStream_t s) {
  constexpr int NW = 4;
  hipLaunchKernelGGL((attn_tree_kernel<KS, QUADS, QT, NW>), dim3((unsigned)(t.a.B * t.a.H)), dim3(64 * NW), 0, s, t);
  return check_launch("attn_tree_kernel");
}

template <int KS, bool QUADS>
int launch_tree_q(const TreeArgs &t, hipStream_t s) {
  switch ((t.a.Tq + 15) / 16) {
    case 1: return launch_tree<KS, QUADS, 1>(t, s);
    case 2: return launch_tree<KS, QUADS, 2>(t, s);
    case 3: return launch_tree<KS, QUADS, 3>(t, s);
    default: return launch_tree<KS, QUADS, 4>(t, s);
  }
}

}  // namespace

int launch_attn_tree(const TreeArgs &t, hipStream_t s) {
  const bool quads = t.a.v_sq != 4;
  if (t.a.D <= 64) return quads ? launch_tree_q<1, true>(t, s) : launch_tree_q<1, false>(t, s);
  return quads ? launch_tree_q<2, true>(t, s) : launch_tree_q<2, false>(t, s);
}

}  // namespace iw
