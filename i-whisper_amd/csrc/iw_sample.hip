// Tokens drawn from rows of logits by given random numbers, and drafted tokens verified
// against the model's probabilities.
//
// A row's weights are w_j = 2^((x_j - M) c) with M its largest logit, c = log2(e) * scale / T,
// and Z their sum; the token that a number u in [0, 1) draws is the least j with
// w_0 + .. + w_j > u Z. At a draft x after node i with the model's probabilities p and the draft's
// q: accepted where u q(x) < p(x), else the token is drawn from max(p - q, 0), which makes the
// tokens those of p whatever q is.
//
// A border between two tokens of a whole vocabulary lies within 2e-5 of the next one, and a sum that is
// off by 1e-8 would draw another token once in a few thousand calls: weights and sums are
// 64-bit numbers (vector units add them as fast as 32-bit ones here). An int8 row has at most 256
// distances from M, whose weights are a table in LDS.
//
// A row is cut into spans of 256 pieces of 16 bytes, a wave each: its maximum and its sum relative to that are all
// that the first launch leaves (the one read of the logits). The row's block then adds up the spans, finds the one
// where the running sum passes u Z, and looks into that again. For drafts a launch between finds the first
// rejection from the sums, and another one the sums of max(p - q, 0) over 64 pieces each. (All of that in one launch, a
// block of 16 waves a row, took 26.4 us for 5 rows of int8 logits in the place of 3.7 + 6.9 + 6.6, and 36.3 for 24 times 6 of
// float32 in the place of 5.4 + 4.8 + 6.0: 40 KB of instructions that every block fetches and runs once.)
#include <algorithm>
#include <type_traits>

#include "iw_common.hpp"
#include "iw_drafts.hpp"
#include "iw_logit_dev.hpp"
#include "iw_tree.hpp"

namespace iw {

namespace {

constexpr int kSpanPieces = 256;
constexpr int kWaves = 4, NT = 64 * kWaves;
constexpr double kLog2E = 1.4426950408889634, kLn2 = 0.6931471805599453;

// The largest logit of a span (-inf: none that counts), for rows that take the most probable token
// its first column, and the sum of the weights relative to it
struct Span {
  float m;
  int32_t col;
  double z;
};

// 2^f for |f| <= 1/2: of the polynomials of degree 8 that are 1 at 0 the one with the smallest relative error, 8.14e-13
// (found by linear programming; 7.8e-13 without that condition, a degree more or less 1.4e-14 or 4.0e-11). The
// largest logit's weight is 1 exactly, so equal ones have exact sums and meet at exact borders. A border's share s of the whole is right
// to 2 s (1 - s) 8.2e-13 then, at most 4.1e-13, and up to 2e-8 of all numbers draw another token of 2^16 than exact ones.
__device__ __forceinline__ double exp2_part(double f) {
  // the two constants of the first step: an instruction reads one from scalar registers
  double second = 0x1.00d8533f3e35fp-16;
  asm("" : "+v"(second));
  double p = fma(0x1.61c4f11ba3bb2p-20, f, second);
  p = fma(p, f, 0x1.430aa882746bep-13);
  p = fma(p, f, 0x1.5d874d0702cb5p-10);
  p = fma(p, f, 0x1.3b2ab5ed6ffb2p-7);
  p = fma(p, f, 0x1.c6b08dced351ap-5);
  p = fma(p, f, 0x1.ebfbdff8ede81p-3);
  p = fma(p, f, 0x1.62e42fef89d1ep-1);
  return fma(p, f, 1.0);
}
// 2^t, 0 far below. A NaN (a masked logit of a row that has no other) gives 0.
__device__ __forceinline__ double exp2_64(double t) {
  t = fmax(t, -1100.0);
  const double k = rint(t);
  return ldexp(exp2_part(t - k), (int)k);
}

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double x) {
  const uint64_t b = __double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, true);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double lane_f64(double x, int l) {
  const uint64_t b = __double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
// Sum over the wave, in every lane
__device__ __forceinline__ double wave_sum_f64(double v) {
  v += dpp_f64<0xB1>(v);
  v += dpp_f64<0x4E>(v);
  v += dpp_f64<0x141>(v);
  v += dpp_f64<0x140>(v);
  return (lane_f64(v, 0) + lane_f64(v, 16)) + (lane_f64(v, 32) + lane_f64(v, 48));
}
// Sum of this lane's and the lower lanes' values: shifts by 1, 2, 4 and 8 within rows of 16 lanes, then the last lane
// of the row before for every other row, and lane 31 for the upper half
template <int CTRL, int ROWS>
__device__ __forceinline__ double scan_step(double x) {
  const uint64_t b = __double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
  return x + __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double wave_scan_f64(double v) {
  v = scan_step<0x111, 0xf>(v);
  v = scan_step<0x112, 0xf>(v);
  v = scan_step<0x114, 0xf>(v);
  v = scan_step<0x118, 0xf>(v);
  v = scan_step<0x142, 0xa>(v);
  return scan_step<0x143, 0xc>(v);
}

__device__ __forceinline__ float clamp_uniform(float u) { return fminf(fmaxf(u, 0.f), 0x1.fffffep-1f); }

// 16 bytes of logits at any address of their type
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef v4u v4u_any __attribute__((aligned(1)));
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T *row, int piece) {
  const v4u x = *reinterpret_cast<const v4u_any *>(reinterpret_cast<const char *>(row) + 16u * (uint32_t)piece);
  return make_uint4(x.x, x.y, x.z, x.w);
}

// The bits of the suppressed ones among a piece's N columns from col on: they lie in one word
template <int N>
__device__ __forceinline__ uint32_t hidden_bits(const uint32_t *words, uint32_t col) {
  return words ? (words[col >> 5] >> (col & 31)) & ((1u << N) - 1u) : 0u;
}

// A row as a distribution, as every launch looks at it. A temperature of 0 (or none at all) gives the first
// of the largest logits all of the weight. Logits lie 2^-149 apart at least: above 2^300, c makes no difference.
struct Row {
  double c;
  bool greedy;
  __device__ __forceinline__ Row(const DistRows &d, int64_t outer) {
    const double t = d.temperatures ? (double)d.temperatures[outer] : d.temperature;
    greedy = !(t > 0.0);
    c = greedy ? 0.0 : fmin(kLog2E * (d.scale / t), 0x1p300);
  }
};
template <typename T>
__device__ __forceinline__ const T *row_of(const DistRows &d, int64_t outer, int inner) {
  return reinterpret_cast<const T *>(d.x) + outer * d.sb + inner * d.st;
}

// Weight of an int8 logit at a distance from the largest, to 44 bits (off by another 2.8e-14): sums of some 64 equal ones are exact,
// so those of suppressed logits leave nothing where they are taken off a span's sum again.
__device__ __forceinline__ double weight_at(double distance, double c) {
  const uint64_t b = __double_as_longlong(exp2_64(-(distance * c)));
  return __longlong_as_double((long long)((b + 0x100u) & ~0x1ffull));
}

// Weight of a logit relative to the largest, m; int8 rows have those of all distances in a table. The
// distance comes first: as a difference of two products it would be lost where c is large.
struct Weigh {
  double c, m;
  const double *table;
  __device__ __forceinline__ Weigh(double c_, float m_, const double *t) : c(c_), m(m_), table(t) {}
  __device__ __forceinline__ double log2_of(float x) const { return ((double)x - m) * c; }
  template <typename T>
  __device__ __forceinline__ double of(float x) const {
    if constexpr (std::is_same<T, int8_t>::value) return table[(int)m - (int)x & 255];
    return exp2_64(log2_of(x));
  }
};
template <int THREADS = NT>
__device__ __forceinline__ void fill_table(double *table, double c, int tid) {
  for (int d = tid; d < 256; d += THREADS) table[d] = weight_at((double)d, c);
}

// A row's pieces, the last of them perhaps in part, and spans
template <typename T>
struct Cut {
  static constexpr int E = Logit<T>::E;
  int cols, full, spans, parts;  // parts of 64 pieces
  __host__ __device__ Cut(int cols_) : cols(cols_), full(cols_ / E) {
    const int pieces = (cols_ + E - 1) / E;
    spans = (pieces + kSpanPieces - 1) / kSpanPieces;
    parts = (pieces + 63) / 64;
  }
};

// ---- the spans' maxima and sums ----
struct SpanArgs {
  DistRows d[2];            // of the rows below `first`, and of the others
  int64_t first = 0;
  const int32_t *counts = nullptr;  // rows of d[i] at or past counts[outer] - i are not looked at
  const uint32_t *suppress = nullptr;
  int cols = 0;
  Span *spans = nullptr;
  int64_t row0 = 0;         // the first of this launch
};

// The larger of two, NaN where either is
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Adds the weight 2^((x - m) c) of a span's logit to its sum: a constant's low word counts the exponents, with which the
// rest's power is multiplied in the addition. Weights below 2^-1000, -inf's too, are 2^-1000, which a sum with the largest's 1
// does not hold. The distance comes first, so that the largest's weight is 1 exactly.
struct SumWeights {
  double c, m, least;
  __device__ __forceinline__ SumWeights(double c_, float m_)
      : c(fmax(c_, 0x1p-900)), m(m_), least(-1000.0 * __builtin_amdgcn_rcp(c)) {}
  __device__ __forceinline__ double add(float x, double sum) const {
    const double d = fmax((double)x - m, least), u = fma(d, c, 0x1.8p52 + 1023.0), n = u - (0x1.8p52 + 1023.0);
    const double whole = __longlong_as_double((long long)((uint64_t)((uint32_t)__double_as_longlong(u) << 20) << 32));
    return fma(exp2_part(fma(d, c, -n)), whole, sum);
  }
};

// The first logit of a piece that is m, the largest, E or more if none: those that `off` hides are less, or m is int8's lowest
template <typename T>
__device__ __forceinline__ uint32_t first_with(const uint4 &w, uint32_t off, float m) {
  constexpr int E = Logit<T>::E;
  if constexpr (std::is_same<T, int8_t>::value) {
    if (m == -128.f) return (uint32_t)__ffs((int)(~off & 0xffffu)) - 1u;
    const uint32_t bits = Logit<T>::reaching(w, (int)m);  // bit 8 i + q: byte i of word q
    uint32_t first = ~0u;
#pragma unroll
    for (int q = 3; q >= 0; --q) {
      const uint32_t word = (bits >> q) & 0x01010101u;
      if (word) first = 4u * q + ((uint32_t)(__ffs((int)word) - 1) >> 3);
    }
    return first;
  } else {
    uint32_t first = ~0u;
#pragma unroll
    for (int e = E - 1; e >= 0; --e)
      if (Logit<T>::get(w, e) == m) first = e;
    return first;
  }
}

// Two waves a block: a row's last block has at most one without a span (one, two or four waves: 128 times 8 drafts of int8
// logits 57, 56 and 61 us, 2048 int8 rows 46, 43 and 47; rows of the other types differ by a few in a hundred).
constexpr int kSpanWaves = 2;
template <typename T>
__global__ __launch_bounds__(64 * kSpanWaves) void row_spans_kernel(SpanArgs a, int groups) {
  using L = Logit<T>;
  constexpr bool I8 = std::is_same<T, int8_t>::value;
  constexpr int E = L::E, P = kSpanPieces / 64;
  constexpr uint32_t ALL = (1u << E) - 1u;
  __shared__ double sTable[I8 ? 256 : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = a.row0 + (uint32_t)blockIdx.x / (uint32_t)groups;
  const bool second = row >= a.first;
  const int64_t r = second ? row - a.first : row;
  const uint32_t inner = (uint32_t)(second ? a.d[1].inner : a.d[0].inner);
  const uint32_t outer = (uint32_t)r / inner, at = (uint32_t)r % inner;
  if (a.counts && (int)at >= a.counts[outer] - (second ? 1 : 0)) return;
  const Cut<T> cut(a.cols);
  const int s = (int)((uint32_t)blockIdx.x % (uint32_t)groups) * kSpanWaves + __builtin_amdgcn_readfirstlane(tid >> 6);
  const T *x = reinterpret_cast<const T *>(second ? a.d[1].x : a.d[0].x) +
               (int64_t)outer * (second ? a.d[1].sb : a.d[0].sb) + (int64_t)at * (second ? a.d[1].st : a.d[0].st);
  // all that the wave reads is on the way before it waits for anything; pieces past the last read that again
  const int p0 = s * kSpanPieces + lane;
  uint4 w[P];
  if (cut.full > 0) {
#pragma unroll
    for (int p = 0; p < P; ++p) w[p] = load_piece(x, min(p0 + 64 * p, cut.full - 1));
  }
  const int extra = cut.full * E + lane;
  const bool has_extra = s == cut.spans - 1 && extra < a.cols && !suppressed(a.suppress, extra);
  const float xe = has_extra ? L::one(x + extra) : -INFINITY;
  uint32_t off[P];  // not counted: past the last piece, or suppressed
#pragma unroll
  for (int p = 0; p < P; ++p)
    off[p] = p0 + 64 * p >= cut.full ? ALL : hidden_bits<E>(a.suppress, (p0 + 64 * p) * E);
  const Row dist = second ? Row(a.d[1], outer) : Row(a.d[0], outer);
  if (I8) {
    if (!dist.greedy) fill_table<64 * kSpanWaves>(sTable, dist.c, tid);
    lds_barrier();
  }
  if (s >= cut.spans) return;

  // int8 logits that do not count are -128, of which `hidden` are taken off the sum again; others -inf
  float m;
  int hidden = 0;
  if constexpr (I8) {
    using v2s = typename L::v2s;
    v2s most{-32768, -32768};
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (off[p] != 0u) {
        hidden += __popc(off[p]);
        uint32_t *v = &w[p].x;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t bits = __umul24((off[p] >> (4 * q)) & 15u, 0x00204081u) & 0x01010101u;
          const uint32_t no = __builtin_amdgcn_perm(0u, 0u, bits | 0x0c0c0c0cu);
          v[q] = (v[q] & ~no) | (0x80808080u & no);
        }
      }
      most = __builtin_elementwise_max(most, L::halves(w[p]));
    }
    // a half's value is its upper byte
    const int top = wave_max_dpp(max(has_extra ? (int)xe : -128, max((int)most.x >> 8, (int)most.y >> 8)));
    const bool any = __any(has_extra || hidden < P * E);
    m = any ? (float)top : -INFINITY;
  } else {
    float top = xe;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (off[p] != 0u) L::mask(w[p], off[p]);
#pragma unroll
      for (int e = 0; e < E; ++e) top = max_nan(top, L::get(w[p], e));
    }
    m = key_value((uint64_t)wave_max_u32_dpp(ordered(top)) << 32);
  }

  Span out{m, -1, 0.0};
  if (dist.greedy) {
    uint32_t col = has_extra && xe == m ? (uint32_t)extra : ~0u;
#pragma unroll
    for (int p = P - 1; p >= 0; --p) {
      const uint32_t first = first_with<T>(w[p], off[p], m);
      if (first < (uint32_t)E) col = (uint32_t)((p0 + 64 * p) * E) + first;
    }
    out.col = (int32_t)~wave_max_u32_dpp(~col);
  } else if (m - m == 0.f) {
    double z = 0.0;
    if constexpr (I8) {
      const uint32_t top = (uint32_t)((int)m + 128) * 0x01010101u;
      const char *table = reinterpret_cast<const char *>(sTable);
      if (has_extra) z = sTable[(int)m - (int)xe];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        // distances from m, byte by byte: none borrows
        const uint32_t v[4] = {top - (w[p].x ^ 0x80808080u), top - (w[p].y ^ 0x80808080u), top - (w[p].z ^ 0x80808080u),
                               top - (w[p].w ^ 0x80808080u)};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const double a0 = *reinterpret_cast<const double *>(table + (v[q] & 0xffu) * 8);
          const double a1 = *reinterpret_cast<const double *>(table + ((v[q] >> 8) & 0xffu) * 8);
          const double a2 = *reinterpret_cast<const double *>(table + ((v[q] >> 16) & 0xffu) * 8);
          const double a3 = *reinterpret_cast<const double *>(table + ((v[q] >> 24) & 0xffu) * 8);
          z += (a0 + a1) + (a2 + a3);
        }
      }
      // exact for lanes with nothing else
      z -= (double)hidden * sTable[(int)m + 128];
    } else {
      const SumWeights sum(dist.c, m);
      if (has_extra) z = sum.add(xe, z);
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (__any(off[p] != ALL)) {
#pragma unroll
          for (int e = 0; e < E; ++e) z = sum.add(L::get(w[p], e), z);
        }
    }
    out.z = wave_sum_f64(z);
  }
  if (lane == 0) a.spans[row * cut.spans + s] = out;
}

// ---- a row's block: from the spans to a token ----
// The place in n numbers where their running sum passes u times the whole, and the sum below it; -1 if none is above 0. Only
// numbers above 0 are asked, as rounding may lift the running sum over another; if none passes, the last of them. A wave
// finds it by itself.
struct Place {
  int at;
  double whole, target, below;
};
template <typename F>
__device__ __forceinline__ Place place_of(int n, double u, F value, int lane) {
  const double first = lane < n ? value(lane) : 0.0;
  double sum = first;
  for (int i = lane + 64; i < n; i += 64) sum += value(i);
  Place r{-1, wave_sum_f64(sum), 0.0, 0.0};
  r.target = u * r.whole;
  double run = 0.0;
  for (int i = 0; i < n; i += 64) {
    const double v = i == 0 ? first : i + lane < n ? value(i + lane) : 0.0, up = run + wave_scan_f64(v);
    const uint64_t some = __ballot(v > 0.0), passed = __ballot(v > 0.0 && up > r.target);
    if (some != 0) {
      const int l = passed != 0 ? __ffsll((long long)passed) - 1 : 63 - __clzll((long long)some);
      r.at = i + l;
      r.below = lane_f64(up - v, l);
    }
    if (passed != 0) break;
    run = lane_f64(up, 63);
  }
  return r;
}

// The token at `place` among the spans of `pieces` pieces, which are looked at again, a piece a thread (weigh(piece, w):
// the weights of its columns, 0 past the last), for the one thread that has it; -1 for the others.
template <typename T, typename G>
__device__ __forceinline__ int draw(const Place &place, int pieces, G weigh, double (&sWave)[kWaves], int tid) {
  constexpr int E = Cut<T>::E;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  double w[E], sum = 0.0;
  if (tid < pieces) {
    weigh(place.at * pieces + tid, w);
#pragma unroll
    for (int e = 0; e < E; ++e) sum += w[e];
  }
  const double up = wave_scan_f64(sum), target = place.target - place.below;
  if (lane == 63) sWave[wave] = up;
  __syncthreads();
  // the wave whose sums pass the target, or the last with one
  double run = 0.0, below = 0.0;
  int owner = -1;
  bool passed = false;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const double t = sWave[i];
    if (!passed && t > 0.0) {
      owner = i;
      below = run;
      passed = run + t > target;
    }
    run += t;
  }
  if (wave != owner) return -1;
  const uint64_t some = __ballot(sum > 0.0), over = __ballot(sum > 0.0 && below + up > target);
  if (lane != (over != 0 ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)some))) return -1;
  // the first whose running sum passes, else the last with a weight
  double base = below + (up - sum);
  int got = 0;
  passed = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (!passed && w[e] > 0.0) {
      got = e;
      base += w[e];
      passed = base > target;
    }
  }
  return (place.at * pieces + tid) * E + got;
}

// The logits of a piece, and the bits of those that count
template <typename T>
__device__ __forceinline__ uint32_t piece_of(const T *x, int piece, const Cut<T> &cut, const uint32_t *suppress, float (&v)[Cut<T>::E]) {
  constexpr int E = Cut<T>::E;
  if (piece < cut.full) {
    const uint4 w = load_piece(x, piece);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = Logit<T>::get(w, e);
    return ~hidden_bits<E>(suppress, piece * E);
  }
  const int left = max(cut.cols - piece * E, 0);  // fewer than E
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = e < left ? Logit<T>::one(x + (int64_t)piece * E + e) : 0.f;
  return left > 0 ? ~hidden_bits<E>(suppress, piece * E) & ((1u << left) - 1u) : 0u;
}

// A span's sum relative to the row's largest logit, as it is where that is the span's; 0 where its logits' weights are next
// to vanishing, so that a span with a sum has a logit with a weight. The factor is the library's power, right to a rounding: the
// polynomial's errors would add up, and a weight is to be off by one of them.
__device__ __forceinline__ double span_sum(const Span &s, const Weigh &row) {
  if (s.m == row.m) return s.z;
  const double z = s.z * exp2(row.log2_of(s.m));
  return z > 1e-290 ? z : 0.0;
}

// A wave's look at a row's spans: the largest logit, and its first column for rows that take it. Lane l has span l;
// more than 64 are read again.
struct RowSpans {
  const Span *spans;
  int n, lane;
  Span mine;
  float m;
  __device__ __forceinline__ RowSpans(const Span *spans_, int n_, int lane_) : spans(spans_), n(n_), lane(lane_) {
    mine = Span{-INFINITY, -1, 0.0};
    if (lane < n) mine = spans[lane];
  }
  __device__ __forceinline__ Span at(int i) const { return i == lane ? mine : spans[i]; }
  __device__ __forceinline__ void find_max() {
    uint32_t top = ordered(mine.m);
    for (int i = lane + 64; i < n; i += 64) top = max(top, ordered(spans[i].m));
    m = key_value((uint64_t)wave_max_u32_dpp(top) << 32);
  }
  __device__ __forceinline__ int column() const {
    const uint32_t top = ordered(m);
    uint32_t c = 0u;
    for (int i = lane; i < n; i += 64)
      if (ordered(at(i).m) == top) c = max(c, ~(uint32_t)at(i).col);
    return (int)~wave_max_u32_dpp(c);
  }
};

template <typename T>
__global__ __launch_bounds__(NT) void sample_pick_kernel(SampleArgs a) {
  using L = Logit<T>;
  constexpr bool I8 = std::is_same<T, int8_t>::value;
  __shared__ double sTable[I8 ? 256 : 1];
  __shared__ double sWave[kWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const Cut<T> cut(a.cols);
  RowSpans spans(static_cast<const Span *>(a.workspace) + row * cut.spans, cut.spans, lane);
  const double u = (double)clamp_uniform(a.uniforms[row]);
  const Row dist(a.d, row);
  const T *x = row_of<T>(a.d, row, 0);
  spans.find_max();
  const float m = spans.m;
  int tok = -1;
  float lp = 0.f;
  bool mine = tid == 0;
  if (!(m - m == 0.f)) {  // no distribution: a NaN, an infinity, nothing to choose from
    lp = __uint_as_float(0x7fc00000u);
  } else if (dist.greedy) {
    tok = spans.column();
  } else {
    if (I8) fill_table(sTable, dist.c, tid);  // seen behind the barrier below
    const Weigh wt(dist.c, m, sTable);
    const Place place = place_of(cut.spans, u, [&](int i) { return span_sum(spans.at(i), wt); }, lane);
    if (I8) __syncthreads();
    tok = draw<T>(place, kSpanPieces,
                  [&](int piece, double (&w)[L::E]) {
                    float v[L::E];
                    const uint32_t on = piece_of(x, piece, cut, a.suppress, v);
#pragma unroll
                    for (int e = 0; e < L::E; ++e) w[e] = (on >> e) & 1u ? wt.of<T>(v[e]) : 0.0;
                  },
                  sWave, tid);
    mine = tok >= 0;
    // the sum has the token's weight in it but may be a rounding below it
    if (mine) lp = (float)fmin(wt.log2_of(L::one(x + tok)) * kLn2 - log(place.whole), 0.0);
  }
  if (mine) {
    a.tokens[row] = tok;
    if (a.logprob) a.logprob[row] = lp;
  }
}

// ---- drafts ----
enum { FROM_TARGET, FROM_REST, FROM_OTHERS, CERTAIN, NONE };
// What the first rejection of a row leaves to be drawn from: the model's distribution, what
// the draft's leaves of it, all tokens but `hot`; or `hot` itself, or nothing
struct Verdict {
  int32_t accepted, mode, hot;
  float m, mq;
  double c, cq, ip, iq;
};

// Sum and maximum of a row by one wave: relative weight sum Z and largest logit M
struct RowSum {
  float m;
  int32_t col;
  double z;
};
__device__ __forceinline__ RowSum row_sum(const Span *from, int n, const Row &dist, int lane) {
  RowSpans spans(from, n, lane);
  spans.find_max();
  RowSum r{spans.m, -1, 1.0};
  if (dist.greedy) {
    r.col = spans.column();
  } else {
    const Weigh wt(dist.c, r.m, nullptr);
    double z = 0.0;
    for (int i = lane; i < n; i += 64) z += span_sum(spans.at(i), wt);
    r.z = wave_sum_f64(z);
  }
  return r;
}

// A probability, rounded: the same number wherever it is compared or taken away, so that a refused draft
// has nothing left and equal distributions leave nothing.
__device__ __forceinline__ double share(double w, double inv) {
#pragma clang fp contract(off)
  return w * inv;
}
__device__ __forceinline__ double left_of(double p, double q) {
#pragma clang fp contract(off)
  return fmax(p - q, 0.0);
}

// the share of the token at col
template <typename T>
__device__ __forceinline__ double share_of(const T *x, int64_t col, int cols, const uint32_t *suppress, const Row &dist,
                                           const RowSum &r) {
  if (col < 0 || col >= cols || suppressed(suppress, (int)col)) return 0.0;
  if (dist.greedy) return col == r.col ? 1.0 : 0.0;
  const Weigh wt(dist.c, r.m, nullptr);
  const float v = Logit<T>::one(x + col);
  const double w = std::is_same<T, int8_t>::value ? weight_at((double)r.m - v, dist.c) : exp2_64(wt.log2_of(v));
  return share(w, 1.0 / r.z);
}

struct VerifyWork {
  Span *spans;      // of the target's rows, then of the draft's
  double *rest;     // [batch][parts]
  Verdict *verdict;
};
template <typename T>
__device__ __forceinline__ VerifyWork verify_work(const VerifyArgs &a, const Cut<T> &cut) {
  VerifyWork w;
  w.verdict = static_cast<Verdict *>(a.workspace);
  w.spans = reinterpret_cast<Span *>(w.verdict + a.batch);
  w.rest = reinterpret_cast<double *>(w.spans + a.batch * (a.draft.x ? 2 * a.nodes - 1 : a.nodes) * cut.spans);
  return w;
}

// The first rejection of batch row b: the waves of its block take the target's and the draft's rows in turn.
template <int W>
struct Nodes {
  RowSum p[kVerifyMaxNodes], q[kVerifyMaxNodes];
  Verdict verdict;
};
template <typename T, int W>
__device__ __forceinline__ void decide(const VerifyArgs &a, const VerifyWork &w, const Cut<T> &cut, int64_t b, Nodes<W> &s, int tid) {
  const int lane = tid & 63;
  const int N = a.nodes, cnt = a.counts ? clampi(a.counts[b], 0, N) : N;
  const Row dp(a.target, b), dq(a.draft, b);
  const int drafts = a.draft.x ? cnt - 1 : 0;
  for (int i = __builtin_amdgcn_readfirstlane(tid >> 6); i < cnt + drafts; i += W) {
    const bool second = i >= cnt;
    const int64_t row = second ? a.batch * N + b * (N - 1) + (i - cnt) : b * N + i;
    const RowSum r = row_sum(w.spans + row * cut.spans, cut.spans, second ? dq : dp, lane);
    if (lane == 0) (second ? s.q[i - cnt] : s.p[i]) = r;
  }
  __syncthreads();
  if (tid >= 64) return;
  // a lane a draft: whether it is accepted
  bool ok = false;
  if (tid + 1 < cnt) {
    const int64_t row = b * N + tid;
    const int64_t x = a.tokens[row + 1];
    const RowSum p = s.p[tid];
    const double px = share_of(row_of<T>(a.target, b, tid), x, a.cols, a.suppress, dp, p);
    double qx = 1.0;
    bool has = true;
    if (a.draft.x) {
      const RowSum q = s.q[tid];
      qx = share_of(row_of<T>(a.draft, b, tid), x, a.cols, a.suppress, dq, q);
      has = q.m - q.m == 0.f;  // else a draft without a distribution
    }
    ok = has && p.m - p.m == 0.f && (double)clamp_uniform(a.uniforms[row]) * qx < px;
  }
  const int n = min((int)__popcll(__ballot(ok) & ~(__ballot(ok) + 1ull)), max(cnt - 1, 0));
  if (tid != 0) return;
  Verdict v{n, NONE, -1, 0.f, 0.f, dp.c, dq.c, 0.0, 0.0};
  if (cnt > 0 && s.p[n].m - s.p[n].m == 0.f) {
    const RowSum p = s.p[n];
    v.mode = FROM_TARGET;
    v.m = p.m;
    v.ip = 1.0 / p.z;
    if (dp.greedy) {
      v.mode = CERTAIN;
      v.hot = p.col;
    } else if (n + 1 < cnt) {
      if (a.draft.x) {
        const RowSum q = s.q[n];
        if (q.m - q.m == 0.f) {
          if (dq.greedy)
            v.mode = FROM_OTHERS, v.hot = q.col;
          else
            v.mode = FROM_REST, v.mq = q.m, v.iq = 1.0 / q.z;
        }
      } else {
        const int64_t x = a.tokens[b * N + n + 1];
        v.mode = FROM_OTHERS, v.hot = x >= 0 && x < a.cols ? (int32_t)x : -1;
      }
    }
  }
  s.verdict = v;
}

// What is left of the weight of the token at col: its value in the model's row, and in the draft's
template <typename T>
struct Rest {
  const T *x, *y;
  Weigh p, q;
  double ip, iq;
  int mode, hot;
  const uint32_t *suppress;
  __device__ __forceinline__ Rest(const VerifyArgs &a, const Verdict &v, int64_t b, const double *tp, const double *tq)
      : x(row_of<T>(a.target, b, v.accepted)), y(x), p(v.c, v.m, tp), q(v.cq, v.mq, tq), ip(v.ip), iq(v.iq),
        mode(v.mode), hot(v.hot), suppress(a.suppress) {
    if (mode == FROM_REST) y = row_of<T>(a.draft, b, v.accepted);
  }
  __device__ __forceinline__ double of(float xv, float yv, int col) const {
    const double w = share(p.of<T>(xv), ip);
    if (mode == FROM_REST) return left_of(w, share(q.of<T>(yv), iq));
    return mode == FROM_OTHERS && col == hot ? 0.0 : w;
  }
  // a piece's logits in both rows, and its weights
  float xv[Cut<T>::E], yv[Cut<T>::E];
  uint32_t on;
  __device__ __forceinline__ void load(int at, const Cut<T> &cut) {
    on = piece_of(x, at, cut, suppress, xv);
    if (mode == FROM_REST) piece_of<T>(y, at, cut, nullptr, yv);
  }
  __device__ __forceinline__ void weigh(int at, double (&w)[Cut<T>::E]) const {
#pragma unroll
    for (int e = 0; e < Cut<T>::E; ++e) w[e] = (on >> e) & 1u ? of(xv[e], mode == FROM_REST ? yv[e] : 0.f, at * Cut<T>::E + e) : 0.0;
  }
};

constexpr int kDecideWaves = 16;
template <typename T>
__global__ __launch_bounds__(64 * kDecideWaves) void verify_decide_kernel(VerifyArgs a) {
  __shared__ Nodes<kDecideWaves> sNodes;
  const Cut<T> cut(a.cols);
  const VerifyWork work = verify_work(a, cut);
  decide<T, kDecideWaves>(a, work, cut, blockIdx.x, sNodes, threadIdx.x);
  if (threadIdx.x == 0) work.verdict[blockIdx.x] = sNodes.verdict;
}

// The sums of what is left of a row over 64 pieces, a piece a lane
template <typename T>
__global__ __launch_bounds__(NT) void verify_rest_kernel(VerifyArgs a, int groups, int64_t b0) {
  constexpr bool I8 = std::is_same<T, int8_t>::value;
  __shared__ double sP[I8 ? 256 : 1], sQ[I8 ? 256 : 1];
  const int tid = threadIdx.x;
  const int64_t b = b0 + (uint32_t)blockIdx.x / (uint32_t)groups;
  const Cut<T> cut(a.cols);
  const VerifyWork work = verify_work(a, cut);
  const Verdict v = work.verdict[b];
  if (v.mode != FROM_REST && v.mode != FROM_OTHERS) return;
  const int i = (int)((uint32_t)blockIdx.x % (uint32_t)groups) * kWaves + __builtin_amdgcn_readfirstlane(tid >> 6);
  Rest<T> rest(a, v, b, sP, sQ);
  const int at = 64 * i + (tid & 63);
  rest.load(at, cut);
  if (I8) {
    fill_table(sP, v.c, tid);
    if (v.mode == FROM_REST) fill_table(sQ, v.cq, tid);
    lds_barrier();
  }
  if (i >= cut.parts) return;
  double w[Cut<T>::E], z = 0.0;
  rest.weigh(at, w);
#pragma unroll
  for (int e = 0; e < Cut<T>::E; ++e) z += w[e];
  z = wave_sum_f64(z);
  if ((tid & 63) == 0) work.rest[b * cut.parts + i] = z;
}

// The token after the accepted drafts
template <typename T>
__global__ __launch_bounds__(NT) void verify_pick_kernel(VerifyArgs a) {
  constexpr bool I8 = std::is_same<T, int8_t>::value;
  __shared__ double sP[I8 ? 256 : 1], sQ[I8 ? 256 : 1];
  __shared__ double sWave[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, N = a.nodes;
  const int64_t b = blockIdx.x;
  const Cut<T> cut(a.cols);
  const VerifyWork work = verify_work(a, cut);
  Verdict v = work.verdict[b];
  const double u = (double)clamp_uniform(a.uniforms[b * N + N - 1]);
  int tok = v.mode == CERTAIN ? v.hot : -1;
  bool mine = tid == 0;
  if (v.mode == FROM_TARGET || v.mode == FROM_REST || v.mode == FROM_OTHERS) {
    if (I8) {  // seen behind the barrier below
      fill_table(sP, v.c, tid);
      if (v.mode == FROM_REST) fill_table(sQ, v.cq, tid);
    }
    Place place{-1, 0.0, 0.0, 0.0};
    if (v.mode != FROM_TARGET) {
      const double *rests = work.rest + b * cut.parts;
      place = place_of(cut.parts, u, [&](int i) { return rests[i]; }, lane);
      if (place.at < 0) v.mode = FROM_TARGET;  // nothing is left: both are the same, or the draft is no token
    }
    Rest<T> rest(a, v, b, sP, sQ);
    const bool target = v.mode == FROM_TARGET;
    if (target) {
      rest.ip = 1.0;  // weights as a sampled row has them
      const RowSpans spans(work.spans + (b * N + v.accepted) * cut.spans, cut.spans, lane);
      place = place_of(cut.spans, u, [&](int i) { return span_sum(spans.at(i), rest.p); }, lane);
    }
    if (I8) __syncthreads();
    tok = draw<T>(place, target ? kSpanPieces : 64, [&](int at, double (&w)[Cut<T>::E]) { rest.load(at, cut), rest.weigh(at, w); }, sWave, tid);
    mine = tok >= 0;
  }
  if (tid < N && tid != v.accepted) a.choice[b * N + tid] = tid < v.accepted ? a.tokens[b * N + tid + 1] : -1;
  if (mine) {
    if (v.accepted < N) a.choice[b * N + v.accepted] = tok;
    a.accepted[b] = v.accepted;
    a.next[b] = tok;
  }
}

// Launches of a row's `groups` blocks: launch(first, rows) for as many rows at a time as a grid takes, which has fewer than
// 2^32 threads.
template <typename F>
int launch_rows(int64_t rows, int64_t groups, int threads, F launch) {
  const int64_t most = ((1LL << 32) - 1) / threads / groups;
  for (int64_t first = 0; first < rows; first += most) {
    const int rc = launch(first, std::min(most, rows - first));
    if (rc) return rc;
  }
  return 0;
}

template <typename T>
int launch_spans(SpanArgs a, int64_t rows, hipStream_t s) {
  const int groups = (Cut<T>(a.cols).spans + kSpanWaves - 1) / kSpanWaves;
  return launch_rows(rows, groups, 64 * kSpanWaves, [&](int64_t first, int64_t n) {
    a.row0 = first;
    hipLaunchKernelGGL((row_spans_kernel<T>), dim3((unsigned)(n * groups)), dim3(64 * kSpanWaves), 0, s, a, groups);
    return check_launch("row_spans_kernel");
  });
}

template <typename T>
int launch_sample(const SampleArgs &a, hipStream_t s) {
  SpanArgs sp;
  sp.d[0] = sp.d[1] = a.d;
  sp.first = a.rows;
  sp.suppress = a.suppress;
  sp.cols = a.cols;
  sp.spans = static_cast<Span *>(a.workspace);
  const int rc = launch_spans<T>(sp, a.rows, s);
  if (rc) return rc;
  hipLaunchKernelGGL((sample_pick_kernel<T>), dim3((unsigned)a.rows), dim3(NT), 0, s, a);
  return check_launch("sample_pick_kernel");
}

template <typename T>
int launch_verify(const VerifyArgs &a, hipStream_t s) {
  SpanArgs sp;
  sp.d[0] = a.target;
  sp.d[1] = a.draft;
  sp.first = a.batch * a.nodes;
  sp.counts = a.counts;
  sp.suppress = a.suppress;
  sp.cols = a.cols;
  sp.spans = reinterpret_cast<Span *>(static_cast<Verdict *>(a.workspace) + a.batch);
  int rc = launch_spans<T>(sp, a.batch * (a.draft.x ? 2 * a.nodes - 1 : a.nodes), s);
  if (rc) return rc;
  hipLaunchKernelGGL((verify_decide_kernel<T>), dim3((unsigned)a.batch), dim3(64 * kDecideWaves), 0, s, a);
  rc = check_launch("verify_decide_kernel");
  if (rc) return rc;
  if (a.nodes > 1) {  // a row of one node has nothing to reject
    const int64_t groups = (Cut<T>(a.cols).parts + kWaves - 1) / kWaves;
    rc = launch_rows(a.batch, groups, NT, [&](int64_t first, int64_t n) {
      hipLaunchKernelGGL((verify_rest_kernel<T>), dim3((unsigned)(n * groups)), dim3(NT), 0, s, a, (int)groups, first);
      return check_launch("verify_rest_kernel");
    });
    if (rc) return rc;
  }
  hipLaunchKernelGGL((verify_pick_kernel<T>), dim3((unsigned)a.batch), dim3(NT), 0, s, a);
  return check_launch("verify_pick_kernel");
}

struct Sizes {
  int64_t spans, parts;
};
template <typename T>
Sizes sizes(int64_t cols) {
  const Cut<T> cut((int)cols);
  return Sizes{cut.spans, cut.parts};
}
Sizes sizes_of(int type, int64_t cols) {
  switch (type) {
    case LOGIT_I8: return sizes<int8_t>(cols);
    case LOGIT_F32: return sizes<float>(cols);
    default: return sizes<__half>(cols);
  }
}

}  // namespace

int64_t sample_workspace(int type, int64_t rows, int64_t cols) {
  return rows * sizes_of(type, cols).spans * (int64_t)sizeof(Span);
}

int64_t verify_workspace(int type, int64_t batch, int64_t nodes, int64_t cols, bool draft) {
  const int64_t rows = draft ? 2 * nodes - 1 : nodes;
  const Sizes n = sizes_of(type, cols);
  return batch * ((int64_t)sizeof(Verdict) + rows * n.spans * (int64_t)sizeof(Span) + n.parts * 8);
}

int launch_sample_tokens(const SampleArgs &a, hipStream_t s) {
  switch (a.type) {
    case LOGIT_I8: return launch_sample<int8_t>(a, s);
    case LOGIT_F32: return launch_sample<float>(a, s);
    case LOGIT_BF16: return launch_sample<__hip_bfloat16>(a, s);
    default: return launch_sample<__half>(a, s);
  }
}

int launch_verify_drafts(const VerifyArgs &a, hipStream_t s) {
  switch (a.type) {
    case LOGIT_I8: return launch_verify<int8_t>(a, s);
    case LOGIT_F32: return launch_verify<float>(a, s);
    case LOGIT_BF16: return launch_verify<__hip_bfloat16>(a, s);
    default: return launch_verify<__half>(a, s);
  }
}

}  // namespace iw
