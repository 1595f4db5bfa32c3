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
// A row is cut into spans of 4 KB, a wave each: its maximum and its sum relative to that are all
// that the first launch leaves (the one read of the logits). The row's block then adds up
// the spans, finds the one where the running sum passes u Z, and looks into that again. For
// drafts a launch between finds the first rejection, and another one the spans of max(p - q, 0).
#include <algorithm>
#include <type_traits>

#include "iw_common.hpp"
#include "iw_drafts.hpp"
#include "iw_logit_dev.hpp"
#include "iw_tree.hpp"

namespace iw {

namespace {

constexpr int kSpanBytes = 4096, kSpanPieces = kSpanBytes / 16;  // one piece a thread of a row's block
constexpr int kWaves = 4, NT = 64 * kWaves;
constexpr double kLog2E = 1.4426950408889634, kLn2 = 0.6931471805599453;

// The largest logit of a span (-inf: none that counts), for rows that take the most probable token
// its first column, and the sum of the weights relative to it
struct Span {
  float m;
  int32_t col;
  double z;
};

// ln(2)^n / n!
constexpr double exp2_term(int n) {
  double t = 1.0;
  for (int i = 1; i <= n; ++i) t = t * kLn2 / i;
  return t;
}

// 2^t, 0 far below: the nearest whole number is the exponent, of the rest (at most 1/2) the Taylor sum to its
// 11th power, off by 6e-15. A NaN (a masked logit of a row that has no other) gives 0.
__device__ __forceinline__ double exp2_64(double t) {
  t = fmax(t, -1100.0);
  const double k = rint(t), f = t - k;
  double p = exp2_term(11);
  p = fma(p, f, exp2_term(10));
  p = fma(p, f, exp2_term(9));
  p = fma(p, f, exp2_term(8));
  p = fma(p, f, exp2_term(7));
  p = fma(p, f, exp2_term(6));
  p = fma(p, f, exp2_term(5));
  p = fma(p, f, exp2_term(4));
  p = fma(p, f, exp2_term(3));
  p = fma(p, f, exp2_term(2));
  p = fma(p, f, exp2_term(1));
  p = fma(p, f, 1.0);
  return ldexp(p, (int)k);
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
// Sum of this lane's and the lower lanes' values
__device__ __forceinline__ double wave_scan_f64(double v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double t = __shfl_up(v, o);
    if (lane >= o) v += t;
  }
  return v;
}

__device__ __forceinline__ float clamp_uniform(float u) { return fminf(fmaxf(u, 0.f), 0x1.fffffep-1f); }

// 16 bytes of logits at any address of their type
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef v4u v4u_any __attribute__((aligned(1)));
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T *p) {
  const v4u x = *reinterpret_cast<const v4u_any *>(p);
  return make_uint4(x.x, x.y, x.z, x.w);
}

// The bits of the suppressed ones among n <= 16 columns from col on
__device__ __forceinline__ uint32_t hidden_bits(const uint32_t *words, int col, int n, int cols) {
  if (!words) return 0u;
  const int i = col >> 5;
  const uint64_t two = (uint64_t)words[min(i + 1, (cols - 1) >> 5)] << 32 | words[i];
  return (uint32_t)(two >> (col & 31)) & ((1u << n) - 1u);
}

// A row as a distribution, as every launch looks at it. A temperature of 0 (or none at all) gives the first
// of the largest logits all of the weight.
struct Row {
  double c;
  bool greedy;
  __device__ __forceinline__ Row(const DistRows &d, int64_t outer) {
    const double t = d.temperatures ? (double)d.temperatures[outer] : d.temperature;
    greedy = !(t > 0.0);
    c = greedy ? 0.0 : kLog2E * (d.scale / t);
  }
};
template <typename T>
__device__ __forceinline__ const T *row_of(const DistRows &d, int64_t row) {
  return reinterpret_cast<const T *>(d.x) + row / d.inner * d.sb + row % d.inner * d.st;
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
__device__ __forceinline__ void fill_table(double *table, double c, int tid) {
  for (int d = tid; d < 256; d += NT) table[d] = exp2_64(-((double)d * c));
}

template <typename T>
struct Cut {
  static constexpr int E = Logit<T>::E;
  int cols, pieces, spans;
  __host__ __device__ Cut(int cols_) : cols(cols_), pieces(cols_ / E) {
    const int n = (pieces + kSpanPieces - 1) / kSpanPieces;
    spans = n > 0 ? n : 1;
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
};

template <typename T>
__global__ __launch_bounds__(NT) void row_spans_kernel(SpanArgs a, int groups) {
  using L = Logit<T>;
  constexpr bool I8 = std::is_same<T, int8_t>::value;
  constexpr int E = L::E, P = kSpanPieces / 64;
  __shared__ double sTable[I8 ? 256 : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = (uint32_t)blockIdx.x / (uint32_t)groups;
  const int which = row >= a.first;
  const DistRows &d = a.d[which];
  const int64_t r = which ? row - a.first : row, outer = r / d.inner;
  if (a.counts && (int)(r % d.inner) >= a.counts[outer] - which) return;
  const Row dist(d, outer);
  if (I8) {
    fill_table(sTable, dist.c, tid);
    lds_barrier();
  }
  const Cut<T> cut(a.cols);
  const int s = (int)((uint32_t)blockIdx.x % (uint32_t)groups) * kWaves + __builtin_amdgcn_readfirstlane(tid >> 6);
  if (s >= cut.spans) return;
  const T *x = row_of<T>(d, r);
  const int p0 = s * kSpanPieces + lane;
  uint4 w[P];
  uint32_t off[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int at = p0 + 64 * p;
    w[p] = make_uint4(0u, 0u, 0u, 0u);
    off[p] = (1u << E) - 1u;
    if (at < cut.pieces) {
      w[p] = load_piece(x + (int64_t)at * E);
      off[p] = hidden_bits(a.suppress, at * E, E, a.cols);
    }
  }
  // what the last piece leaves, one logit a lane
  const int extra = cut.pieces * E + lane;
  const bool has_extra = s == cut.spans - 1 && extra < a.cols && !suppressed(a.suppress, extra);
  const float xe = has_extra ? L::one(x + extra) : -INFINITY;

  // NaN is the largest
  uint32_t top = has_extra ? ordered(xe) : ordered(-INFINITY);
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (!((off[p] >> e) & 1u)) top = max(top, ordered(L::get(w[p], e)));
  top = wave_max_u32_dpp(top);
  const float m = key_value((uint64_t)top << 32);

  Span out{m, -1, 0.0};
  if (dist.greedy) {
    uint32_t col = has_extra && ordered(xe) == top ? (uint32_t)extra : ~0u;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!((off[p] >> e) & 1u) && ordered(L::get(w[p], e)) == top) col = min(col, (uint32_t)((p0 + 64 * p) * E + e));
    out.col = (int32_t)~wave_max_u32_dpp(~col);
  } else {
    const Weigh wt(dist.c, m, sTable);
    double z = 0.0;
    if (has_extra) z = wt.of<T>(xe);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const double v = wt.of<T>(L::get(w[p], e));
        z += (off[p] >> e) & 1u ? 0.0 : v;
      }
    out.z = wave_sum_f64(z);
  }
  if (lane == 0) a.spans[row * cut.spans + s] = out;
}

// ---- a row's block: from the spans to a token ----
struct Block {
  double wave[kWaves];
  uint32_t max[kWaves];
  int owner;
  int found;
  double base;
};

// The largest of every thread's values, in every thread
__device__ __forceinline__ uint32_t block_max(uint32_t v, Block &s, int tid) {
  v = wave_max_u32_dpp(v);
  if ((tid & 63) == 0) s.max[tid >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v = max(v, s.max[w]);
  __syncthreads();
  return v;
}

// Which thread holds the place where the running sum of the threads' sums passes a target (made from the whole),
// and the sum below it. Only threads with a sum are asked, as rounding may lift the running sum over one without.
// If none passes, the last thread with a sum; -1 if there is none.
template <typename F>
__device__ __forceinline__ int find_owner(double sum, F target_of, double *target, double *base, Block &s, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  const double up = wave_scan_f64(sum, lane);
  if (tid == 0) s.owner = -1;
  if (lane == 63) s.wave[wave] = up;
  __syncthreads();
  double below = 0.0, total = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) below = total;
    total += s.wave[w];
  }
  *target = target_of(total);
  const uint64_t some = __ballot(sum > 0.0), passed = __ballot(sum > 0.0 && below + up > *target);
  if (lane == 0 && passed != 0) atomicMax(&s.owner, (1 << 20) + (NT - 1 - (64 * wave + __ffsll((long long)passed) - 1)));
  if (lane == 0 && some != 0) atomicMax(&s.owner, 64 * wave + 63 - __clzll((long long)some));
  __syncthreads();
  const int o = s.owner;
  const int owner = o >= 1 << 20 ? NT - 1 - (o - (1 << 20)) : o;
  if (tid == owner) s.base = below + (up - sum);
  __syncthreads();
  *base = s.base;
  __syncthreads();
  return owner;
}

// The first of a thread's n numbers whose running sum from `base` passes target, else the last above 0, else `none`
template <typename F>
__device__ __forceinline__ int find_at(int n, double *base, double target, F value, int none) {
  int got = none;
  double run = *base;
  for (int i = 0; i < n; ++i) {
    const double v = value(i);
    if (!(v > 0.0)) continue;
    got = i;
    *base = run;
    run += v;
    if (run > target) break;
  }
  return got;
}

// The token of a row whose spans have the sums span_sum(s): the place of u times their sum, found again among
// the weights(col, e) of that span's logits.
template <typename T, typename F, typename G>
__device__ __forceinline__ int draw(const Cut<T> &cut, double u, F span_sum, G weight, double *whole, Block &s, int tid) {
  constexpr int E = Cut<T>::E;
  const int each = (cut.spans + NT - 1) / NT, s0 = tid * each, n = clampi(cut.spans - s0, 0, each);
  double sum = 0.0;
  for (int i = 0; i < n; ++i) sum += span_sum(s0 + i);
  double target, base;
  int owner = find_owner(sum, [&](double total) { *whole = total; return u * total; }, &target, &base, s, tid);
  if (owner < 0) return -1;  // no weight at all
  if (tid == owner) {
    s.found = s0 + find_at(n, &base, target, [&](int i) { return span_sum(s0 + i); }, 0);
    s.base = base;
  }
  __syncthreads();
  const int span = s.found;
  const double below = s.base;
  __syncthreads();
  // a piece a thread, the row's last logits with the last piece
  const int first = span * kSpanPieces, here = min(cut.pieces - first, kSpanPieces);
  const int col = (first + tid) * E;
  int m = tid < here ? E : 0;
  if (span == cut.spans - 1 && tid == max(here - 1, 0)) m = cut.cols - col;
  sum = 0.0;
  for (int i = 0; i < m; ++i) sum += weight(col + i);
  owner = find_owner(sum, [&](double) { return target - below; }, &target, &base, s, tid);
  if (owner < 0) return -1;
  if (tid == owner) s.found = col + find_at(m, &base, target, [&](int i) { return weight(col + i); }, 0);
  __syncthreads();
  return s.found;
}

// a row's largest logit; its first column for rows that take it
template <typename T>
__device__ __forceinline__ float row_max(const Span *spans, const Cut<T> &cut, bool greedy, int *col, Block &s, int tid) {
  uint32_t top = 0;
  for (int i = tid; i < cut.spans; i += NT) top = max(top, ordered(spans[i].m));
  top = block_max(top, s, tid);
  if (greedy) {
    uint32_t c = 0;
    for (int i = tid; i < cut.spans; i += NT)
      if (ordered(spans[i].m) == top) c = max(c, ~(uint32_t)spans[i].col);
    *col = (int)~block_max(c, s, tid);
  }
  return key_value((uint64_t)top << 32);
}

// A span's sum relative to the row's largest logit; 0 where its logits' weights are next to vanishing, so that
// a span with a sum has a logit with a weight.
__device__ __forceinline__ double span_sum(const Span &s, const Weigh &row) {
  const double z = s.z * exp2_64(row.log2_of(s.m));
  return z > 1e-290 ? z : 0.0;
}

template <typename T>
__global__ __launch_bounds__(NT) void sample_pick_kernel(SampleArgs a) {
  using L = Logit<T>;
  constexpr bool I8 = std::is_same<T, int8_t>::value;
  __shared__ double sTable[I8 ? 256 : 1];
  __shared__ Block s;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const Cut<T> cut(a.cols);
  const Row dist(a.d, row / a.d.inner);
  const Span *spans = static_cast<const Span *>(a.workspace) + row * cut.spans;
  const T *x = row_of<T>(a.d, row);
  if (I8) fill_table(sTable, dist.c, tid);
  int tok = -1;
  const float m = row_max(spans, cut, dist.greedy, &tok, s, tid);
  float lp = 0.f;
  if (!(m - m == 0.f)) {  // no distribution: a NaN, an infinity, nothing to choose from
    tok = -1;
    lp = __uint_as_float(0x7fc00000u);
  } else if (!dist.greedy) {
    const Weigh wt(dist.c, m, sTable);
    double z = 0.0;
    tok = draw(cut, (double)clamp_uniform(a.uniforms[row]),
               [&](int i) { return span_sum(spans[i], wt); },
               [&](int col) { return suppressed(a.suppress, col) ? 0.0 : wt.of<T>(L::one(x + col)); }, &z, s, tid);
    if (tid == 0) lp = (float)(wt.log2_of(L::one(x + tok)) * kLn2 - log(z));
  }
  if (tid == 0) {
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
__device__ __forceinline__ RowSum row_sum(const Span *spans, int n, const Row &dist, int lane) {
  uint32_t top = 0;
  for (int i = lane; i < n; i += 64) top = max(top, ordered(spans[i].m));
  top = wave_max_u32_dpp(top);
  RowSum r;
  r.m = key_value((uint64_t)top << 32);
  r.col = -1;
  r.z = 1.0;
  if (dist.greedy) {
    uint32_t c = 0;
    for (int i = lane; i < n; i += 64)
      if (ordered(spans[i].m) == top) c = max(c, ~(uint32_t)spans[i].col);
    r.col = (int32_t)~wave_max_u32_dpp(c);
  } else {
    const Weigh wt(dist.c, r.m, nullptr);
    double z = 0.0;
    for (int i = lane; i < n; i += 64) z += span_sum(spans[i], wt);
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
  return share(exp2_64(wt.log2_of(Logit<T>::one(x + col))), 1.0 / r.z);
}

struct VerifyWork {
  Span *spans;      // of the target's rows, then of the draft's
  double *rest;     // [batch][spans]
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

// One block per batch row, its waves take the nodes in turn.
template <typename T>
__global__ __launch_bounds__(NT) void verify_decide_kernel(VerifyArgs a) {
  __shared__ RowSum sP[kVerifyMaxNodes], sQ[kVerifyMaxNodes];
  __shared__ int sOk[kVerifyMaxNodes];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t b = blockIdx.x;
  const Cut<T> cut(a.cols);
  const VerifyWork w = verify_work(a, cut);
  const int N = a.nodes, cnt = a.counts ? clampi(a.counts[b], 0, N) : N;
  const Row dp(a.target, b), dq(a.draft, b);
  for (int i = tid >> 6; i < cnt; i += kWaves) {
    const int64_t row = b * N + i, drow = b * (N - 1) + i;
    const RowSum p = row_sum(w.spans + row * cut.spans, cut.spans, dp, lane);
    RowSum q{0.f, -1, 1.0};
    bool ok = false;
    if (i + 1 < cnt) {
      const int64_t x = a.tokens[row + 1];
      const double px = share_of(row_of<T>(a.target, row), x, a.cols, a.suppress, dp, p);
      double qx = 1.0;
      if (a.draft.x) {
        q = row_sum(w.spans + (a.batch * N + drow) * cut.spans, cut.spans, dq, lane);
        qx = share_of(row_of<T>(a.draft, drow), x, a.cols, a.suppress, dq, q);
        if (!(q.m - q.m == 0.f)) qx = __longlong_as_double(0x7ff8000000000000ll);  // a draft without a distribution
      }
      ok = p.m - p.m == 0.f && (double)clamp_uniform(a.uniforms[row]) * qx < px;
    }
    if (lane == 0) sP[i] = p, sQ[i] = q, sOk[i] = ok;
  }
  __syncthreads();
  if (tid != 0) return;
  int n = 0;
  while (n + 1 < cnt && sOk[n]) ++n;
  Verdict v{n, NONE, -1, 0.f, 0.f, dp.c, dq.c, 0.0, 0.0};
  if (cnt > 0 && sP[n].m - sP[n].m == 0.f) {
    const RowSum p = sP[n], q = sQ[n];
    v.mode = FROM_TARGET;
    v.m = p.m;
    v.ip = 1.0 / p.z;
    if (dp.greedy) {
      v.mode = CERTAIN;
      v.hot = p.col;
    } else if (n + 1 < cnt) {
      if (a.draft.x && !dq.greedy) {
        if (q.m - q.m == 0.f) v.mode = FROM_REST, v.mq = q.m, v.iq = 1.0 / q.z;
      } else {
        const int64_t x = a.draft.x ? q.col : a.tokens[b * N + n + 1];
        if (!a.draft.x || q.m - q.m == 0.f) v.mode = FROM_OTHERS, v.hot = x >= 0 && x < a.cols ? (int32_t)x : -1;
      }
    }
  }
  w.verdict[b] = v;
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
      : x(row_of<T>(a.target, b * a.nodes + v.accepted)), y(x), p(v.c, v.m, tp), q(v.cq, v.mq, tq), ip(v.ip), iq(v.iq),
        mode(v.mode), hot(v.hot), suppress(a.suppress) {
    if (mode == FROM_REST) y = row_of<T>(a.draft, b * (a.nodes - 1) + v.accepted);
  }
  __device__ __forceinline__ double of(float xv, float yv, int col) const {
    const double w = share(p.of<T>(xv), ip);
    if (mode == FROM_REST) return left_of(w, share(q.of<T>(yv), iq));
    return mode == FROM_OTHERS && col == hot ? 0.0 : w;
  }
  __device__ __forceinline__ double at(int col) const {
    if (suppressed(suppress, col)) return 0.0;
    return of(Logit<T>::one(x + col), mode == FROM_REST ? Logit<T>::one(y + col) : 0.f, col);
  }
};

template <typename T>
__global__ __launch_bounds__(NT) void verify_rest_kernel(VerifyArgs a, int groups) {
  using L = Logit<T>;
  constexpr bool I8 = std::is_same<T, int8_t>::value;
  constexpr int E = L::E, P = kSpanPieces / 64;
  __shared__ double sP[I8 ? 256 : 1], sQ[I8 ? 256 : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t b = (uint32_t)blockIdx.x / (uint32_t)groups;
  const Cut<T> cut(a.cols);
  const VerifyWork w = verify_work(a, cut);
  const Verdict v = w.verdict[b];
  if (v.mode != FROM_REST && v.mode != FROM_OTHERS) return;
  if (I8) {
    fill_table(sP, v.c, tid);
    fill_table(sQ, v.cq, tid);
    lds_barrier();
  }
  const int s = (int)((uint32_t)blockIdx.x % (uint32_t)groups) * kWaves + __builtin_amdgcn_readfirstlane(tid >> 6);
  if (s >= cut.spans) return;
  const Rest<T> rest(a, v, b, sP, sQ);
  double z = 0.0;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int at = s * kSpanPieces + 64 * p + lane;
    if (at < cut.pieces) {
      const uint4 xp = load_piece(rest.x + (int64_t)at * E), yp = load_piece(rest.y + (int64_t)at * E);
      const uint32_t off = hidden_bits(a.suppress, at * E, E, a.cols);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const double one = rest.of(L::get(xp, e), L::get(yp, e), at * E + e);
        z += (off >> e) & 1u ? 0.0 : one;
      }
    }
  }
  const int extra = cut.pieces * E + lane;
  if (s == cut.spans - 1 && extra < a.cols) z += rest.at(extra);
  z = wave_sum_f64(z);
  if (lane == 0) w.rest[b * cut.spans + s] = z;
}

template <typename T>
__global__ __launch_bounds__(NT) void verify_pick_kernel(VerifyArgs a) {
  constexpr bool I8 = std::is_same<T, int8_t>::value;
  __shared__ double sP[I8 ? 256 : 1], sQ[I8 ? 256 : 1];
  __shared__ Block s;
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x;
  const Cut<T> cut(a.cols);
  const VerifyWork w = verify_work(a, cut);
  Verdict v = w.verdict[b];
  const int N = a.nodes;
  if (I8) {
    fill_table(sP, v.c, tid);
    fill_table(sQ, v.cq, tid);
    __syncthreads();
  }
  int tok = v.mode == CERTAIN ? v.hot : -1;
  const double u = (double)clamp_uniform(a.uniforms[b * N + N - 1]);
  double whole;
  if (v.mode == FROM_REST || v.mode == FROM_OTHERS) {
    const Rest<T> rest(a, v, b, sP, sQ);
    const double *sums = w.rest + b * cut.spans;
    tok = draw(cut, u, [&](int i) { return sums[i]; }, [&](int col) { return rest.at(col); }, &whole, s, tid);
    if (tok < 0) v.mode = FROM_TARGET;  // nothing is left: both are the same, or the draft is no token
    __syncthreads();
  }
  if (v.mode == FROM_TARGET) {
    const Rest<T> rest(a, v, b, sP, sQ);
    const Span *spans = w.spans + (b * N + v.accepted) * cut.spans;
    tok = draw(cut, u, [&](int i) { return rest.ip * span_sum(spans[i], rest.p); },
               [&](int col) { return rest.at(col); }, &whole, s, tid);
  }
  if (tid < N) {
    int64_t c = -1;
    if (tid < v.accepted) c = a.tokens[b * N + tid + 1];
    if (tid == v.accepted) c = tok;
    a.choice[b * N + tid] = c;
  }
  if (tid == 0) {
    a.accepted[b] = v.accepted;
    a.next[b] = tok;
  }
}

template <typename T>
int launch_spans(SpanArgs a, int64_t rows, hipStream_t s) {
  const int groups = (Cut<T>(a.cols).spans + kWaves - 1) / kWaves;
  if (rows * groups >= (1LL << 32) / NT) return fail("too many logits for one call");
  hipLaunchKernelGGL((row_spans_kernel<T>), dim3((unsigned)(rows * groups)), dim3(NT), 0, s, a, groups);
  return check_launch("row_spans_kernel");
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
  hipLaunchKernelGGL((verify_decide_kernel<T>), dim3((unsigned)a.batch), dim3(NT), 0, s, a);
  rc = check_launch("verify_decide_kernel");
  if (rc) return rc;
  const int groups = (Cut<T>(a.cols).spans + kWaves - 1) / kWaves;
  if (a.nodes > 1) {  // a row of one node has nothing to reject
    hipLaunchKernelGGL((verify_rest_kernel<T>), dim3((unsigned)(a.batch * groups)), dim3(NT), 0, s, a, groups);
    rc = check_launch("verify_rest_kernel");
    if (rc) return rc;
  }
  hipLaunchKernelGGL((verify_pick_kernel<T>), dim3((unsigned)a.batch), dim3(NT), 0, s, a);
  return check_launch("verify_pick_kernel");
}

int64_t spans_of(int type, int64_t cols) {
  switch (type) {
    case LOGIT_I8: return Cut<int8_t>((int)cols).spans;
    case LOGIT_F32: return Cut<float>((int)cols).spans;
    default: return Cut<__half>((int)cols).spans;
  }
}

}  // namespace

int64_t sample_workspace(int type, int64_t rows, int64_t cols) {
  return rows * spans_of(type, cols) * (int64_t)sizeof(Span);
}

int64_t verify_workspace(int type, int64_t batch, int64_t nodes, int64_t cols, bool draft) {
  const int64_t rows = draft ? 2 * nodes - 1 : nodes, spans = spans_of(type, cols);
  return batch * ((int64_t)sizeof(Verdict) + rows * spans * (int64_t)sizeof(Span) + spans * 8);
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
