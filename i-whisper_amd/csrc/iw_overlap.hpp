// Whether strided operands share memory: host arithmetic on their addresses, for
// entry points whose outputs lie apart from what their blocks still read.
#pragma once

#include <cstdint>

namespace iw {

// `count` runs of `bytes` bytes, `stride` bytes apart in either direction
struct Runs {
  __int128 at, bytes, stride, count;
  Runs(__int128 first, __int128 len, __int128 step, __int128 n) : at(first), bytes(len), stride(n > 1 ? step : 0), count(n) {
    if (stride < 0) at += stride * (count - 1), stride = -stride;
  }
  Runs(const void *p, __int128 len, __int128 step, __int128 n)
      : Runs((__int128) reinterpret_cast<uintptr_t>(p), len, step, n) {}
  // bytes from the first run's first to the last one's last
  __int128 reach() const { return bytes + stride * (count - 1); }
  Runs moved(__int128 by) const { return Runs(at + by, bytes, stride, count); }
};

// No run of a shares a byte with one of b. Runs of one stride may interleave; of others
// only those are taken for apart that lie behind one another.
inline bool apart(const Runs &a, const Runs &b) {
  if (a.at + a.reach() <= b.at || b.at + b.reach() <= a.at) return true;
  if (a.stride != b.stride || a.stride == 0) return false;
  // b's run i - k lies d = b.at - a.at - k * stride behind a's run i; they meet where -b.bytes < d < a.bytes
  const auto floor_div = [](__int128 x, __int128 y) { return x >= 0 ? x / y : -((y - 1 - x) / y); };
  const __int128 behind = b.at - a.at;
  const __int128 lo = floor_div(behind - a.bytes, a.stride) + 1, hi = -floor_div(-behind - b.bytes, a.stride) - 1;
  return (lo > 1 - b.count ? lo : 1 - b.count) > (hi < a.count - 1 ? hi : a.count - 1);
}

// Rows of `bytes` bytes of each batch row's nodes, at base + b * sb + i * st
struct NodeRows {
  const void *base;
  int64_t sb, st, batch, nodes, bytes;
  Runs of_row() const { return Runs(base, bytes, st, nodes); }
  // each batch row's nodes taken as one run
  Runs of_batch() const {
    const Runs r = of_row();
    return Runs(r.at, r.reach(), sb, batch);
  }
  bool same(const NodeRows &o) const {
    return base == o.base && (batch == 1 || sb == o.sb) && (nodes == 1 || st == o.st);
  }
};

// No row of x shares a byte with one of y (as many). Rows that interleave, as the columns of one
// fused projection do, are told apart where x and y have the same strides.
inline bool apart(const NodeRows &x, const NodeRows &y) {
  if (apart(x.of_batch(), y.of_batch())) return true;
  if (x.batch > 1 && x.sb != y.sb) return false;
  for (int64_t d = 1 - x.batch; d < x.batch; ++d)
    if (!apart(x.of_row(), y.of_row().moved((__int128)d * y.sb))) return false;
  return true;
}

// The rows share no byte with one another.
inline bool rows_apart(const NodeRows &x) {
  const Runs r = x.of_row(), s(x.base, x.bytes, x.sb, x.batch);
  if ((r.count > 1 && r.stride < x.bytes) || (s.count > 1 && s.stride < x.bytes)) return false;
  if (r.count == 1 || s.count == 1 || s.stride >= r.reach() || r.stride >= s.reach()) return true;
  for (__int128 d = 1; d < s.count; ++d)
    if (!apart(r, r.moved(d * s.stride))) return false;
  return true;
}

}  // namespace iw
