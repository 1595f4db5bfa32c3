// Trees of drafted tokens: the plan (which node sees which, at what position)
// and the acceptance of a path, with its K and V appended to the caches.
#include "iw_common.hpp"
#include "iw_tree.hpp"

namespace iw {

namespace {

// One wave per row, one lane per node. A node's word starts as its own bit;
// each of six rounds adds the word of the node 2^r levels above, so that a
// path of up to 64 nodes is closed. A parent that is no earlier node in use
// makes the node a root. A few hundred bytes a row and six exchanges: the launch
// bounds it (8 nodes 2.1 us in a graph, 128 rows of 64 2.4, both 8.8 from Python).
__global__ __launch_bounds__(256) void tree_plan_kernel(const int32_t *__restrict__ parents, int64_t p_ld,
                                                        const int32_t *__restrict__ counts,
                                                        const int32_t *__restrict__ lengths, int64_t batch,
                                                        int nodes, int32_t max_positions,
                                                        uint64_t *__restrict__ visible,
                                                        int32_t *__restrict__ positions) {
  const int lane = threadIdx.x & 63;
  const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= batch) return;
  const int cnt = counts ? clampi(counts[b], 0, nodes) : nodes;
  const bool used = lane < cnt;
  int up = used ? parents[b * p_ld + lane] : -1;
  if (up >= lane) up = -1;
  uint64_t seen = 1ull << lane;
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    const uint64_t above = __shfl(seen, max(up, 0));
    const int next = __shfl(up, max(up, 0));
    if (up >= 0) seen |= above, up = next;
  }
  if (lane >= nodes) return;
  visible[b * nodes + lane] = used ? seen : 0ull;
  if (positions) {
    const int depth = used ? __popcll(seen) - 1 : 0;
    const int64_t at = (lengths ? (int64_t)lengths[b] : 0) + depth;
    positions[b * nodes + lane] = (int32_t)max((int64_t)0, min(at, (int64_t)max_positions - 1));
  }
}

// One block per (row, layer). Every block finds the accepted path for itself:
// lane j of a wave holds node j, and the next node of the path is the first
// lane whose parent is the current node and whose token is the choice made
// after it. The path's K and V then go to the row's next cache positions. Finding the
// path again costs less than a launch to hand it over: a step of it is one ballot, and
// the K and V of an accepted node are a few KB a layer. Bound by that chain of loads and
// ballots after the launch: 1 row over 6 layers 3.0 us in a graph, 16 rows over 12 layers 4.8
// (11.7 and 12.0 from Python, whose checks and call are the most of them).
__global__ __launch_bounds__(256) void tree_accept_kernel(TreeAcceptArgs t, TreeLayers l, int layers, int write) {
  __shared__ int sPath[kTreeMaxNodes];
  __shared__ int sLen;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t b = blockIdx.x;
  const int layer = blockIdx.y;
  const int len = clampi(t.lengths[b], 0, t.cap);
  const int cnt = t.counts ? clampi(t.counts[b], 0, t.nodes) : t.nodes;
  if (tid < 64) {
    const bool used = lane < cnt;
    const int parent = used && lane > 0 ? t.parents[b * t.p_ld + lane] : -1;
    const int64_t token = used ? t.tokens[b * t.tok_ld + lane] : 0;
    const int64_t choice = used ? t.choice[b * t.ch_ld + lane] : 0;
    const int room = t.cap - len;
    int n = 0, cur = 0, mine = -1;
    int64_t want = -1;
    if (cnt > 0 && room > 0) {
      n = 1;
      if (lane == 0) mine = 0;
      for (;;) {
        want = __shfl(choice, cur);
        if (n >= room || (t.eot >= 0 && want == t.eot)) break;
        const uint64_t hit = __ballot(used && lane > cur && parent == cur && token == want);
        if (hit == 0) break;
        cur = __ffsll((long long)hit) - 1;
        if (lane == n) mine = cur;
        ++n;
      }
    }
    sPath[lane] = mine;
    if (lane == 0) sLen = n;
    if (write && layer == 0) {
      if (lane < t.nodes) t.path[b * t.nodes + lane] = mine;
      if (lane == 0) {
        t.accepted[b] = n;
        t.next[b] = want;
        t.lengths_out[b] = len + n;
      }
    }
  }
  if (layer >= layers) return;
  __syncthreads();
  const int n = sLen;
  const int8_t *kn = l.kn[layer] + b * t.kn_sb, *vn = l.vn[layer] + b * t.vn_sb;
  int8_t *kc = l.k[layer] + b * t.k_sb, *vc = l.v[layer] + b * t.v_sb;
  const int words = t.heads * t.D / 4;
  for (int i = tid; i < n * words; i += 256) {
    const int j = i / words, w = i % words, h = 4 * w / t.D, d = 4 * w % t.D;
    const int node = sPath[j], at = len + j;
    *reinterpret_cast<uint32_t *>(kc + h * t.k_sh + at * t.k_st + d) =
        *reinterpret_cast<const uint32_t *>(kn + node * t.kn_st + 4 * w);
    const uint32_t v = *reinterpret_cast<const uint32_t *>(vn + node * t.vn_st + 4 * w);
    int8_t *to = vc + h * t.v_sh + (at >> 2) * t.v_sq + (at & 3);
#pragma unroll
    for (int c = 0; c < 4; ++c) to[(d + c) * t.v_sd] = (int8_t)(v >> (8 * c));
  }
}

}  // namespace

int launch_tree_plan(const int32_t *parents, int64_t p_ld, const int32_t *counts, const int32_t *lengths,
                     int64_t batch, int nodes, int32_t max_positions, uint64_t *visible, int32_t *positions,
                     hipStream_t s) {
  hipLaunchKernelGGL(tree_plan_kernel, dim3((unsigned)((batch + 3) / 4)), dim3(256), 0, s, parents, p_ld, counts,
                     lengths, batch, nodes, max_positions, visible, positions);
  return check_launch("tree_plan_kernel");
}

int launch_tree_accept(const TreeAcceptArgs &t, const TreeLayers &l, int layers, int64_t batch, bool first,
                       hipStream_t s) {
  hipLaunchKernelGGL(tree_accept_kernel, dim3((unsigned)batch, (unsigned)(layers > 0 ? layers : 1)), dim3(256), 0, s,
                     t, l, layers, first ? 1 : 0);
  return check_launch("tree_accept_kernel");
}

}  // namespace iw
