// Launch wrappers of the drafted-token operators: trees of drafted tokens over
// the KV caches (iw_attn_tree.hip, iw_tree.hip) and token scores
// (iw_logprobs.hip).
#pragma once

#include "iw_kernels.hpp"

namespace iw {

constexpr int kTreeMaxNodes = 64;   // nodes of a tree: the bits of its visibility words
constexpr int kTreeMaxLayers = 64;  // layers per launch of tree_accept

// Attention of drafted nodes: `a` holds the query (q_sb, q_st), the caches
// (V transposed, v_sq == 4, or in key quads), the output and the scalars;
// a.Tq is the nodes of a row and a.Tk the positions of the caches.
struct TreeArgs {
  AttnArgs a;
  const int8_t *kn = nullptr, *vn = nullptr;  // the nodes' own K and V: [b][node][h * D + d]
  int64_t kn_sb = 0, kn_st = 0, vn_sb = 0, vn_st = 0;
  const int32_t *lengths = nullptr;           // cached keys of each row
  const uint64_t *visible = nullptr;          // [b][node] bits of the nodes that a node sees
  int64_t vis_sb = 0;
  const int32_t *counts = nullptr;            // nodes in use of each row; null = a.Tq
  uint32_t *workspace = nullptr;              // attn_tree_workspace bytes
};
int64_t attn_tree_workspace(int64_t heads, int64_t nodes, int64_t head_dim, int64_t cap);  // heads of all rows
int launch_attn_tree(const TreeArgs &t, hipStream_t s);

int launch_tree_plan(const int32_t *parents, int64_t p_ld, const int32_t *counts, const int32_t *lengths,
                     int64_t batch, int nodes, int32_t max_positions, uint64_t *visible, int32_t *positions,
                     hipStream_t s);

struct TreeAcceptArgs {
  const int64_t *tokens = nullptr, *choice = nullptr;
  const int32_t *parents = nullptr, *counts = nullptr, *lengths = nullptr;
  int64_t tok_ld = 0, ch_ld = 0, p_ld = 0;
  int64_t eot = -1;
  int32_t *path = nullptr, *accepted = nullptr, *lengths_out = nullptr;
  int64_t *next = nullptr;
  int nodes = 0, cap = 0, heads = 0, D = 0;
  int64_t kn_sb = 0, kn_st = 0, vn_sb = 0, vn_st = 0;
  int64_t k_sb = 0, k_sh = 0, k_st = 0, v_sb = 0, v_sh = 0, v_sd = 0, v_sq = 0;
};
struct TreeLayers {
  const int8_t *kn[kTreeMaxLayers], *vn[kTreeMaxLayers];
  int8_t *k[kTreeMaxLayers], *v[kTreeMaxLayers];
};
int launch_tree_accept(const TreeAcceptArgs &t, const TreeLayers &l, int layers, int64_t batch, bool first,
                       hipStream_t s);

enum LogitType { LOGIT_I8 = 0, LOGIT_F32 = 1, LOGIT_BF16 = 2, LOGIT_F16 = 3 };
constexpr int kScoreMaxTop = 32;
struct ScoreArgs {
  const void *x = nullptr;
  int type = LOGIT_I8;
  int64_t rows = 0, ld = 0;
  int cols = 0;
  float scale = 1.f, log2_hi = 0.f, log2_lo = 0.f;  // log2(e) * scale in two parts, set at launch
  float log2_far = 0.f;                             // times log2_hi: -200
  const uint32_t *suppress = nullptr;
  const int64_t *targets = nullptr;
  float *logprob = nullptr, *entropy = nullptr;
  int top = 0;
  int64_t *top_ids = nullptr;
  float *top_lp = nullptr;
  void *workspace = nullptr;
};
// bytes of the workspace for rows of cols logits
int64_t score_workspace(int type, int64_t rows, int64_t cols, int64_t top);
int launch_token_scores(const ScoreArgs &a, hipStream_t s);

}  // namespace iw
