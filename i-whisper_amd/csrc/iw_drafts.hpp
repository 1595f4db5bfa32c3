// Launch wrappers of the operators of sampled decoding with drafts: attention over a
// window of the keys and a few first ones (iw_attn_window.hip), tokens drawn by given
// random numbers and drafted tokens verified (iw_sample.hip).
#pragma once

#include "iw_kernels.hpp"

namespace iw {

// `a` holds the query (q_sb, q_st), the caches (V transposed, v_sq == 4, or in key
// quads), the output and the scalars; a.Tq is the queries of a row and a.Tk the
// positions of the caches.
struct WindowArgs {
  AttnArgs a;
  const int32_t *lengths = nullptr;    // keys of each row; null = a.Tk
  const int32_t *positions = nullptr;  // of each query: [b][query] with pos_sb between rows; null = the row's last ones
  int64_t pos_sb = 0;
  const int32_t *counts = nullptr;     // queries in use of each row; null = a.Tq
  int64_t before = 0, after = 0;       // keys before and after a query's position that it sees
  int32_t sinks = 0;                   // first keys that stay visible
  uint32_t *workspace = nullptr;       // attn_window_workspace bytes
  int64_t scores = 0;                  // words of scores in it
};
// heads of all rows
int64_t attn_window_workspace(int64_t heads, int64_t queries, int64_t head_dim, int64_t cap, int64_t before,
                              int64_t after, int64_t sinks);
int launch_attn_window(const WindowArgs &t, hipStream_t s);

// Rows of logits as distributions: weight 2^((x - max) c) with c = log2(e) * scale / T
struct DistRows {
  const void *x = nullptr;
  int64_t sb = 0, st = 0;              // row r at x + (r / inner) * sb + (r % inner) * st, in logits
  int64_t inner = 1;
  double scale = 1.0;
  double temperature = 1.0;            // of all rows, or
  const float *temperatures = nullptr; // one of each outer row
};
struct SampleArgs {
  DistRows d;
  int type = 0;                        // LogitType
  int64_t rows = 0;
  int cols = 0;
  const uint32_t *suppress = nullptr;
  const float *uniforms = nullptr;
  int64_t *tokens = nullptr;
  float *logprob = nullptr;
  void *workspace = nullptr;
};
int64_t sample_workspace(int type, int64_t rows, int64_t cols);
int launch_sample_tokens(const SampleArgs &a, hipStream_t s);

constexpr int kVerifyMaxNodes = 64;
struct VerifyArgs {
  DistRows target, draft;              // draft.x null: the drafts were certain
  int type = 0;
  int64_t batch = 0;
  int nodes = 0, cols = 0;
  const uint32_t *suppress = nullptr;
  const int64_t *tokens = nullptr;     // [batch][nodes]
  const int32_t *counts = nullptr;
  const float *uniforms = nullptr;     // [batch][nodes]
  int64_t *choice = nullptr, *next = nullptr;
  int32_t *accepted = nullptr;
  void *workspace = nullptr;
};
int64_t verify_workspace(int type, int64_t batch, int64_t nodes, int64_t cols, bool draft);
int launch_verify_drafts(const VerifyArgs &a, hipStream_t s);

}  // namespace iw
