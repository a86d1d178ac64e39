// What the kernels of xkv_tree_decode share: which rows a query token sees, and the partial results of KV splits.
//
// The num_tokens query tokens of the G heads that share a KV head are stacked into R = G * num_tokens query rows (row r:
// head r / T, token r % T), so that one pass over the keys and values serves all of them.  A KV split leaves, per
// row, its unnormalised output and (m, l): the running maximum of the scores in the log2 domain and the sum of
// exp2(score - m).  tree_merge joins the splits in split order.
#pragma once
#include "xkv_internal.h"
#include <cuda_fp8.h>
#include <math_constants.h>

namespace xkv {
namespace tree {

struct Args {
  xkv_tree_params p;
  int rows;                // R
  int splits;              // KV splits per (sequence, KV head)
  float scale_log2;        // sm_scale * log2(e)
  float* part_o;           // [batch * KVH * R][splits][head_dim]
  float2* part_ml;         // [batch * KVH * R][splits]
  int* status;
};

// Cache rows of one sequence: [0, first) is seen by every token, [first, len) holds the drafted tokens.
struct Span {
  int len, first;
};
__device__ __forceinline__ Span span_of(const xkv_tree_params& p, int b) {
  Span s;
  s.len = p.kv_lens ? min(max(p.kv_lens[b], 0), p.kv_len) : p.kv_len;
  s.first = s.len - p.num_tokens;      // negative: the first drafted tokens are absent
  return s;
}
// Whether query token t sees cache row `at` (0 <= at < len).
__device__ __forceinline__ bool sees(const xkv_tree_params& p, int b, int t, int at, int first) {
  if (at < first) return true;
  const int u = at - first;
  return p.tree_mask ? p.tree_mask[(int64_t)b * p.tm_sb + (int64_t)t * p.tm_st + u] != 0 : u <= t;
}

}  // namespace tree

// ---- host side -------------------------------------------------------------------------------------------------
struct TreePlan {
  enum Kernel { kPortable, kStream } kernel;
  const char* name;
  int rows, splits;
  size_t off_o, off_ml, total_bytes;
};
void tree_layout(const xkv_tree_params& p, TreePlan* pl);      // fills the offsets from rows and splits
int tree_merge(const tree::Args& a, cudaStream_t st);

// few query rows on mma.sync (tree_stream_sm100.cu): head_dim 64 or 128, 16-byte aligned rows
bool tree_stream_supported(const xkv_tree_params& p);
void tree_stream_plan(const xkv_tree_params& p, TreePlan* pl);     // pl->rows set
int tree_stream_decode(const tree::Args& a, cudaStream_t st);

}  // namespace xkv
