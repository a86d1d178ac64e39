// What the kernels of xkv_tree_decode share: which rows a query token sees, how the work is dealt to blocks, and the
// partial results.
//
// The num_tokens query tokens of the G heads that share a KV head are stacked into R = G * num_tokens query rows (row r:
// head r / T, token r % T), so that one pass over the keys and values serves all of them; a kernel takes them in blocks of
// `block_rows`.  A strip is one (sequence, KV head, row block); strips are numbered in that order.
//
// Work is dealt in units of `unit_tokens` cache rows.  All units of all strips form one line, cut into equal shares for
// the blocks of a single wave: sequences of any lengths keep every block equally busy, and one long sequence is spread
// over all of them.  The lengths are on the device, so every block finds its own share (a scan over the batch).  A
// block's stretch of one strip is a piece.  A piece that covers its strip is finished by its block.  At most two pieces of a
// block do not: its first, which goes on with a strip that another block began, and its last, which begins one; block c
// keeps them in the places 2c and 2c + 1.  Of such a piece it leaves, per row, the unnormalised output and (m, l): the reference of the exponents in the log2
// domain and the sum of exp2(score - m), and the merge joins a strip's pieces in their order.
#pragma once
#include "xkv_internal.h"
#include <cuda_fp8.h>
#include <math_constants.h>

namespace xkv {
namespace tree {

struct Args {
  xkv_tree_params p;
  int rows;                // R
  int block_rows, blocks;  // rows per strip, strips per (sequence, KV head)
  int unit_tokens;
  int grid;                // blocks that share the units
  float scale_log2;        // sm_scale * log2(e)
  float* part_o;           // [place][block_rows][head_dim]
  float2* part_ml;         // [place][block_rows]
  int* status;
  int map_b[2], map_h[2];  // tensor maps of K and V: 0 where the sequences / KV heads share one (stride 0)
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

// units of a strip of sequence b: at least one, so that empty sequences are written (as zeros) too
__device__ __forceinline__ int units_of(const Args& a, int len) { return max(1, (len + a.unit_tokens - 1) / a.unit_tokens); }

// Where the line stands; computed by every warp for itself.
struct Line {
  int64_t total, share;      // units of all strips; units per block
};
struct Spot {
  int b, units;              // sequence, units of each of its strips
  int64_t before;            // units of the sequences in front of it
};
__device__ __forceinline__ int strip_units(const Args& a, int b) {
  return units_of(a, a.p.kv_lens ? min(max(a.p.kv_lens[b], 0), a.p.kv_len) : a.p.kv_len);
}
__device__ __forceinline__ Line line_of(const Args& a, int lane) {
  Line l;
  const int64_t per = (int64_t)a.p.num_kv_heads * a.blocks;
  if (!a.p.kv_lens) {
    l.total = per * a.p.batch * units_of(a, a.p.kv_len);
  } else {
    int64_t sum = 0;
    for (int b = lane; b < a.p.batch; b += 32) sum += strip_units(a, b);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l.total = per * sum;
  }
  l.share = (l.total + a.grid - 1) / a.grid;
  return l;
}
// the sequence that holds unit x of the line (0 <= x < total)
__device__ __forceinline__ Spot find_unit(const Args& a, int64_t x, int lane) {
  Spot s;
  const int64_t per = (int64_t)a.p.num_kv_heads * a.blocks;
  if (!a.p.kv_lens) {
    s.units = units_of(a, a.p.kv_len);
    s.b = (int)(x / (per * s.units));
    s.before = s.b * per * s.units;
    return s;
  }
  int64_t before = 0;
  for (int b0 = 0;; b0 += 32) {
    const int u = b0 + lane < a.p.batch ? strip_units(a, b0 + lane) : 0;
    int64_t upto = u;                  // inclusive scan
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, before + upto * per > x);
    if (hit || b0 + 32 >= a.p.batch) {
      const int at = hit ? __ffs(hit) - 1 : 31;
      s.b = b0 + at;
      s.units = __shfl_sync(0xffffffffu, u, at);
      s.before = before + (__shfl_sync(0xffffffffu, upto, at) - s.units) * per;
      return s;
    }
    before += __shfl_sync(0xffffffffu, upto, 31) * per;
  }
}
// the units of the sequences in front of sequence b
__device__ __forceinline__ Spot find_sequence(const Args& a, int b, int lane) {
  Spot s;
  s.b = b;
  s.units = strip_units(a, b);
  const int64_t per = (int64_t)a.p.num_kv_heads * a.blocks;
  if (!a.p.kv_lens) {
    s.before = b * per * s.units;
    return s;
  }
  int64_t sum = 0;
  for (int i = lane; i < b; i += 32) sum += strip_units(a, i);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  s.before = per * sum;
  return s;
}

// A block's walk over its share: `next` gives one piece after the other.
struct Piece {
  int b, h, rb;              // sequence, KV head, row block
  int begin, end;            // units
  bool whole;                // covers its strip
  int64_t id;                // its place among the partial results
};
struct Walk {
  int64_t x, stop;
  Spot at;
};
__device__ __forceinline__ Walk walk_of(const Args& a, int lane) {
  const Line l = line_of(a, lane);
  Walk w;
  w.x = blockIdx.x * l.share;
  w.stop = min(w.x + l.share, l.total);
  if (w.x < w.stop) w.at = find_unit(a, w.x, lane);
  return w;
}
__device__ __forceinline__ bool next_piece(const Args& a, Walk& w, Piece& pc) {
  if (w.x >= w.stop) return false;
  const int per = a.p.num_kv_heads * a.blocks;
  if (w.x - w.at.before >= (int64_t)per * w.at.units) {
    w.at.before += (int64_t)per * w.at.units;
    w.at.units = strip_units(a, ++w.at.b);
  }
  const int64_t y = w.x - w.at.before;
  const int strip = (int)(y / w.at.units);
  pc.b = w.at.b;
  pc.h = strip / a.blocks;
  pc.rb = strip - pc.h * a.blocks;
  pc.begin = (int)(y - (int64_t)strip * w.at.units);
  pc.end = (int)min((int64_t)w.at.units, pc.begin + (w.stop - w.x));
  pc.whole = pc.begin == 0 && pc.end == w.at.units;
  pc.id = 2 * (int64_t)blockIdx.x + (pc.begin == 0);
  w.x += pc.end - pc.begin;
  return true;
}

// Whole powers of two, for the references of the exponents and the factors between them.
// 2^x for a whole x up to 127; 0 below the smallest fp32 (x = -infinity included)
__device__ __forceinline__ float pow2(float x) {
  const int k = (int)fmaxf(x, -150.f);
  return k >= -126 ? __uint_as_float((uint32_t)(k + 127) << 23) : k >= -149 ? __uint_as_float(1u << (k + 149)) : 0.f;
}
// the factor from reference `from` to `to`
__device__ __forceinline__ float moved(float from, float to) { return from == to ? 1.f : pow2(from - to); }
// log2 |x|, absolute error below 2^-20; -infinity for 0 and for what is not finite
__device__ __forceinline__ float log2_size(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(fabsf(x)));
  return y < CUDART_INF_F ? y : -CUDART_INF_F;
}

// Over 8-bit caches the product takes weight * value scale, and the reference of the exponents (a whole number) follows the
// largest such product, not the largest scale: a row without weight takes no bits from the others, however large its values.
// The weights and their sum l carry the same reference.  It stays within FLOOR bits below the largest score, so that they stay below
// 2^127; above it lies at most the largest scale (up to 2^112 weights down to 2^-20 of the largest remain in fp32).
constexpr float FLOOR = 90.f;
constexpr float LARGEST_PRODUCT = 32768.f, LARGEST_SUM = 8.5070592e37f;      // 2^15 (fp16 ends at 65504); 2^126
// References of pieces may lie far apart, so sums are brought to 1..2 before pieces are joined by their weights: returns the factor
// on O and moves l and m accordingly.
__device__ __forceinline__ float settle_sum(float& m, float& l) {
  if (!(l > 0.f && l < CUDART_INF_F)) return 1.f;
  const float e = (float)((int)(__float_as_uint(l) >> 23) - 127), f = pow2(-e);
  l *= f;
  m += e;
  return f;
}

}  // namespace tree

// ---- host side -------------------------------------------------------------------------------------------------
struct TreePlan {
  enum Kernel { kPortable, kStream, kTc } kernel;
  const char* name;
  int rows, block_rows, unit_tokens, slots;      // slots: blocks of the kernel that the device holds at once
  int blocks, grid;
  bool merged;                                   // some strip may be cut into pieces
  size_t off_o, off_ml, total_bytes;
};
int tree_merge(const tree::Args& a, cudaStream_t st);

// few query rows on mma.sync (tree_stream_sm100.cu): head_dim 64 or 128, 16-byte aligned rows
bool tree_stream_supported(const xkv_tree_params& p);
void tree_stream_plan(const xkv_tree_params& p, TreePlan* pl);
int tree_stream_decode(const tree::Args& a, cudaStream_t st);

// many query rows on tcgen05 (tree_tc_sm100.cu): what the stream kernel takes, 16-bit queries, more than 16 rows
bool tree_tc_supported(const xkv_tree_params& p, int rows);
void tree_tc_plan(const xkv_tree_params& p, TreePlan* pl);
int tree_tc_decode(const tree::Args& a, cudaStream_t st);

}  // namespace xkv
