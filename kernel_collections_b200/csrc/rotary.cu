// Rotary positions of new tokens' queries and keys: both pair layouts, part of the head, per-token positions.
//
// Every element is read and written once, so the pass is bound by HBM for prompts and by the launch for single
// tokens.  cos / sin depend on (token, pair) only: a block computes them once for its tokens into shared memory and
// then streams all heads of those tokens through, 16 bytes per access.  The angle in turns, position * inv_freq /
// 2 pi, is formed and reduced to [-1/2, 1/2] in fp64 (three operations per pair): in fp32 the product alone is off by
// 0.004 rad at position 131071.
#include "xkv_internal.h"

namespace xkv {
namespace {

constexpr int NT = 256;
constexpr int UNROLL = 4;      // accesses a thread has in flight before it stores
constexpr int MAX_TOKENS = 64; // per block

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T x[V]; };

struct Args {
  xkv_rotary_params p;
  int64_t tokens;          // batch * num_tokens
  int tokens_per_block, heads_per_block, heads;   // heads: queries and keys together
  int turn_items, items;   // per row: accesses that rotate, and all of them
  uint64_t items_inv, heads_inv;   // ceil(2^32 / items), ceil(2^32 / heads_per_block): exact quotients of small numbers
};

// How an access covers pairs.  MATES: V elements that are one end of V pairs, with the other ends `half` further on;
// INSIDE: V / 2 whole neighbouring pairs; SINGLE: one neighbouring pair as two scalars, for rows that cannot be read in
// wide accesses.  Behind the rotated part an access is V elements to copy.
enum { MATES, INSIDE, SINGLE };

template <typename T, int V, int MODE>
__global__ void __launch_bounds__(NT) rotary_kernel(const Args a) {
  extern __shared__ float2 cs[];          // [tokens_per_block][half]: magnitude * {cos, sin}
  __shared__ int64_t from[MAX_TOKENS][4];   // offsets of a token in q, k and the outputs
  const xkv_rotary_params& p = a.p;
  const int half = p.rotary_dim / 2;
  const int mate = MODE == SINGLE ? 1 : half;
  const int64_t tok0 = (int64_t)blockIdx.x * a.tokens_per_block;
  const int ntok = (int)min((int64_t)a.tokens_per_block, a.tokens - tok0);
  const int h0 = blockIdx.y * a.heads_per_block;
  const int nh = min(a.heads_per_block, a.heads - h0);

  if (threadIdx.x < ntok) {
    const int64_t b = (tok0 + threadIdx.x) / p.num_tokens, t = (tok0 + threadIdx.x) - b * p.num_tokens;
    from[threadIdx.x][0] = b * p.q_sb + t * p.q_st;
    from[threadIdx.x][1] = b * p.k_sb + t * p.k_st;
    from[threadIdx.x][2] = b * p.qo_sb + t * p.qo_st;
    from[threadIdx.x][3] = b * p.ko_sb + t * p.ko_st;
  }
  for (int i = threadIdx.x; i < ntok * half; i += NT) {
    const int tl = i / half, j = i - tl * half;
    const int64_t b = (tok0 + tl) / p.num_tokens, t = (tok0 + tl) - b * p.num_tokens;
    const int64_t at = !p.positions ? p.position + t
                       : p.pos_st == 0 ? p.positions[b * p.pos_sb] + t : (int64_t)p.positions[b * p.pos_sb + t * p.pos_st];
    const double turns = (double)at * (p.inv_freq[j] * 0.15915494309189533577);
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[i] = make_float2(p.magnitude * c, p.magnitude * s);
  }
  __syncthreads();

  using VT = Vec<T, V>;
  const int total = ntok * nh * a.items;
  for (int base = threadIdx.x; base < total; base += NT * UNROLL) {
    VT x[UNROLL], y[UNROLL];
    T* dst[UNROLL];
    int pair[UNROLL];                     // index into cs of the first pair, -1: copy
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = base + u * NT;
      if (i >= total) break;
      const int row = (int)((uint32_t)i * a.items_inv >> 32), c = i - row * a.items;
      const int tl = nh == a.heads_per_block ? (int)((uint32_t)row * a.heads_inv >> 32) : row / nh, h = h0 + (row - tl * nh);
      const T* src;
      if (h < p.num_heads) {
        src = static_cast<const T*>(p.q) + from[tl][0] + (int64_t)h * p.q_sh;
        dst[u] = static_cast<T*>(p.q_out) + from[tl][2] + (int64_t)h * p.qo_sh;
      } else {
        const int hk = h - p.num_heads;
        src = static_cast<const T*>(p.k) + from[tl][1] + (int64_t)hk * p.k_sh;
        dst[u] = static_cast<T*>(p.k_out) + from[tl][3] + (int64_t)hk * p.ko_sh;
      }
      int off;
      if (c < a.turn_items) {
        off = MODE == SINGLE ? 2 * c : c * V;
        pair[u] = tl * half + (MODE == MATES ? off : off / 2);
      } else {
        off = p.rotary_dim + (c - a.turn_items) * V;
        pair[u] = -1;
      }
      dst[u] += off;
      x[u] = *reinterpret_cast<const VT*>(src + off);
      if (MODE != INSIDE && c < a.turn_items) y[u] = *reinterpret_cast<const VT*>(src + off + mate);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (base + u * NT >= total) break;
      if (pair[u] >= 0) {
        if (MODE == INSIDE) {
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            const float2 w = cs[pair[u] + e / 2];
            const float a0 = to_f(x[u].x[e]), a1 = to_f(x[u].x[e + 1]);
            x[u].x[e] = from_f<T>(a0 * w.x - a1 * w.y);
            x[u].x[e + 1] = from_f<T>(a1 * w.x + a0 * w.y);
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float2 w = cs[pair[u] + e];
            const float a0 = to_f(x[u].x[e]), a1 = to_f(y[u].x[e]);
            x[u].x[e] = from_f<T>(a0 * w.x - a1 * w.y);
            y[u].x[e] = from_f<T>(a1 * w.x + a0 * w.y);
          }
          *reinterpret_cast<VT*>(dst[u] + mate) = y[u];
        }
      }
      *reinterpret_cast<VT*>(dst[u]) = x[u];
    }
  }
}

bool vec_ok(const void* ptr, int64_t sb, int64_t sh, int64_t st, int es, int vec) {
  return (reinterpret_cast<uintptr_t>(ptr) % (size_t)(es * vec)) == 0 && sb % vec == 0 && sh % vec == 0 && st % vec == 0;
}

template <typename T, int V, int MODE>
int launch(Args a, cudaStream_t st) {
  const xkv_rotary_params& p = a.p;
  const int half = p.rotary_dim / 2;
  a.turn_items = MODE == INSIDE ? p.rotary_dim / V : half / V;
  // rotated in place, the elements behind the rotated part stay where they are
  const bool in_place = p.q_out == p.q && (!p.k || p.k_out == p.k);
  a.items = a.turn_items + (in_place ? 0 : (p.head_dim - p.rotary_dim) / V);
  a.heads = p.num_heads + p.num_kv_heads;
  a.tokens = (int64_t)p.batch * p.num_tokens;
  // A block wants a few accesses per thread so that the sine / cosine prologue is shared by much data; with few
  // tokens the heads are spread over blocks instead, one access per thread.
  const int per_token = a.heads * a.items;
  const bool few = a.tokens * per_token < (int64_t)2 * device_sm_count() * NT * UNROLL;
  a.heads_per_block = few ? (NT + a.items - 1) / a.items : a.heads;
  a.heads_per_block = a.heads_per_block < a.heads ? a.heads_per_block : a.heads;
  a.heads_per_block = a.heads_per_block < 256 ? a.heads_per_block : 256;
  int tpb = few ? 1 : (2 * NT * UNROLL + per_token - 1) / per_token;
  const int most = 32 * 1024 / ((int)sizeof(float2) * half);
  tpb = tpb > most ? most : tpb;
  tpb = tpb > MAX_TOKENS ? MAX_TOKENS : tpb;
  a.tokens_per_block = tpb < 1 ? 1 : tpb;
  a.items_inv = (0x100000000ull + a.items - 1) / a.items;
  a.heads_inv = (0x100000000ull + a.heads_per_block - 1) / a.heads_per_block;
  // the quotients are exact while number * divisor < 2^32
  if ((int64_t)a.tokens_per_block * a.heads_per_block * a.items * a.items >= 0x100000000ll ||
      (int64_t)a.tokens_per_block * a.heads_per_block * a.heads_per_block >= 0x100000000ll)
    return XKV_ERR_UNSUPPORTED;
  const int64_t gx = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  const int gy = ceil_div(a.heads, a.heads_per_block);
  const size_t smem = (size_t)a.tokens_per_block * half * sizeof(float2);
  if (gx > 0x7fffffff || gy > 65535 || smem > 48 * 1024) return XKV_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)gx, (unsigned)gy);
  rotary_kernel<T, V, MODE><<<grid, NT, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? XKV_OK : XKV_ERR_LAUNCH;
}

template <typename T>
int dispatch(const Args& a, cudaStream_t st) {
  const xkv_rotary_params& p = a.p;
  constexpr int V = 16 / sizeof(T);
  const int es = sizeof(T), half = p.rotary_dim / 2;
  const bool wide = (p.interleaved ? p.rotary_dim : half) % V == 0 && p.head_dim % V == 0 &&
                    vec_ok(p.q, p.q_sb, p.q_sh, p.q_st, es, V) && vec_ok(p.q_out, p.qo_sb, p.qo_sh, p.qo_st, es, V) &&
                    (!p.k || (vec_ok(p.k, p.k_sb, p.k_sh, p.k_st, es, V) && vec_ok(p.k_out, p.ko_sb, p.ko_sh, p.ko_st, es, V)));
  if (p.interleaved) return wide ? launch<T, V, INSIDE>(a, st) : launch<T, 1, SINGLE>(a, st);
  return wide ? launch<T, V, MATES>(a, st) : launch<T, 1, MATES>(a, st);
}

}  // namespace

int launch_rotary(const xkv_rotary_params& p, cudaStream_t st) {
  Args a;
  a.p = p;
  switch (p.dtype) {
    case XKV_F32: return dispatch<float>(a, st);
    case XKV_BF16: return dispatch<__nv_bfloat16>(a, st);
    case XKV_F16: return dispatch<__half>(a, st);
    default: return XKV_ERR_BAD_ARG;
  }
}

}  // namespace xkv
