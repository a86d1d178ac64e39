// Rotary positions of new tokens' queries and keys: both pair layouts, part of the head, per-token positions.
//
// Every element is read and written once, so the pass is bound by HBM for prompts and by the launch for single
// tokens.  cos / sin depend on (token, pair) only: a block computes them once for its tokens into shared memory.  A thread
// has one place in the heads (16 bytes of a row, or 16 and the 16 that they are paired with) and takes it through the
// block's tokens, so that an access costs an addition and no division.  The angle in turns, position * inv_freq /
// 2 pi, is formed and reduced to [-1/2, 1/2] in fp64 (three operations per pair): in fp32 the product alone is off by
// 0.004 rad at position 131071.
// Occupancy carries it: two tokens in flight per thread (40 to 52 registers) beat four (48 to 96).  Two prompts of 8192 tokens
// with 40 heads of 128 fp16 elements, half of them turned (336 MB): 62 us, 5.4 TB/s; 11 us for 8 single tokens, which is the
// host's time to issue the call.
#include "xkv_internal.h"

namespace xkv {
namespace {

constexpr int NT = 256;
constexpr int AHEAD = 2;       // tokens that a thread has in flight
constexpr int MAX_TOKENS = 16; // per block

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T x[V]; };

// elements e, e + 1 of an access as fp32 and back
template <int V> __device__ __forceinline__ float2 two(const Vec<float, V>& v, int e) { return make_float2(v.x[e], v.x[e + 1]); }
template <int V> __device__ __forceinline__ float2 two(const Vec<__half, V>& v, int e) { return __half22float2(*reinterpret_cast<const __half2*>(v.x + e)); }
template <int V> __device__ __forceinline__ float2 two(const Vec<__nv_bfloat16, V>& v, int e) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(v.x + e));
}
template <int V> __device__ __forceinline__ void put(Vec<float, V>& v, int e, float2 f) { v.x[e] = f.x; v.x[e + 1] = f.y; }
template <int V> __device__ __forceinline__ void put(Vec<__half, V>& v, int e, float2 f) { *reinterpret_cast<__half2*>(v.x + e) = __floats2half2_rn(f.x, f.y); }
template <int V> __device__ __forceinline__ void put(Vec<__nv_bfloat16, V>& v, int e, float2 f) {
  *reinterpret_cast<__nv_bfloat162*>(v.x + e) = __floats2bfloat162_rn(f.x, f.y);
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 z, x, y, z;\n\t"
      "mov.b64 {%0, %1}, z;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

struct Args {
  xkv_rotary_params p;
  int64_t tokens;          // batch * num_tokens
  int tokens_per_block, heads;     // heads: queries and keys together
  int turn_items, items;   // per row: accesses that rotate, and all of them
};

// How an access covers pairs.  MATES: V elements that are one end of V pairs, with the other ends `half` further on;
// INSIDE: V / 2 whole neighbouring pairs; SINGLE: one neighbouring pair as two scalars, for rows that cannot be read in
// wide accesses.  Behind the rotated part an access is V elements to copy.
enum { MATES, INSIDE, SINGLE };

template <typename T, int V, int MODE>
__global__ void __launch_bounds__(NT) rotary_kernel(const Args a) {
  extern __shared__ __align__(16) float cs[];     // [tokens_per_block]{cos[half], sin[half]}, times the magnitude
  __shared__ int64_t from[MAX_TOKENS][4];   // where a token is in q, the q output, k and the k output
  const xkv_rotary_params& p = a.p;
  const int half = p.rotary_dim / 2;
  const int mate = MODE == SINGLE ? 1 : half;
  const int64_t tok0 = (int64_t)blockIdx.x * a.tokens_per_block;
  const int ntok = (int)min((int64_t)a.tokens_per_block, a.tokens - tok0);
  if (threadIdx.x < ntok) {
    const int64_t b = (tok0 + threadIdx.x) / p.num_tokens, t = (tok0 + threadIdx.x) - b * p.num_tokens;
    from[threadIdx.x][0] = b * p.q_sb + t * p.q_st;
    from[threadIdx.x][1] = b * p.qo_sb + t * p.qo_st;
    from[threadIdx.x][2] = b * p.k_sb + t * p.k_st;
    from[threadIdx.x][3] = b * p.ko_sb + t * p.ko_st;
  }
  for (int i = threadIdx.x; i < ntok * half; i += NT) {
    const int tl = i / half, j = i - tl * half;
    const int64_t b = (tok0 + tl) / p.num_tokens, t = (tok0 + tl) - b * p.num_tokens;
    const int64_t at = !p.positions ? (int64_t)p.position + t
                       : p.pos_st == 0 ? (int64_t)p.positions[b * p.pos_sb] + t : (int64_t)p.positions[b * p.pos_sb + t * p.pos_st];
    const double turns = (double)at * (p.inv_freq[j] * 0.15915494309189533577);
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[tl * p.rotary_dim + j] = p.magnitude * c;
    cs[tl * p.rotary_dim + half + j] = p.magnitude * s;
  }
  __syncthreads();

  using VT = Vec<T, V>;
  const int64_t place = (int64_t)blockIdx.y * NT + threadIdx.x;
  if (place >= (int64_t)a.heads * a.items) return;
  const int h = (int)(place / a.items), c = (int)(place - (int64_t)h * a.items);
  const bool turn = c < a.turn_items, is_q = h < p.num_heads;
  const int off = !turn ? p.rotary_dim + (c - a.turn_items) * V : MODE == SINGLE ? 2 * c : c * V;
  const float* w0 = cs + (MODE == MATES ? off : off / 2);               // of the first pair, if it turns
  const T* src = (is_q ? static_cast<const T*>(p.q) + h * p.q_sh : static_cast<const T*>(p.k) + (h - p.num_heads) * p.k_sh) + off;
  T* dst = (is_q ? static_cast<T*>(p.q_out) + h * p.qo_sh : static_cast<T*>(p.k_out) + (h - p.num_heads) * p.ko_sh) + off;
  const int which = is_q ? 0 : 2;
  for (int t0 = 0; t0 < ntok; t0 += AHEAD) {
    VT x[AHEAD], y[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (t0 + u >= ntok) break;
      const T* from_t = src + from[t0 + u][which];
      x[u] = *reinterpret_cast<const VT*>(from_t);
      if (MODE != INSIDE && turn) y[u] = *reinterpret_cast<const VT*>(from_t + mate);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (t0 + u >= ntok) break;
      T* to = dst + from[t0 + u][which + 1];
      if (turn) {
        const float* w = w0 + (t0 + u) * p.rotary_dim;
        if constexpr (V == 1) {
          const float cv = w[0], sv = w[half], a0 = to_f(x[u].x[0]), a1 = to_f(y[u].x[0]);
          x[u].x[0] = from_f<T>(a0 * cv - a1 * sv);
          y[u].x[0] = from_f<T>(a1 * cv + a0 * sv);
          *reinterpret_cast<VT*>(to + mate) = y[u];
        } else if constexpr (MODE == INSIDE) {
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            const float cv = w[e / 2], sv = w[half + e / 2];
            const float2 v = two(x[u], e);
            put(x[u], e, fma2(v, make_float2(cv, cv), mul2(make_float2(v.y, v.x), make_float2(-sv, sv))));
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            const float2 cv = *reinterpret_cast<const float2*>(w + e), sv = *reinterpret_cast<const float2*>(w + half + e);
            const float2 v = two(x[u], e), m = two(y[u], e);
            put(x[u], e, fma2(v, cv, mul2(m, make_float2(-sv.x, -sv.y))));
            put(y[u], e, fma2(m, cv, mul2(v, sv)));
          }
          *reinterpret_cast<VT*>(to + mate) = y[u];
        }
      }
      *reinterpret_cast<VT*>(to) = x[u];
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
  // tokens per block: as many as leave two blocks for each resident one, up to MAX_TOKENS
  const int64_t gy = ((int64_t)a.heads * a.items + NT - 1) / NT;
  const int64_t share = a.tokens * gy / (16 * device_sm_count());
  int tpb = share < 1 ? 1 : share > MAX_TOKENS ? MAX_TOKENS : (int)share;
  const int most = 32 * 1024 / ((int)sizeof(float2) * half);
  tpb = tpb > most ? most : tpb;
  a.tokens_per_block = tpb < 1 ? 1 : tpb;
  const int64_t gx = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  const size_t smem = (size_t)a.tokens_per_block * half * sizeof(float2);
  if (gx > 0x7fffffff || gy > 65535 || smem > 40 * 1024) return XKV_ERR_UNSUPPORTED;
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
