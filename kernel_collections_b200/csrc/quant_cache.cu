// Writing rows to an 8-bit key / value cache and reading them back.
//
// One row (token, KV head) is reduced to its largest magnitude, scaled and rounded: scale = top * (1 / C), code =
// rn(x * (C * (1 / top))), every operation rounded to fp32.  Both directions move every byte once and are bound by HBM for long stretches and by the launch for single
// tokens.  A row is held in registers by a power-of-two group of lanes (16 bytes per lane and access), so the
// reduction is a few shuffles and nothing is read twice.  Sequence and head come from the block's indices: one 64-bit
// division per row costs more than the row's arithmetic.
// int8 codes are made and read by byte permutes and additions of a power of two instead of conversion instructions, 16-bit
// maxima in pairs: at 8 elements per SM and clock of HBM traffic the conversions were the bound.  4 x 8192 rows of 8 heads
// of 128 fp16 elements written as e4m3 and read back (407 MB): 99 us, 4.1 TB/s; 100003 rows of 8 x 64 int8 codes read
// as bf16 (314 MB): 71 us, 4.4 TB/s.
#include "xkv_internal.h"
#include <cuda_fp8.h>
#include <math_constants.h>

namespace xkv {
namespace {

constexpr int NT = 128;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T x[V]; };

template <int CODE> __device__ __forceinline__ constexpr float largest() { return CODE == XKV_CACHE_INT8 ? 127.f : 448.f; }

__device__ __forceinline__ float max_nan(float a, float b) {      // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ __half2 abs_max(__half2 a, __half2 b) { return __hmax2_nan(a, __habs2(b)); }
__device__ __forceinline__ __nv_bfloat162 abs_max(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, __habs2(b)); }
template <typename T> struct Pair;
template <> struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ float2 up(__half2 v) { return __half22float2(v); }
  static __device__ __forceinline__ __half2 down(float2 v) { return __floats2half2_rn(v.x, v.y); }
};
template <> struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ float2 up(__nv_bfloat162 v) { return __bfloat1622float2(v); }
  static __device__ __forceinline__ __nv_bfloat162 down(float2 v) { return __floats2bfloat162_rn(v.x, v.y); }
};

// the largest magnitude, or NaN; 16-bit types compare in pairs (exact)
template <typename T, int V> __device__ __forceinline__ float largest_of(const Vec<T, V>& x) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    using P = typename Pair<T>::type;
    const P* q = reinterpret_cast<const P*>(x.x);
    P m = __habs2(q[0]);
#pragma unroll
    for (int e = 1; e < V / 2; ++e) m = abs_max(m, q[e]);
    const float2 f = Pair<T>::up(m);
    return max_nan(f.x, f.y);
  } else {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) m = max_nan(m, fabsf(to_f(x.x[e])));
    return m;
  }
}
template <typename T, int V> __device__ __forceinline__ float2 two_of(const Vec<T, V>& x, int e) {
  if constexpr (sizeof(T) == 2) return Pair<T>::up(reinterpret_cast<const typename Pair<T>::type*>(x.x)[e / 2]);
  else return make_float2(x.x[e], x.x[e + 1]);
}

// codes of x * per.  |x * per| is at most C (1 + 2^-22) (a reciprocal and two products, each rounded once), which still
// rounds to C: nothing to clamp.  int8: adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the
// low byte.
template <typename T, int CODE, int V> __device__ __forceinline__ Vec<uint8_t, V> encode(const Vec<T, V>& x, float per) {
  Vec<uint8_t, V> c;
  if constexpr (V % 4 == 0) {
    uint32_t* out = reinterpret_cast<uint32_t*>(c.x);
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      float2 a = two_of(x, e), b = two_of(x, e + 2);
      if (CODE == XKV_CACHE_INT8) {
        // the product is rounded before the sum: paired instructions were seen to become one fused multiply-add here
        a.x = __fadd_rn(__fmul_rn(a.x, per), 12582912.f);
        a.y = __fadd_rn(__fmul_rn(a.y, per), 12582912.f);
        b.x = __fadd_rn(__fmul_rn(b.x, per), 12582912.f);
        b.y = __fadd_rn(__fmul_rn(b.y, per), 12582912.f);
        out[e / 4] = __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040u),
                                 __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040u), 0x5410u);
      } else {
        a = mul2(a, make_float2(per, per));
        b = mul2(b, make_float2(per, per));
        out[e / 4] = (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
                     (uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float y = __fmul_rn(to_f(x.x[e]), per);
      c.x[e] = CODE == XKV_CACHE_INT8 ? (uint8_t)__float_as_uint(__fadd_rn(y, 12582912.f)) : __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
    }
  }
  return c;
}
// code * scale.  int8: a code with its sign bit flipped under the upper bytes of 2^23 is the float 2^23 + 128 + code.
template <typename T, int CODE, int V> __device__ __forceinline__ Vec<T, V> decode(const Vec<uint8_t, V>& c, float scale) {
  Vec<T, V> x;
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(c.x)[e / 4];
      float2 a, b;
      if (CODE == XKV_CACHE_INT8) {
        const uint32_t y = w ^ 0x80808080u;
        const float2 off = make_float2(-8388736.f, -8388736.f);
        a = add2(make_float2(__uint_as_float(__byte_perm(y, 0x4b000000u, 0x7440u)), __uint_as_float(__byte_perm(y, 0x4b000000u, 0x7441u))), off);
        b = add2(make_float2(__uint_as_float(__byte_perm(y, 0x4b000000u, 0x7442u)), __uint_as_float(__byte_perm(y, 0x4b000000u, 0x7443u))), off);
      } else {
        a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3)));
        b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3)));
      }
      a = mul2(a, make_float2(scale, scale));
      b = mul2(b, make_float2(scale, scale));
      if constexpr (sizeof(T) == 2) {
        reinterpret_cast<typename Pair<T>::type*>(x.x)[e / 2] = Pair<T>::down(a);
        reinterpret_cast<typename Pair<T>::type*>(x.x)[e / 2 + 1] = Pair<T>::down(b);
      } else {
        x.x[e] = a.x; x.x[e + 1] = a.y; x.x[e + 2] = b.x; x.x[e + 3] = b.y;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float y = CODE == XKV_CACHE_INT8 ? (float)(int8_t)c.x[e] : __half2float(__half(__nv_cvt_fp8_to_halfraw(c.x[e], __NV_E4M3)));
      x.x[e] = from_f<T>(y * scale);
    }
  }
  return x;
}

// A block works on one (sequence, KV head) of the keys or of the values: grid (token chunks, KV heads, 2 x
// sequences).  `lanes` (a power of two, at most 32) lanes hold one row; a thread has its accesses of U rows in flight.
// Many small blocks that sweep memory in order reach more of HBM than one wave of blocks that loop with the next rows
// asked for ahead, each in a stretch of its own (four prompts of 8192 rows written and read back: 101 us against 148).
struct Place {
  int64_t start;      // cache row of token 0
  int tokens;         // of this sequence
  bool values;
  int group, groups, lane;
};
__device__ __forceinline__ Place place_of(const xkv_cache_params& p, int lanes) {
  Place w;
  const int b = blockIdx.z >> 1;
  w.values = blockIdx.z & 1;
  w.start = p.positions ? p.positions[b] : p.position;
  w.tokens = p.num_tokens;
  w.groups = NT / lanes;
  w.group = threadIdx.x / lanes;
  w.lane = threadIdx.x & (lanes - 1);
  return w;
}

// NV accesses of V elements per lane and row.
template <typename T, int CODE, int V, int NV, int U>
__global__ void __launch_bounds__(NT, NV == 1 ? 12 : 1) append_kernel(const xkv_cache_params p, int lanes) {
  const int h = blockIdx.y, b = blockIdx.z >> 1;
  Place w = place_of(p, lanes);
  if (p.lengths) w.tokens = min(w.tokens, p.lengths[b]);
  const int t0 = blockIdx.x * (w.groups * U) + w.group;
  const int64_t st = w.values ? p.v_st : p.k_st;
  const T* src = (w.values ? static_cast<const T*>(p.v) + b * p.v_sb + h * p.v_sh : static_cast<const T*>(p.k) + b * p.k_sb + h * p.k_sh);
  Vec<T, V> x[U][NV];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = t0 + u * w.groups;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int d = (i * lanes + w.lane) * V;
      if (t < w.tokens && d < p.head_dim) x[u][i] = *reinterpret_cast<const Vec<T, V>*>(src + t * st + d);
    }
  }
  uint8_t* codes = w.values ? static_cast<uint8_t*>(p.v_codes) + b * p.vc_sb + h * p.vc_sh : static_cast<uint8_t*>(p.k_codes) + b * p.kc_sb + h * p.kc_sh;
  float* scales = w.values ? p.v_scales + b * p.vs_sb + h * p.vs_sh : p.k_scales + b * p.ks_sb + h * p.ks_sh;
  const int64_t sl = w.values ? p.vc_sl : p.kc_sl;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = t0 + u * w.groups;
    const int64_t at = w.start + t;
    const bool live = t < w.tokens && at >= 0 && at < p.capacity;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t < w.tokens && (i * lanes + w.lane) * V < p.head_dim) top = max_nan(top, largest_of(x[u][i]));
    for (int o = lanes >> 1; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live) continue;
    const bool finite = top < CUDART_INF_F;      // not an infinity, not a NaN
    float scale = __fmul_rn(top, 1.0f / largest<CODE>());
    float per = 0.f;
    if (!finite) scale = CUDART_NAN_F;
    else if (scale < 1.17549435e-38f) scale = 0.f;
    else per = __fmul_rn(largest<CODE>(), __frcp_rn(top));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int d = (i * lanes + w.lane) * V;
      if (d < p.head_dim) {
        Vec<uint8_t, V> c = {};
        if (finite) c = encode<T, CODE, V>(x[u][i], per);
        *reinterpret_cast<Vec<uint8_t, V>*>(codes + at * sl + d) = c;
      }
    }
    if (w.lane == 0) scales[at] = scale;
  }
}

template <typename T, int CODE, int V, int U>
__global__ void __launch_bounds__(NT, 12) read_kernel(const xkv_cache_params p, int lanes) {
  const int h = blockIdx.y, b = blockIdx.z >> 1;
  const Place w = place_of(p, lanes);
  const int t0 = blockIdx.x * (w.groups * U) + w.group;
  const uint8_t* codes = w.values ? static_cast<const uint8_t*>(p.v_codes) + b * p.vc_sb + h * p.vc_sh
                                  : static_cast<const uint8_t*>(p.k_codes) + b * p.kc_sb + h * p.kc_sh;
  const float* scales = w.values ? p.v_scales + b * p.vs_sb + h * p.vs_sh : p.k_scales + b * p.ks_sb + h * p.ks_sh;
  const int64_t sl = w.values ? p.vc_sl : p.kc_sl, st = w.values ? p.v_st : p.k_st;
  T* dst = w.values ? static_cast<T*>(p.v) + b * p.v_sb + h * p.v_sh : static_cast<T*>(p.k) + b * p.k_sb + h * p.k_sh;
  for (int d = w.lane * V; d < p.head_dim; d += lanes * V) {
    Vec<uint8_t, V> c[U];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * w.groups;
      const int64_t at = w.start + t;
      c[u] = {};
      scale[u] = 0.f;
      if (t < w.tokens && at >= 0 && at < p.capacity) {
        c[u] = *reinterpret_cast<const Vec<uint8_t, V>*>(codes + at * sl + d);
        scale[u] = scales[at];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * w.groups;
      if (t >= w.tokens) break;
      // outside the cache: zeros (code 0, scale 0)
      const Vec<T, V> x = decode<T, CODE, V>(c[u], scale[u]);
      *reinterpret_cast<Vec<T, V>*>(dst + t * st + d) = x;
    }
  }
}

bool aligned(const void* ptr, int64_t sb, int64_t sh, int64_t sl, int es, int vec) {
  return reinterpret_cast<uintptr_t>(ptr) % (size_t)(es * vec) == 0 && sb % vec == 0 && sh % vec == 0 && sl % vec == 0;
}
bool all_aligned(const xkv_cache_params& p, int es, int vec) {
  return p.head_dim % vec == 0 && aligned(p.k, p.k_sb, p.k_sh, p.k_st, es, vec) && aligned(p.v, p.v_sb, p.v_sh, p.v_st, es, vec) &&
         aligned(p.k_codes, p.kc_sb, p.kc_sh, p.kc_sl, 1, vec) && aligned(p.v_codes, p.vc_sb, p.vc_sh, p.vc_sl, 1, vec);
}
int lanes_for(int accesses) {      // per row
  int lanes = 1;
  while (lanes < 32 && lanes < accesses) lanes *= 2;
  return lanes;
}

// rows in flight per thread: four where there are tokens enough to keep every SM busy all the same
template <int U>
bool grid_of(const xkv_cache_params& p, int lanes, dim3* grid) {
  const int64_t chunks = ((int64_t)p.num_tokens + NT / lanes * U - 1) / (NT / lanes * U);
  if (p.num_tokens > 0x7fffffff - 4096 || p.num_kv_heads > 65535 || p.batch > 32767) return false;
  *grid = dim3((unsigned)chunks, (unsigned)p.num_kv_heads, (unsigned)(2*p.batch));
  return true;
}
bool many_tokens(const xkv_cache_params& p, int lanes) {
  return (int64_t)p.num_tokens * p.num_kv_heads * p.batch * 2 * lanes >= (int64_t)device_sm_count() * 2048 * 4;
}

template <typename T, int CODE, int V, int NV, int U>
int append_u(const xkv_cache_params& p, int lanes, cudaStream_t st) {
  dim3 grid;
  if (!grid_of<U>(p, lanes, &grid)) return XKV_ERR_UNSUPPORTED;
  append_kernel<T, CODE, V, NV, U><<<grid, NT, 0, st>>>(p, lanes);
  return cudaGetLastError() == cudaSuccess ? XKV_OK : XKV_ERR_LAUNCH;
}
template <typename T, int CODE, int V>
int append_v(const xkv_cache_params& p, cudaStream_t st) {
  const int accesses = ceil_div(p.head_dim, V), lanes = lanes_for(accesses), nv = ceil_div(accesses, lanes);
  if (nv == 1) return many_tokens(p, lanes) ? append_u<T, CODE, V, 1, 4>(p, lanes, st) : append_u<T, CODE, V, 1, 1>(p, lanes, st);
  if (nv <= 4) return append_u<T, CODE, V, 4, 1>(p, lanes, st);
  return append_u<T, CODE, V, 32, 1>(p, lanes, st);       // head_dim <= 1024 = 32 lanes x 32
}
template <typename T, int CODE, int V, int U>
int read_u(const xkv_cache_params& p, int lanes, cudaStream_t st) {
  dim3 grid;
  if (!grid_of<U>(p, lanes, &grid)) return XKV_ERR_UNSUPPORTED;
  read_kernel<T, CODE, V, U><<<grid, NT, 0, st>>>(p, lanes);
  return cudaGetLastError() == cudaSuccess ? XKV_OK : XKV_ERR_LAUNCH;
}
template <typename T, int CODE, int V>
int read_v(const xkv_cache_params& p, cudaStream_t st) {
  const int lanes = lanes_for(ceil_div(p.head_dim, V));
  return many_tokens(p, lanes) ? read_u<T, CODE, V, 4>(p, lanes, st) : read_u<T, CODE, V, 1>(p, lanes, st);
}

template <typename T, int CODE>
int run(const xkv_cache_params& p, bool write, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = all_aligned(p, sizeof(T), V);
  if (write) return wide ? append_v<T, CODE, V>(p, st) : append_v<T, CODE, 1>(p, st);
  return wide ? read_v<T, CODE, V>(p, st) : read_v<T, CODE, 1>(p, st);
}
template <typename T>
int by_code(const xkv_cache_params& p, bool write, cudaStream_t st) {
  return p.cache_code == XKV_CACHE_INT8 ? run<T, XKV_CACHE_INT8>(p, write, st) : run<T, XKV_CACHE_E4M3>(p, write, st);
}

}  // namespace

int launch_cache(const xkv_cache_params& p, bool write, cudaStream_t st) {
  switch (p.dtype) {
    case XKV_F32: return by_code<float>(p, write, st);
    case XKV_BF16: return by_code<__nv_bfloat16>(p, write, st);
    case XKV_F16: return by_code<__half>(p, write, st);
    default: return XKV_ERR_BAD_ARG;
  }
}

}  // namespace xkv
