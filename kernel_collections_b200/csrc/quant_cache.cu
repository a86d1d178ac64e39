// Writing rows to an 8-bit key / value cache and reading them back.
//
// One row (token, KV head) is reduced to its largest magnitude, scaled and rounded: scale = top * (1 / C), code =
// rn(x * (C * (1 / top))), every operation rounded to fp32.  Both directions move every byte once and are bound by HBM for long stretches and by the launch for single
// tokens.  A row is held in registers by a power-of-two group of lanes (16 bytes per lane and access), so the
// reduction is a few shuffles and nothing is read twice; keys and values are the two halves of the grid.
#include "xkv_internal.h"
#include <cuda_fp8.h>
#include <math_constants.h>

namespace xkv {
namespace {

constexpr int NT = 256;

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

// y is within +-C (1 + 2^-22): a reciprocal and two products, each rounded once
template <int CODE> __device__ __forceinline__ uint8_t encode(float y) {
  if (CODE == XKV_CACHE_INT8) return (uint8_t)(int8_t)__float2int_rn(fminf(fmaxf(y, -127.f), 127.f));
  return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}
template <int CODE> __device__ __forceinline__ float decode(uint8_t c) {
  if (CODE == XKV_CACHE_INT8) return (float)(int8_t)c;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

struct Row {
  int b, h, t;
  int64_t at;      // cache row
};
__device__ __forceinline__ Row row_of(const xkv_cache_params& p, int64_t r) {
  Row w;
  const int64_t bh = r / p.num_tokens;
  w.t = (int)(r - bh * p.num_tokens);
  w.b = (int)(bh / p.num_kv_heads);
  w.h = (int)(bh - (int64_t)w.b * p.num_kv_heads);
  w.at = (int64_t)(p.positions ? p.positions[w.b] : p.position) + w.t;
  return w;
}

// NV accesses of V elements per lane; `lanes` (a power of two, at most 32) lanes hold one row.
template <typename T, int CODE, int V, int NV>
__global__ void __launch_bounds__(NT) append_kernel(const xkv_cache_params p, int64_t rows, int lanes) {
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t r = (int64_t)blockIdx.x * (NT / lanes) + threadIdx.x / lanes;
  const bool values = blockIdx.y != 0;
  Row w = {0, 0, 0, -1};
  bool live = r < rows;
  if (live) {
    w = row_of(p, r);
    live = w.at >= 0 && w.at < p.capacity && (!p.lengths || w.t < p.lengths[w.b]);
  }
  const T* src = static_cast<const T*>(values ? p.v : p.k) +
                 (values ? w.b * p.v_sb + w.h * p.v_sh + w.t * p.v_st : w.b * p.k_sb + w.h * p.k_sh + w.t * p.k_st);
  Vec<T, V> x[NV];
  float top = 0.f;
  bool odd = false;       // an infinity or a NaN
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int d = (i * lanes + lane) * V;
    if (live && d < p.head_dim) {
      x[i] = *reinterpret_cast<const Vec<T, V>*>(src + d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float m = fabsf(to_f(x[i].x[e]));
        odd |= !(m <= 3.402823466e38f);
        top = fmaxf(top, m);
      }
    }
  }
  if (odd) top = CUDART_INF_F;       // fmaxf passes a NaN over, an infinity survives it
  for (int o = lanes >> 1; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (!live) return;
  const bool finite = top < CUDART_INF_F;
  float scale = __fmul_rn(top, 1.0f / largest<CODE>());
  float per = 0.f;
  if (!finite) scale = CUDART_NAN_F;
  else if (scale < 1.17549435e-38f) scale = 0.f;
  else per = __fmul_rn(largest<CODE>(), __frcp_rn(top));
  uint8_t* dst = static_cast<uint8_t*>(values ? p.v_codes : p.k_codes) +
                 (values ? w.b * p.vc_sb + w.h * p.vc_sh + w.at * p.vc_sl : w.b * p.kc_sb + w.h * p.kc_sh + w.at * p.kc_sl);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int d = (i * lanes + lane) * V;
    if (d < p.head_dim) {
      Vec<uint8_t, V> c;
#pragma unroll
      for (int e = 0; e < V; ++e) c.x[e] = finite ? encode<CODE>(to_f(x[i].x[e]) * per) : 0;
      *reinterpret_cast<Vec<uint8_t, V>*>(dst + d) = c;
    }
  }
  if (lane == 0) {
    if (values) p.v_scales[w.b * p.vs_sb + w.h * p.vs_sh + w.at] = scale;
    else p.k_scales[w.b * p.ks_sb + w.h * p.ks_sh + w.at] = scale;
  }
}

template <typename T, int CODE, int V>
__global__ void __launch_bounds__(NT) read_kernel(const xkv_cache_params p, int64_t rows, int lanes) {
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t r = (int64_t)blockIdx.x * (NT / lanes) + threadIdx.x / lanes;
  if (r >= rows) return;
  const bool values = blockIdx.y != 0;
  const Row w = row_of(p, r);
  const bool live = w.at >= 0 && w.at < p.capacity;
  const int64_t at = live ? w.at : 0;
  const uint8_t* src = static_cast<const uint8_t*>(values ? p.v_codes : p.k_codes) +
                       (values ? w.b * p.vc_sb + w.h * p.vc_sh + at * p.vc_sl : w.b * p.kc_sb + w.h * p.kc_sh + at * p.kc_sl);
  const float scale = !live ? 0.f : values ? p.v_scales[w.b * p.vs_sb + w.h * p.vs_sh + at]
                                           : p.k_scales[w.b * p.ks_sb + w.h * p.ks_sh + at];
  T* dst = static_cast<T*>(values ? p.v : p.k) +
           (values ? w.b * p.v_sb + w.h * p.v_sh + w.t * p.v_st : w.b * p.k_sb + w.h * p.k_sh + w.t * p.k_st);
  for (int d = lane * V; d < p.head_dim; d += lanes * V) {
    Vec<uint8_t, V> c = {};
    if (live) c = *reinterpret_cast<const Vec<uint8_t, V>*>(src + d);
    Vec<T, V> x;
#pragma unroll
    for (int e = 0; e < V; ++e) x.x[e] = live ? from_f<T>(decode<CODE>(c.x[e]) * scale) : from_f<T>(0.f);
    *reinterpret_cast<Vec<T, V>*>(dst + d) = x;
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

template <typename T, int CODE, int V>
int append_v(const xkv_cache_params& p, cudaStream_t st) {
  const int64_t rows = (int64_t)p.batch * p.num_kv_heads * p.num_tokens;
  const int accesses = ceil_div(p.head_dim, V), lanes = lanes_for(accesses), nv = ceil_div(accesses, lanes);
  const int64_t gx = (rows + NT / lanes - 1) / (NT / lanes);
  if (gx > 0x7fffffff) return XKV_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)gx, 2);
  if (nv == 1) append_kernel<T, CODE, V, 1><<<grid, NT, 0, st>>>(p, rows, lanes);
  else if (nv <= 4) append_kernel<T, CODE, V, 4><<<grid, NT, 0, st>>>(p, rows, lanes);
  else append_kernel<T, CODE, V, 32><<<grid, NT, 0, st>>>(p, rows, lanes);   // head_dim <= 1024 = 32 lanes x 32
  return cudaGetLastError() == cudaSuccess ? XKV_OK : XKV_ERR_LAUNCH;
}
template <typename T, int CODE, int V>
int read_v(const xkv_cache_params& p, cudaStream_t st) {
  const int64_t rows = (int64_t)p.batch * p.num_kv_heads * p.num_tokens;
  const int lanes = lanes_for(ceil_div(p.head_dim, V));
  const int64_t gx = (rows + NT / lanes - 1) / (NT / lanes);
  if (gx > 0x7fffffff) return XKV_ERR_UNSUPPORTED;
  read_kernel<T, CODE, V><<<dim3((unsigned)gx, 2), NT, 0, st>>>(p, rows, lanes);
  return cudaGetLastError() == cudaSuccess ? XKV_OK : XKV_ERR_LAUNCH;
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
