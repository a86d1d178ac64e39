// xkv_tree_decode: kernel selection, the portable kernel (every type, head size and stride) and the merge of KV splits.
#include "tree_common.cuh"

namespace xkv {
namespace tree {
namespace {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// ---- portable kernel -------------------------------------------------------------------------------------------
// A block of 128 threads owns 16 query rows of one (KV split, KV head, sequence) and walks 32-token tiles held in shared
// memory as fp32.  Scores: lane = token, a warp has four rows (one 16-byte read of K feeds 16 multiply-adds).  Output:
// a thread owns the columns d, d + 128 of all 16 rows.  Everything is fp32 on the CUDA cores, which bounds it.
constexpr int NT = 128, RB = 16, TT = 32;

template <typename T, int CODE>
__device__ __forceinline__ float cache_value(const void* base, int64_t i, float scale) {
  if (CODE == XKV_CACHE_DENSE) return to_f(static_cast<const T*>(base)[i]);
  const uint8_t c = static_cast<const uint8_t*>(base)[i];
  if (CODE == XKV_CACHE_INT8) return (float)(int8_t)c * scale;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))) * scale;
}

__host__ __device__ inline int padded(int d) { return (d + 3) / 4 * 4 + 4; }   // row stride: 16-byte reads without conflicts

template <typename T, int CODE, int ND>     // ND: columns per thread
__global__ void __launch_bounds__(NT) portable_kernel(const Args a) {
  extern __shared__ __align__(16) float sm[];
  const xkv_tree_params& p = a.p;
  const int D = p.head_dim, DS = padded(D);
  float* qs = sm;                      // [RB][DS], scaled to the log2 domain
  float* ks = qs + RB * DS;            // [TT][DS]
  float* vs = ks + TT * DS;            // [TT][DS]
  float* ps = vs + TT * DS;            // [TT][RB]
  float* al = ps + TT * RB;            // [RB] factor on the output of a tile
  uint32_t* seen = reinterpret_cast<uint32_t*>(al + RB);   // [TT] rows that see the token
  const int blocks = (a.rows + RB - 1) / RB;
  int id = blockIdx.x;
  const int split = id % a.splits; id /= a.splits;
  const int rb = id % blocks; id /= blocks;
  const int h = id % p.num_kv_heads, b = id / p.num_kv_heads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int T_ = p.num_tokens, G = p.num_heads / p.num_kv_heads;
  const Span sp = span_of(p, b);
  const int tiles = (sp.len + TT - 1) / TT;
  if (blockIdx.x == 0 && tid < 8) a.status[tid] = 0;       // nothing here waits: the status is always good
  const int begin = (int)((int64_t)split * tiles / a.splits), end = (int)((int64_t)(split + 1) * tiles / a.splits);

  for (int i = tid; i < RB * DS; i += NT) {
    const int r = i / DS, d = i - r * DS, row = rb * RB + r;
    float v = 0.f;
    if (row < a.rows && d < D)
      v = to_f(static_cast<const T*>(p.q)[(int64_t)b * p.q_sb + (int64_t)(h * G + row / T_) * p.q_sh + (int64_t)(row % T_) * p.q_st + d]) *
          a.scale_log2;
    qs[i] = v;
  }
  float m[4], l[4], o[ND][RB];
#pragma unroll
  for (int i = 0; i < 4; ++i) { m[i] = -CUDART_INF_F; l[i] = 0.f; }
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int r = 0; r < RB; ++r) o[n][r] = 0.f;

  for (int tile = begin; tile < end; ++tile) {
    const int t0 = tile * TT;
    __syncthreads();
    for (int i = tid; i < TT * DS; i += NT) {
      const int t = i / DS, d = i - t * DS, at = t0 + t;
      float kv = 0.f, vv = 0.f;
      if (at < sp.len && d < D) {
        float sk = 1.f, sv = 1.f;
        if (CODE != XKV_CACHE_DENSE) {
          sk = p.k_scales[(int64_t)b * p.ks_sb + (int64_t)h * p.ks_sh + at];
          sv = p.v_scales[(int64_t)b * p.vs_sb + (int64_t)h * p.vs_sh + at];
        }
        kv = cache_value<T, CODE>(p.k, (int64_t)b * p.k_sb + (int64_t)h * p.k_sh + (int64_t)at * p.k_sl + d, sk);
        vv = cache_value<T, CODE>(p.v, (int64_t)b * p.v_sb + (int64_t)h * p.v_sh + (int64_t)at * p.v_sl + d, sv);
      }
      ks[i] = kv;
      vs[i] = vv;
    }
    if (tid < TT) seen[tid] = 0;
    __syncthreads();
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int d = 0; d < DS - 4; d += 4) {
      const float4 k4 = *reinterpret_cast<const float4*>(ks + lane * DS + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 q4 = *reinterpret_cast<const float4*>(qs + (warp * 4 + i) * DS + d);
        s[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[i]))));
      }
    }
    const int at = t0 + lane;
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = rb * RB + warp * 4 + i;
      const bool vis = at < sp.len && row < a.rows && sees(p, b, row % T_, at, sp.first);
      if (vis) mine |= 1u << (warp * 4 + i);
      const float x = vis ? s[i] : -CUDART_INF_F;
      float mx = x;
#pragma unroll
      for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float mn = fmaxf(m[i], mx);
      const float use = mn == -CUDART_INF_F ? 0.f : mn;
      const float alpha = exp2f(m[i] - use);
      const float w = exp2f(x - use);
      float sum = w;
#pragma unroll
      for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      l[i] = l[i] * alpha + sum;
      m[i] = mn;
      ps[lane * RB + warp * 4 + i] = w;
      if (lane == 0) al[warp * 4 + i] = alpha;
    }
    if (mine) atomicOr(&seen[lane], mine);
    __syncthreads();
    const int n_tok = min(TT, sp.len - t0);
    const bool drafted = t0 + TT > sp.first;      // rows may be hidden from some query rows
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int r = 0; r < RB; ++r) o[n][r] *= al[r];
    for (int t = 0; t < n_tok; ++t) {
      float w[RB];
#pragma unroll
      for (int r = 0; r < RB; r += 4) *reinterpret_cast<float4*>(w + r) = *reinterpret_cast<const float4*>(ps + t * RB + r);
      const uint32_t sb = drafted ? seen[t] : 0xffffu;
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        const int d = tid + n * NT;
        const float v = d < D ? vs[t * DS + d] : 0.f;
        if (sb == 0xffffu) {
#pragma unroll
          for (int r = 0; r < RB; ++r) o[n][r] = fmaf(w[r], v, o[n][r]);
        } else {          // 0 * NaN would reach rows that do not see the token
#pragma unroll
          for (int r = 0; r < RB; ++r)
            if (sb >> r & 1) o[n][r] = fmaf(w[r], v, o[n][r]);
        }
      }
    }
  }
  const int64_t row0 = (int64_t)(b * p.num_kv_heads + h) * a.rows;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int row = rb * RB + r;
    if (row < a.rows) {
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        const int d = tid + n * NT;
        if (d < D) a.part_o[((row0 + row) * a.splits + split) * D + d] = o[n][r];
      }
    }
  }
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = rb * RB + warp * 4 + i;
      if (row < a.rows) a.part_ml[(row0 + row) * a.splits + split] = make_float2(m[i], l[i]);
    }
  }
}

size_t portable_smem(int D) { return ((size_t)(RB + 2 * TT) * padded(D) + TT * RB + RB + TT) * sizeof(float); }

template <typename T, int CODE, int ND>
int portable_launch(const Args& a, cudaStream_t st) {
  auto kern = portable_kernel<T, CODE, ND>;
  const size_t smem = portable_smem(a.p.head_dim);
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    cudaGetLastError();
    return XKV_ERR_LAUNCH;
  }
  const int64_t grid = (int64_t)a.splits * ceil_div(a.rows, RB) * a.p.num_kv_heads * a.p.batch;
  if (grid > 0x7fffffff) return XKV_ERR_UNSUPPORTED;
  kern<<<(unsigned)grid, NT, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? XKV_OK : XKV_ERR_LAUNCH;
}
template <typename T>
int portable(const Args& a, cudaStream_t st) {
  const bool one = a.p.head_dim <= NT;
  switch (a.p.cache_code) {
    case XKV_CACHE_DENSE: return one ? portable_launch<T, XKV_CACHE_DENSE, 1>(a, st) : portable_launch<T, XKV_CACHE_DENSE, 2>(a, st);
    case XKV_CACHE_INT8: return one ? portable_launch<T, XKV_CACHE_INT8, 1>(a, st) : portable_launch<T, XKV_CACHE_INT8, 2>(a, st);
    default: return one ? portable_launch<T, XKV_CACHE_E4M3, 1>(a, st) : portable_launch<T, XKV_CACHE_E4M3, 2>(a, st);
  }
}

// ---- merge -----------------------------------------------------------------------------------------------------
// out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.  WARPS warps per row, each with every WARPS-th split; the partial
// sums are then added in warp order.  A row with l = 0 everywhere sees nothing and gives zeros; a NaN score has made
// its split's l a NaN and reaches the output.
template <typename T, int WARPS>
__global__ void __launch_bounds__(128) merge_kernel(const Args a) {
  constexpr int ROWS = 4 / WARPS;
  __shared__ float4 acc[WARPS > 1 ? WARPS : 1][64];
  __shared__ float tot[WARPS > 1 ? WARPS : 1];
  const xkv_tree_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.head_dim;
  const int64_t row = (int64_t)blockIdx.x * ROWS + warp / WARPS;
  const int part = warp % WARPS;
  const int64_t all = (int64_t)p.batch * p.num_kv_heads * a.rows;
  const bool live = row < all;
  asm volatile("griddepcontrol.wait;" ::: "memory");      // the splits' results
  const float2* ml = a.part_ml + (live ? row : 0) * a.splits;
  float M = -CUDART_INF_F;
  for (int s = lane; s < a.splits; s += 32) M = fmaxf(M, ml[s].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (M == -CUDART_INF_F) M = 0.f;
  const float* po = a.part_o + (live ? row : 0) * a.splits * D;
  const int64_t b = row / ((int64_t)p.num_kv_heads * a.rows), r = row - b * p.num_kv_heads * a.rows;
  T* out = static_cast<T*>(p.out) + b * p.o_sb + r * p.o_sr;
  const bool quads = D % 4 == 0;
  for (int d0 = 0; d0 < D; d0 += quads ? 128 : 32) {        // 4 columns per lane, or one
    const int d = d0 + (quads ? lane * 4 : lane);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    if (live)
      for (int s = part; s < a.splits; s += WARPS) {
        const float2 x = ml[s];
        const float w = exp2f(x.x - M);
        l = fmaf(w, x.y, l);
        if (d < D && quads) {
          const float4 y = *reinterpret_cast<const float4*>(po + (int64_t)s * D + d);
          o.x = fmaf(w, y.x, o.x); o.y = fmaf(w, y.y, o.y); o.z = fmaf(w, y.z, o.z); o.w = fmaf(w, y.w, o.w);
        } else if (d < D) {
          o.x = fmaf(w, po[(int64_t)s * D + d], o.x);
        }
      }
    if (WARPS > 1) {
      acc[part][lane] = o;
      if (lane == 0) tot[part] = l;
      __syncthreads();
      if (part == 0) {
#pragma unroll
        for (int i = 1; i < WARPS; ++i) {
          const float4 y = acc[i][lane];
          o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
          l += tot[i];
        }
      }
      __syncthreads();
    }
    if (live && part == 0 && d < D) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      out[d] = from_f<T>(o.x * inv);
      if (quads) {
        out[d + 1] = from_f<T>(o.y * inv);
        out[d + 2] = from_f<T>(o.z * inv);
        out[d + 3] = from_f<T>(o.w * inv);
      }
    }
  }
}

template <typename T>
int merge(const Args& a, cudaStream_t st) {
  const int64_t rows = (int64_t)a.p.batch * a.p.num_kv_heads * a.rows;
  const int64_t grid = a.splits >= 4 ? rows : (rows + 3) / 4;
  if (grid > 0x7fffffff) return XKV_ERR_UNSUPPORTED;
  // launched early: its blocks wait on the device for the kernel before it, not on the stream
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  const cudaError_t e = a.splits >= 4 ? cudaLaunchKernelEx(&cfg, merge_kernel<T, 4>, a) : cudaLaunchKernelEx(&cfg, merge_kernel<T, 1>, a);
  if (e != cudaSuccess) cudaGetLastError();
  return e == cudaSuccess ? XKV_OK : XKV_ERR_LAUNCH;
}

int validate(const xkv_tree_params* p) {
  if (!p) return XKV_ERR_BAD_ARG;
  if (p->dtype < XKV_F32 || p->dtype > XKV_F16) return XKV_ERR_BAD_ARG;
  if (p->cache_code < XKV_CACHE_DENSE || p->cache_code > XKV_CACHE_E4M3) return XKV_ERR_BAD_ARG;
  if (p->batch <= 0 || p->num_heads <= 0 || p->num_kv_heads <= 0 || p->num_tokens <= 0 || p->kv_len <= 0 || p->head_dim <= 0)
    return XKV_ERR_BAD_ARG;
  if (p->num_heads % p->num_kv_heads != 0 || p->num_splits < 0) return XKV_ERR_BAD_ARG;
  if (!p->q || !p->k || !p->v || !p->out) return XKV_ERR_BAD_ARG;
  if (p->cache_code != XKV_CACHE_DENSE && (!p->k_scales || !p->v_scales)) return XKV_ERR_BAD_ARG;
  if (p->head_dim > 256) return XKV_ERR_UNSUPPORTED;
  if ((int64_t)p->batch * p->num_heads * p->num_tokens > 0x7fffffff) return XKV_ERR_UNSUPPORTED;
  if (p->kv_len > 0x7fffffff - 4096) return XKV_ERR_UNSUPPORTED;      // token indices past the last tile stay 32-bit
  return XKV_OK;
}

void portable_plan(const xkv_tree_params& p, TreePlan* pl) {
  pl->kernel = TreePlan::kPortable;
  pl->name = "portable";
  const int64_t ctas = (int64_t)p.batch * p.num_kv_heads * ceil_div(pl->rows, RB);
  const int tiles = ceil_div(p.kv_len, TT);
  int64_t s = (4 * device_sm_count() + ctas - 1) / ctas;      // about four blocks per SM fit
  const int most = tiles > 4 ? tiles / 4 : 1;                 // at least 128 tokens per split
  if (s > most) s = most;
  if (s > 64) s = 64;
  pl->splits = s < 1 ? 1 : (int)s;
}

bool make_plan(const xkv_tree_params& p, TreePlan* pl) {
  pl->rows = p.num_heads / p.num_kv_heads * p.num_tokens;
  if (!(p.flags & XKV_FLAG_FORCE_GENERIC) && tree_stream_supported(p)) tree_stream_plan(p, pl);
  else portable_plan(p, pl);
  if (p.num_splits > 0) pl->splits = p.num_splits < 64 ? p.num_splits : 64;
  tree_layout(p, pl);
  return true;
}

}  // namespace
}  // namespace tree

void tree_layout(const xkv_tree_params& p, TreePlan* pl) {
  const size_t rows = (size_t)p.batch * p.num_kv_heads * pl->rows * pl->splits;
  size_t off = 256;
  pl->off_o = off;
  off += align_up(rows * p.head_dim * sizeof(float), 256);
  pl->off_ml = off;
  off += align_up(rows * sizeof(float2), 256);
  pl->total_bytes = off;
}

int tree_merge(const tree::Args& a, cudaStream_t st) {
  switch (a.p.dtype) {
    case XKV_F32: return tree::merge<float>(a, st);
    case XKV_BF16: return tree::merge<__nv_bfloat16>(a, st);
    default: return tree::merge<__half>(a, st);
  }
}

}  // namespace xkv

using namespace xkv;

extern "C" {

size_t xkv_tree_params_size(void) { return sizeof(xkv_tree_params); }

const char* xkv_tree_decode_plan(const xkv_tree_params* p) {
  TreePlan pl;
  if (tree::validate(p) != XKV_OK || !tree::make_plan(*p, &pl)) return nullptr;
  return pl.name;
}

size_t xkv_tree_decode_workspace_bytes(const xkv_tree_params* p) {
  TreePlan pl;
  if (tree::validate(p) != XKV_OK || !tree::make_plan(*p, &pl)) return 0;
  return pl.total_bytes;
}

int xkv_tree_decode(const xkv_tree_params* p, void* ws, size_t ws_bytes, void* stream) {
  const int rc = tree::validate(p);
  if (rc != XKV_OK) return rc;
  TreePlan pl;
  if (!tree::make_plan(*p, &pl)) return XKV_ERR_UNSUPPORTED;
  if (!ws || ws_bytes < pl.total_bytes) return XKV_ERR_WORKSPACE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* w = static_cast<char*>(ws);
  tree::Args a;
  a.p = *p;
  a.rows = pl.rows;
  a.splits = pl.splits;
  a.scale_log2 = p->sm_scale * 1.4426950408889634f;
  a.part_o = reinterpret_cast<float*>(w + pl.off_o);
  a.part_ml = reinterpret_cast<float2*>(w + pl.off_ml);
  a.status = reinterpret_cast<int*>(w);
  if (pl.kernel == TreePlan::kStream) return tree_stream_decode(a, st);
  int e;
  switch (p->dtype) {
    case XKV_F32: e = tree::portable<float>(a, st); break;
    case XKV_BF16: e = tree::portable<__nv_bfloat16>(a, st); break;
    default: e = tree::portable<__half>(a, st); break;
  }
  return e != XKV_OK ? e : tree_merge(a, st);
}

}  // extern "C"
