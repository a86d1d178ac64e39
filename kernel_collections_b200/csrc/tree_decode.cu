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
// A block of 128 threads takes strips of 16 query rows and walks 32-token tiles held in shared memory as fp32.  Scores: lane = token, a warp has four rows (one 16-byte read of K feeds 16 multiply-adds).  Output:
// a thread owns the columns d, d + 128 of all 16 rows.  Everything is fp32 on the CUDA cores, which bounds it.
constexpr int NT = 128, RB = 16, TT = 32, UNIT = 4 * TT;

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
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int T_ = p.num_tokens, G = p.num_heads / p.num_kv_heads;
  if (blockIdx.x == 0 && tid < 8) a.status[tid] = 0;       // nothing here waits: the status is always good
  Walk walk = walk_of(a, lane);
  Piece pc;
  while (next_piece(a, walk, pc)) {
    const int b = pc.b, h = pc.h, rb = pc.rb;
    const Span sp = span_of(p, b);
    const int begin = pc.begin * (UNIT / TT), end = min(pc.end * (UNIT / TT), (sp.len + TT - 1) / TT);
    __syncthreads();
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
    // the sums of all rows to shared memory, then rows out
    __syncthreads();
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<float2*>(ps)[warp * 4 + i] = make_float2(m[i], l[i]);
    }
    __syncthreads();
    const float2* ml = reinterpret_cast<const float2*>(ps);
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int row = rb * RB + r;
      if (row < a.rows) {
        const float inv = ml[r].y == 0.f ? 0.f : 1.f / ml[r].y;
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const int d = tid + n * NT;
          if (d >= D) continue;
          if (pc.whole) static_cast<T*>(p.out)[(int64_t)b * p.o_sb + ((int64_t)h * a.rows + row) * p.o_sr + d] = from_f<T>(o[n][r] * inv);
          else a.part_o[(pc.id * RB + r) * D + d] = o[n][r];
        }
      }
    }
    if (!pc.whole && tid < RB) a.part_ml[pc.id * RB + tid] = ml[tid];
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
  kern<<<(unsigned)a.grid, NT, smem, st>>>(a);
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
// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over a strip's pieces.  WARPS warps per row, each with every
// WARPS-th piece; their sums are then added in warp order.  A row with l = 0 everywhere sees nothing and gives zeros; a
// NaN score has made its piece's l a NaN and reaches the output.
constexpr int MERGE_AHEAD = 4;      // pieces whose loads are in flight together

template <typename T, int WARPS>
__global__ void __launch_bounds__(128) merge_kernel(const Args a) {
  constexpr int ROWS = 4 / WARPS;
  __shared__ float4 acc[WARPS > 1 ? WARPS : 1][32];
  __shared__ float tot[WARPS > 1 ? WARPS : 1];
  const xkv_tree_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.head_dim;
  const int64_t row = (int64_t)blockIdx.x * ROWS + warp / WARPS;
  const int part = warp % WARPS;
  const int per_b = p.num_kv_heads * a.rows;
  const int b = (int)(row / per_b);
  if (b >= p.batch) {
    asm volatile("griddepcontrol.wait;" ::: "memory");    // no block ends before the kernel that it was launched early after
    return;
  }
  const int hr = (int)(row - (int64_t)b * per_b), h = hr / a.rows, r = hr - h * a.rows;
  // the strip's stretch of the line and the blocks that share it (kv_lens is the caller's, not the kernel's before)
  const Line line = line_of(a, lane);
  const Spot at = find_sequence(a, b, lane);
  const int64_t strip = (int64_t)h * a.blocks + r / a.block_rows;
  const int64_t begin = at.before + strip * at.units;
  const int first = (int)(begin / line.share), last = (int)((begin + at.units - 1) / line.share);
  asm volatile("griddepcontrol.wait;" ::: "memory");      // the pieces
  if (first == last) return;                              // one piece: its block has written the row
  const int n = last - first + 1, rr = r % a.block_rows;
  // row of piece i among the partial results: the strip begins in block `first` (its second place)
  auto place = [&](int i) { return (2 * (int64_t)(first + i) + (i == 0)) * a.block_rows + rr; };
  float M = -CUDART_INF_F;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, a.part_ml[place(i)].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (M == -CUDART_INF_F) M = 0.f;
  T* out = static_cast<T*>(p.out) + (int64_t)b * p.o_sb + (int64_t)hr * p.o_sr;
  const bool quads = D % 4 == 0;
  for (int d0 = 0; d0 < D; d0 += quads ? 128 : 32) {        // 4 columns per lane, or one
    const int d = d0 + (quads ? lane * 4 : lane);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int i0 = part; i0 < n; i0 += WARPS * MERGE_AHEAD) {
      float2 x[MERGE_AHEAD];
      float4 y[MERGE_AHEAD];
#pragma unroll
      for (int k = 0; k < MERGE_AHEAD; ++k) {
        const int i = i0 + k * WARPS;
        x[k] = make_float2(-CUDART_INF_F, 0.f);
        y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < n) {
          const int64_t at = place(i);
          x[k] = a.part_ml[at];
          if (d < D && quads) y[k] = *reinterpret_cast<const float4*>(a.part_o + at * D + d);
          else if (d < D) y[k].x = a.part_o[at * D + d];
        }
      }
#pragma unroll
      for (int k = 0; k < MERGE_AHEAD; ++k) {
        const float w = exp2f(x[k].x - M);
        l = fmaf(w, x[k].y, l);
        o.x = fmaf(w, y[k].x, o.x); o.y = fmaf(w, y[k].y, o.y); o.z = fmaf(w, y[k].z, o.z); o.w = fmaf(w, y[k].w, o.w);
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
    if (part == 0 && d < D) {
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
  // four warps per row where a strip has eight pieces or more on average
  const bool many = a.grid >= (int64_t)8 * a.p.batch * a.p.num_kv_heads * a.blocks;
  const int64_t grid = many ? rows : (rows + 3) / 4;
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
  const cudaError_t e = many ? cudaLaunchKernelEx(&cfg, merge_kernel<T, 4>, a) : cudaLaunchKernelEx(&cfg, merge_kernel<T, 1>, a);
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
  pl->block_rows = RB;
  pl->unit_tokens = UNIT;
  // Four blocks fit an SM over dense caches at head sizes up to 128 (119 registers a thread), three over 8-bit ones (151), two
  // near head size 256 (86 KB of shared memory): there the last shares run behind the others.
  pl->slots = 4 * device_sm_count();
}

bool make_plan(const xkv_tree_params& p, TreePlan* pl) {
  pl->rows = p.num_heads / p.num_kv_heads * p.num_tokens;
  if (!(p.flags & XKV_FLAG_FORCE_GENERIC) && tree_stream_supported(p)) {
    if (tree_tc_supported(p, pl->rows)) tree_tc_plan(p, pl);
    else tree_stream_plan(p, pl);
  } else {
    portable_plan(p, pl);
  }
  pl->blocks = ceil_div(pl->rows, pl->block_rows);
  const int64_t strips = (int64_t)p.batch * p.num_kv_heads * pl->blocks;
  if (strips > 0x7fffffff / 2) return false;
  const int units = ceil_div(p.kv_len, pl->unit_tokens);
  // as many blocks as run at once, never more than there are units (each block has at least one then)
  int64_t grid = p.num_splits > 0 ? strips * (p.num_splits < 64 ? p.num_splits : 64) : pl->slots;
  if (grid > strips * units) grid = strips * units;
  if (grid > 0x3fffffff) return false;
  pl->grid = (int)grid;
  pl->merged = units > 1;
  size_t off = XKV_STATUS_BYTES;
  const size_t rows = pl->merged ? (size_t)(2 * grid) * pl->block_rows : 0;
  pl->off_o = off;
  off += align_up(rows * p.head_dim * sizeof(float), 256);
  pl->off_ml = off;
  off += align_up(rows * sizeof(float2), 256);
  pl->total_bytes = off;
  return true;
}

}  // namespace
}  // namespace tree

int tree_merge(const tree::Args& a, cudaStream_t st) {
  switch (a.p.dtype) {
    case XKV_F32: return tree::merge<float>(a, st);
    case XKV_BF16: return tree::merge<__nv_bfloat16>(a, st);
    default: return tree::merge<__half>(a, st);
  }
}

}  // namespace xkv

using namespace xkv;

static __device__ __align__(256) unsigned char g_status_scratch[XKV_STATUS_BYTES];

extern "C" {

void* xkv_tree_status_scratch(void) {
  void* sym = nullptr;
  if (cudaGetSymbolAddress(&sym, g_status_scratch) == cudaSuccess) return sym;
  cudaGetLastError();
  return nullptr;
}

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
  a.block_rows = pl.block_rows;
  a.blocks = pl.blocks;
  a.unit_tokens = pl.unit_tokens;
  a.grid = pl.grid;
  a.scale_log2 = p->sm_scale * 1.4426950408889634f;
  a.part_o = reinterpret_cast<float*>(w + pl.off_o);
  a.part_ml = reinterpret_cast<float2*>(w + pl.off_ml);
  a.status = reinterpret_cast<int*>(w);
  int e;
  if (pl.kernel == TreePlan::kTc) e = tree_tc_decode(a, st);
  else if (pl.kernel == TreePlan::kStream) e = tree_stream_decode(a, st);
  else if (p->dtype == XKV_F32) e = tree::portable<float>(a, st);
  else if (p->dtype == XKV_BF16) e = tree::portable<__nv_bfloat16>(a, st);
  else e = tree::portable<__half>(a, st);
  return e != XKV_OK || !pl.merged ? e : tree_merge(a, st);
}

}  // extern "C"
