// Tree attention for many query rows (drafted tokens x heads of a KV head) on tcgen05.
//
// With R query rows every cache element takes part in 2 R multiply-adds per product: from some 30 rows on that is too
// much for mma.sync next to HBM, and from about 250 rows the tensor cores themselves are the bound.  A block works on
// strips of MB x 128 query rows (MB = 1 up to 128 rows, else 2) in 128-token tiles; S and O live in tensor memory:
//   S = Q . K^T   A = Q (shared memory, resident for the strip), B = the K tile (K-major)
//   O += P . V    A = P (tensor memory, written by the softmax threads over the S it came from), B = the V tile (MN-major)
// Two groups of four softmax warps, one thread per query row, alternate: while one turns its S into P, the tensor core
// multiplies for the other.  MB = 2: the groups own one half of the rows each and share the tiles.  MB = 1: they own the
// same rows and take alternate tiles, each with its own O; the two are joined at the end.  An "item" is one tile for one
// group; S of item j + 2 is issued right after P.V of item j, into the same columns (MMAs run in order).
//   warps 0-7  softmax          warp 8  MMA issuer (one thread) and tensor-memory allocation
//   16-bit caches: warp 9 brings tiles by TMA.  8-bit caches: warps 12-19 load codes into registers one tile ahead, widen
//   them to fp16 (exact) and store them in the layout that TMA would have made; scales go to the softmax threads.
// The softmax takes one pass over S as long as no row's reference has to move (lazily, see SLACK below): weights are
// taken against the old reference while the new maximum is formed, kept in registers, and taken again in the rare tile that
// moves a reference or holds drafted tokens.  Number ranges (query scaling, LIFT, products with the value scales) are those of
// tree_stream_sm100.cu.  P is rounded to the 16-bit type of the product; over 16-bit caches l
// sums the rounded values.
// What bounds it.  Per 128 x 128 item the tensor core needs 1024 cycles and the exponentials 1024 of the 16-per-clock unit; a
// group's chain (softmax 1800, then P.V and S with their latencies 1400) leaves about 2000 per item over 16-bit caches.  Over
// 8-bit caches it was 3800 when counted: every element takes a key and a value scale from shared memory more, and the softmax
// does not fit its 144 registers (144 to 284 bytes stored and 396 to 676 loaded per thread as spills; the 16-bit kernels 0 to 16).  What
// each of the two costs was not separated.  512 fp16 rows over 4 x 32768 rows of 8 heads, calls queued: 16-bit cache 300 us
// (916 TFLOP/s), int8 440 to 457 (600 to 625), e4m3 490 to 494.  104 rows over 8 x 16384 ragged rows: bf16 95 to 105 us, steady tiles at the
// rate of HBM, the rest set-up and ends of the strips; int8 158 to 160, e4m3 179 to 182 (the scales come with V: the softmax
// of a tile waits for a widening of V that it does not need yet).  Handing the exponentials from one group to the other in strict turns was
// measured slower (536 us against 474).
// All waits are bounded; a group that gives up raises the abort flag, which ends the others' waits.
#include "tree_common.cuh"
#include "sm100_common.cuh"
#include <type_traits>

namespace xkv {
namespace tree {
using namespace sm100;
namespace {

constexpr int TK = 128;                     // tokens per tile
constexpr int STAGES = 2;                   // of K and of V each
constexpr int BOX = TK * 128;               // bytes of [128 tokens or rows] x 64 dims
constexpr int MAX_T = 256;                  // drafted tokens whose mask fits its place

// 16-bit caches: three warps per scheduler, 168 registers each.  8-bit: five, 96 at launch, moved from the issuer's and the
// wideners' warpgroups to the softmax (2 x 144 + 3 x 64 = 5 x 96).
constexpr int WIDENERS = 8;                 // warps
template <int CODE> constexpr int threads() { return CODE == XKV_CACHE_DENSE ? 320 : 640; }

template <int D, int MB>
struct Smem {
  static constexpr int HALVES = D / 64;
  static constexpr int TILE = HALVES * BOX;                     // K or V tile; also 128 query rows
  static constexpr int Q = 0;                                   // two row blocks (the second also takes part in the join)
  static constexpr int K = Q + 2 * TILE;
  static constexpr int V = K + STAGES * TILE;
  static constexpr int SCALES = V + STAGES * TILE;              // [stage]{key scales, value scales, log2 of these}[128]
  static constexpr int MASK = SCALES + STAGES * 3 * TK * 4;   // [token][words]
  static constexpr int BAD = MASK + MAX_T * (MAX_T / 32) * 4;   // drafted tokens with values that are not finite
  static constexpr int ML = BAD + MAX_T / 32 * 4;               // [128] of the second group, MB == 1
  static constexpr int SCALE = ML + TK * 8;                     // [row] of the strip: factor on its scores
  static constexpr int BAR = SCALE + 2 * TK * 4;
  static constexpr int MISC = BAR + 16 * 8;
  static constexpr int BYTES = MISC + 16 + 1024;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
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
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
template <typename T> __device__ __forceinline__ float to_float(T v) { return TypeTraits<T>::to_f(v); }
template <typename T> __device__ __forceinline__ T from_float(float v) { return TypeTraits<T>::from_f(v); }

// one lane of the warp, the same one every time
__device__ __forceinline__ bool elect() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

// bytes 0, 1 of x (high = 0) or 2, 3 as two halves; int8 with its sign bits flipped beforehand
template <int CODE> __device__ __forceinline__ uint32_t widen(uint32_t x, int high) {
  if (CODE == XKV_CACHE_INT8) {
    const uint32_t y = __byte_perm(x, 0x64646464u, high ? 0x4342u : 0x4140u);      // {code + 128, 0x64} twice: halves 1152 + code
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&y), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  uint32_t r;
  const uint16_t two = (uint16_t)(high ? x >> 16 : x);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
  return r;
}

template <typename T, int CODE, int D, int MB>
__global__ void __launch_bounds__(threads<CODE>(), 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
  constexpr bool Q8 = CODE != XKV_CACHE_DENSE;
  using M = typename std::conditional<Q8, __half, T>::type;
  using S = Smem<D, MB>;
  constexpr bool CLEANS = CODE != XKV_CACHE_INT8;      // values may be infinite (16-bit) or NaN (16-bit, e4m3 codes 0x7f and 0xff)
  // weights are 2^(score - reference + LIFT); the reference follows the maximum when it is passed by more than SLACK
  // (fp16: below 2^15 always, and all 11 bits down to 2^-20 of the reference; bf16 has the range of fp32, and stays below 2^8
  // so that products with large values do)
  constexpr float LIFT = std::is_same<M, __half>::value ? 6.f : -12.f, SLACK = std::is_same<M, __half>::value ? 9.f : 20.f;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const xkv_tree_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int T_ = p.num_tokens, G = p.num_heads / p.num_kv_heads;

  const uint32_t bar0 = base + S::BAR;
  auto bar_kfull = [&](int s) { return bar0 + 8u * s; };
  auto bar_kempty = [&](int s) { return bar0 + 8u * (2 + s); };
  auto bar_vfull = [&](int s) { return bar0 + 8u * (4 + s); };
  auto bar_vempty = [&](int s) { return bar0 + 8u * (6 + s); };
  auto bar_s = [&](int w) { return bar0 + 8u * (8 + w); };          // S of the group's next item is there
  auto bar_p = [&](int w) { return bar0 + 8u * (10 + w); };         // its P is
  const uint32_t bar_q = bar0 + 8u * 12;                            // queries and mask of the strip are in place, the issuer is there
  const uint32_t bar_end = bar0 + 8u * 13;                          // softmax threads meet
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(sm + S::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + S::MISC + 4);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_kfull(s), Q8 ? WIDENERS : 1);        // one arrival per warp
      mbar_init(bar_vfull(s), Q8 ? WIDENERS : 1);
      mbar_init(bar_kempty(s), 1);
      mbar_init(bar_vempty(s), 1);
    }
    for (int w = 0; w < 2; ++w) { mbar_init(bar_s(w), 1); mbar_init(bar_p(w), 4); }
    mbar_init(bar_q, 9);                   // the softmax warps and the issuer
    mbar_init(bar_end, 8);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + S::MISC), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);        // columns: S / P of the groups at 0 and 128, O at 256 and 384
  asm volatile("griddepcontrol.launch_dependents;");
  if (blockIdx.x == 0 && threadIdx.x < 8) a.status[threadIdx.x] = 0;      // a wait takes far longer than this to give up

  Walk walk = walk_of(a, lane);
  Piece pc = {};
  auto tiles_of = [&](const Piece& x, int len) { return max(0, min(x.end, (len + TK - 1) / TK) - x.begin); };

  if constexpr (Q8) {                       // whole warpgroups: 0 1 | 2 (the issuer's) 3 4 (the wideners')
    if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  }
  if (warp < 8) {
    // ================================ softmax ================================================================
    const int w = warp >> 2, r = threadIdx.x & 127;         // group; row of its 128 = tensor-memory lane
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + (uint32_t)w * 128u, t_o = tmem + lanes + 256u + (uint32_t)w * 128u;
    const int words = (T_ + 31) / 32;
    uint32_t* mask_s = reinterpret_cast<uint32_t*>(sm + S::MASK);
    uint32_t* bad_s = reinterpret_cast<uint32_t*>(sm + S::BAD);
    float2* ml_s = reinterpret_cast<float2*>(sm + S::ML);
    float* scale_s = reinterpret_cast<float*>(sm + S::SCALE);
    float* join_s = reinterpret_cast<float*>(sm + S::Q);    // [dim][row] of the second group, MB == 1
    uint32_t q_phase = 0, end_phase = 0, s_phase = 0;
    int tiles_seen = 0;                                     // of the pieces before
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity, int role) {
      if (__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag))) return true;
      if (lane == 0) report(a.status, XKV_ERR_TIMEOUT, role, pc.b, pc.h, pc.begin);
      return false;
    };
    auto arrive = [&](uint32_t bar) {       // for the warp, once all its lanes are there
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto meet = [&]() {
      arrive(bar_end);
      const bool good = wait(bar_end, end_phase, 53);
      end_phase ^= 1u;
      return good;
    };
    while (ok && next_piece(a, walk, pc)) {
      const Span sp = span_of(p, pc.b);
      const int ntiles = tiles_of(pc, sp.len);
      // ---- queries of this strip, in the layout of a K-major operand; mask rows as bits ------------------------
      const int blk = MB == 2 ? w : 0;
      const int row = pc.rb * (MB * 128) + blk * 128 + r;
      const bool live = row < a.rows;
      const int tok = live ? row % T_ : 0;
      const bool busy = (pc.rb * MB + blk) * 128 + (warp & 3) * 32 < a.rows;      // some row of this warp is one
      float row_scale = 1.f;
      {
        // a warp takes its rows one after the other, so that the reads are contiguous; MB == 1: the groups hold the same
        // rows and take half of them each
        constexpr int PER = D / 32, AHEAD = 16;
        const bool wide = reinterpret_cast<uintptr_t>(p.q) % (PER * 2) == 0 && p.q_sb % PER == 0 && p.q_sh % PER == 0 && p.q_st % PER == 0;
        using Few = typename std::conditional<PER == 4, uint2, uint32_t>::type;       // a lane's PER elements
        const int first_row = (pc.rb * MB + blk) * 128 + (warp & 3) * 32, from_row = first_row + (MB == 1 ? w * 16 : 0);
        int qh = from_row / T_, qt = from_row - qh * T_;
        const int64_t next_head = p.q_sh - (T_ - 1) * p.q_st;   // from a head's last token to the next head's first
        const T* src = static_cast<const T*>(p.q) + (int64_t)pc.b * p.q_sb + (int64_t)(pc.h * G + qh) * p.q_sh + (int64_t)qt * p.q_st + lane * PER;
        for (int i0 = MB == 1 ? w * 16 : 0; i0 < (MB == 1 ? w * 16 + 16 : 32) && busy; i0 += AHEAD) {
          Few q[AHEAD] = {};
          auto rows = [&](auto read) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
              if (first_row + i0 + i < a.rows) q[i] = read(src);
              const bool last = ++qt == T_;
              qt = last ? 0 : qt;
              src += last ? next_head : p.q_st;
            }
          };
          if (wide) {
            rows([](const T* s) { return *reinterpret_cast<const Few*>(s); });
          } else {
            rows([](const T* s) {
              Few f;
              T* x = reinterpret_cast<T*>(&f);
#pragma unroll
              for (int e = 0; e < PER; ++e) x[e] = s[e];
              return f;
            });
          }
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {
            float2 x[PER / 2];
#pragma unroll
            for (int e = 0; e < PER / 2; ++e) x[e] = TypeTraits<T>::unpack2(reinterpret_cast<const uint32_t*>(&q[i])[e]);
            // the sign of the scale goes to the queries, so that the largest product is the largest score; a scale of zero too
            float up = a.scale_log2 < 0.f ? -1.f : 1.f, scale = fmaxf(fabsf(a.scale_log2), 1.17549435e-38f);
            if (a.scale_log2 == 0.f) {
              up = 0.f;
              scale = 1.f;
            } else if (Q8) {
              float top = 0.f;
#pragma unroll
              for (int e = 0; e < PER / 2; ++e) top = fmaxf(top, fmaxf(fabsf(x[e].x), fabsf(x[e].y)));
              top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
              if (top > 0.f && top < CUDART_INF_F) {
                const int e = min(max(14 - (int)(((__float_as_uint(top) >> 23) & 255u)) + 127, -120), 120);
                up *= __uint_as_float((uint32_t)(e + 127) << 23);
                scale = fmaxf(scale * __uint_as_float((uint32_t)(127 - e) << 23), 1.17549435e-38f);
              }
            }
            const int rr = (warp & 3) * 32 + i0 + i, d = lane * PER;
            uint32_t* to = reinterpret_cast<uint32_t*>(sm + S::Q + blk * S::TILE + (d >> 6) * BOX + rr * 128 +
                                                       ((((d & 63) >> 3) ^ (rr & 7)) << 4) + (d & 7) * 2);
#pragma unroll
            for (int e = 0; e < PER / 2; ++e) to[e] = TypeTraits<M>::pack2(x[e].x * up, x[e].y * up);
            if (lane == 0) scale_s[blk * 128 + rr] = scale;
          }
        }
        if ((pc.begin + ntiles) * TK > sp.first) {            // drafted tokens in this piece
#pragma unroll 8
          for (int i = warp; i < T_ * words; i += 8) {
            const int t = i / words, u = (i - t * words) * 32 + lane;
            const bool see = u < T_ && (p.tree_mask ? p.tree_mask[(int64_t)pc.b * p.tm_sb + (int64_t)t * p.tm_st + u] != 0 : u <= t);
            const uint32_t bits = __ballot_sync(0xffffffffu, see);
            if (lane == 0) mask_s[i] = bits;
          }
        }
        if (threadIdx.x < MAX_T / 32) bad_s[threadIdx.x] = 0;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        arrive(bar_q);
        if (!(ok = wait(bar_q, q_phase, 50))) break;
        q_phase ^= 1u;
        if (busy) row_scale = scale_s[blk * 128 + r];
      }
      float ref = -CUDART_INF_F;                             // of the scores; over 8-bit caches of score + log2 |value scale|
      float2 l = make_float2(0.f, 0.f);
      int items = 0;
      for (int i = MB == 2 ? 0 : w; i < ntiles; i += MB == 2 ? 1 : 2, ++items) {
        const int t0 = (pc.begin + i) * TK;
        const int stage = (tiles_seen + i) % STAGES;
        const uint32_t v_parity = (uint32_t)((tiles_seen + i) / STAGES) & 1u;
        const float* ks = reinterpret_cast<const float*>(sm + S::SCALES + stage * 3 * TK * 4);
        const float* vs = ks + TK;
        if (Q8 && !(ok = wait(bar_vfull(stage), v_parity, 51))) break;       // the scales come with the values
        if (!(ok = wait(bar_s(w), s_phase, 52))) break;
        s_phase ^= 1u;
        tc_fence_after();
        const bool plain = t0 + TK <= sp.first;
        // tokens c .. c + 31 of the tile that this row sees: all in front of the drafted ones, then by the mask's bits
        auto seen = [&](int c) -> uint32_t {
          const int u0 = t0 + c - sp.first, k = u0 >> 5;          // drafted token of the first one
          auto word = [&](int i) { return i < 0 ? 0xffffffffu : i < words ? mask_s[tok * words + i] : 0u; };
          return __funnelshift_r(word(k), word(k + 1), u0 & 31);
        };
        if (busy) {
          const float2 rs2 = make_float2(row_scale, row_scale);
          // columns c .. c + 31 as scores (without row_scale)
          auto scores = [&](int c, float2 (&x)[16]) {
            uint32_t v[32];
            tmem_ld32(t_s + c, v);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              x[k] = make_float2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1]));
              x[k + 1] = make_float2(__uint_as_float(v[2 * k + 2]), __uint_as_float(v[2 * k + 3]));
              if (Q8) {
                const float4 f = *reinterpret_cast<const float4*>(ks + c + 2 * k);
                x[k] = mul2(x[k], make_float2(f.x, f.y));
                x[k + 1] = mul2(x[k + 1], make_float2(f.z, f.w));
              }
            }
          };
          float b1;                                           // weights are 2^(score + b1)
          auto settle = [&]() { b1 = ref == -CUDART_INF_F ? 0.f : LIFT - ref; };
          settle();
          // their weights against the reference (over 8-bit caches times the value scales), packed, and the sum of them
          auto weights = [&](int c, const float2 (&x)[16], uint32_t bits, float2& sum, uint32_t* pk) {
            float4 v = {};
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float2 y = fma2(x[k], rs2, make_float2(b1, b1));
              float2 e = make_float2(ex2(y.x), ex2(y.y));
              if (bits != 0xffffffffu) {                      // what a hidden token holds may be anything
                if (!(bits >> (2 * k) & 1u)) e.x = 0.f;
                if (!(bits >> (2 * k + 1) & 1u)) e.y = 0.f;
              }
              if (Q8) {
                sum = add2(sum, e);
                if (k % 2 == 0) v = *reinterpret_cast<const float4*>(vs + c + 2 * k);
                e = mul2(e, k % 2 == 0 ? make_float2(v.x, v.y) : make_float2(v.z, v.w));
                if (bits != 0xffffffffu) {
                  if (!(bits >> (2 * k) & 1u)) e.x = 0.f;
                  if (!(bits >> (2 * k + 1) & 1u)) e.y = 0.f;
                }
              }
              pk[k] = TypeTraits<M>::pack2(e.x, e.y);
              if (!Q8) sum = add2(sum, TypeTraits<M>::unpack2(pk[k]));
            }
          };
          float mx = -CUDART_INF_F;
          bool done = false, known = false;                   // the row's maximum is known
          if (__all_sync(0xffffffffu, plain && ref > -CUDART_INF_F)) {
            uint32_t pk[2][32];
            float2 sum = l;
#pragma unroll
            for (int c = 0; c < TK; c += 32) {
              float2 x[16];
              scores(c, x);
              if (!Q8)
#pragma unroll
                for (int k = 0; k < 16; ++k) mx = fmaxf(mx, fmaxf(x[k].x, x[k].y));
              weights(c, x, 0xffffffffu, sum, pk[c / 64] + (c & 32) / 2);
            }
            bool good;
            if (Q8) {                                         // the products show by themselves whether the reference has to move
              __half2 top[4];
#pragma unroll
              for (int k = 0; k < 64; ++k) {
                const __half2 y = __habs2(*reinterpret_cast<const __half2*>(&pk[k / 32][k & 31]));
                top[k & 3] = k < 4 ? y : __hmax2(top[k & 3], y);
              }
              const float2 t = __half22float2(__hmax2(__hmax2(top[0], top[1]), __hmax2(top[2], top[3])));
              good = fmaxf(t.x, t.y) <= LARGEST_PRODUCT && !(fmaxf(sum.x, sum.y) >= LARGEST_SUM);
            } else {
              good = mx * row_scale <= ref + SLACK;
            }
            done = __all_sync(0xffffffffu, good);
            known = !Q8;
            if (done) {
              l = sum;
              tmem_st32(t_s, pk[0]);
              tmem_st32(t_s + 32, pk[1]);
            }
          }
          if (!done) {                                        // S is still there: P has not been stored
            float px = -CUDART_INF_F;                         // the largest score + log2 |value scale|
#pragma unroll 1
            for (int c = 0; c < TK && !known; c += 32) {
              float2 x[16];
              scores(c, x);
              const uint32_t bits = plain ? 0xffffffffu : seen(c);
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const uint32_t two = bits >> (2 * k);
                if (two & 1u) mx = fmaxf(mx, x[k].x);
                if (two & 2u) mx = fmaxf(mx, x[k].y);
                if (Q8) {
                  const float2 v = *reinterpret_cast<const float2*>(vs + TK + c + 2 * k);
                  if (two & 1u) px = fmaxf(px, fmaf(x[k].x, row_scale, v.x));
                  if (two & 2u) px = fmaxf(px, fmaf(x[k].y, row_scale, v.y));
                }
              }
            }
            mx *= row_scale;
            if (Q8) mx = ceilf(fmaxf(px, mx - FLOOR));
            const float to = mx > ref + SLACK ? mx : ref;     // by the row's own scores: rows stay independent
            const float f = Q8 ? moved(ref, to) : to == -CUDART_INF_F ? 1.f : exp2f(ref - to);
            ref = to;
            l = mul2(l, make_float2(f, f));
            if (items > 0 && __any_sync(0xffffffffu, f != 1.f)) {      // S of this item is behind P.V of the last one
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                uint32_t v[32];
                tmem_ld32(t_o + c, v);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
                tmem_st32(t_o + c, v);
              }
            }
            settle();
#pragma unroll 1
            for (int c = 0; c < TK; c += 32) {                // P of 32 columns takes 16, behind what is still to be read
              float2 x[16];
              uint32_t pk[16];
              scores(c, x);
              weights(c, x, plain ? 0xffffffffu : seen(c), l, pk);
              tmem_st16(t_s + c / 2, pk);
            }
          }
          tmem_wait_st();
        }
        if (CLEANS && !plain) {
          // Drafted rows may be hidden from some query rows only, and 0 * NaN is NaN: elements that are not finite leave
          // the tile here and are added at the end, to the rows that see their token.
          if (!Q8 && !(ok = wait(bar_vfull(stage), v_parity, 51))) break;
          // MB == 2: both groups multiply with the tile, so each cleans one half of every row, and they meet before either
          // hands its P over (their S is issued one tile ahead: neither's MMAs wait for the other's P).
          const int at = t0 + r;
          bool hit = false;
          if (at >= sp.first) {
            constexpr uint32_t EXP = std::is_same<M, __half>::value ? 0x7c00u : 0x7f80u;
            constexpr int PIECES = D / 8 / MB;
            for (int c = MB == 2 ? w * PIECES : 0, end = c + PIECES; c < end; ++c) {
              uint4* ad = reinterpret_cast<uint4*>(sm + S::V + stage * S::TILE + (c >> 3) * BOX + r * 128 + ((c & 7) << 4));
              uint32_t v[4] = {ad->x, ad->y, ad->z, ad->w};
              bool here = false;
#pragma unroll
              for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 32; e += 16)
                  if ((v[k] >> e & EXP) == EXP) { v[k] &= ~(0xffffu << e); here = true; }
              if (here) *ad = make_uint4(v[0], v[1], v[2], v[3]);
              hit |= here;
            }
            const int u = at - sp.first;
            if (hit && at >= 0 && at < sp.len) atomicOr(&bad_s[u >> 5], 1u << (u & 31));
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // before the MMA reads the tile
          if (MB == 2 && !(ok = meet())) break;
        }
        tc_fence_before();
        arrive(bar_p(w));
      }
      if (!ok) break;
      tiles_seen += ntiles;
      // ---- the last P.V: the issuer commits it to the group's S barrier ------------------------------------------
      if (items > 0) {
        if (!(ok = wait(bar_s(w), s_phase, 54))) break;
        s_phase ^= 1u;
        tc_fence_after();
      }
      if (!(ok = meet())) break;                            // both groups are through: queries, mask and flags are final
      float l1 = l.x + l.y, m1 = ref == -CUDART_INF_F ? ref : ref - LIFT;
      float f0 = 1.f, f2 = 0.f;                              // on this group's O, on the other's
      if (Q8) f0 = settle_sum(m1, l1);
      if (MB == 1) {
        if (w == 1) {
          ml_s[r] = make_float2(m1, l1);
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t v[32] = {};
            if (items > 0) { tmem_ld32(t_o + c, v); tmem_wait_ld(); }
#pragma unroll
            for (int k = 0; k < 32; ++k) join_s[(c + k) * 128 + r] = __uint_as_float(v[k]) * f0;
          }
        }
        if (!(ok = meet())) break;
        if (w == 0) {
          const float2 o = ml_s[r];
          const float m = fmaxf(m1, o.x), use = m == -CUDART_INF_F ? 0.f : m;
          const float e1 = exp2f(m1 - use);
          f2 = exp2f(o.x - use);
          f0 *= e1;
          l1 = fmaf(l1, e1, o.y * f2);
          m1 = m;
        }
      }
      if ((MB == 2 || w == 0) && busy) {
        const float inv = !pc.whole ? 1.f : l1 == 0.f ? 0.f : 1.f / l1;
        uint32_t any_bad = 0;
        if (CLEANS)
          for (int k = 0; k < words; ++k) any_bad |= bad_s[k];
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t v[32] = {};
          float x[32];
          if (items > 0) { tmem_ld32(t_o + c, v); tmem_wait_ld(); }
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            x[k] = __uint_as_float(v[k]) * f0;
            if (MB == 1) x[k] = fmaf(join_s[(c + k) * 128 + r], f2, x[k]);
          }
          if (any_bad && live) {
            for (int u = 0; u < T_; ++u)
              if ((bad_s[u >> 5] >> (u & 31) & 1u) && (mask_s[tok * words + (u >> 5)] >> (u & 31) & 1u)) {
                const int64_t vr = (int64_t)pc.b * p.v_sb + (int64_t)pc.h * p.v_sh + (int64_t)(sp.first + u) * p.v_sl + c;
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                  const float y = Q8 ? __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(p.v)[vr + k], __NV_E4M3)))
                                     : to_float(static_cast<const T*>(p.v)[vr + k]);
                  if (!(fabsf(y) < CUDART_INF_F)) x[k] += y;
                }
              }
          }
          if (live && pc.whole) {
            T* out = static_cast<T*>(p.out) + (int64_t)pc.b * p.o_sb + ((int64_t)pc.h * a.rows + row) * p.o_sr + c;
            if (p.o_sb % 8 == 0 && p.o_sr % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0) {
#pragma unroll
              for (int k = 0; k < 32; k += 8)
                *reinterpret_cast<uint4*>(out + k) =
                    make_uint4(TypeTraits<T>::pack2(x[k] * inv, x[k + 1] * inv), TypeTraits<T>::pack2(x[k + 2] * inv, x[k + 3] * inv),
                               TypeTraits<T>::pack2(x[k + 4] * inv, x[k + 5] * inv), TypeTraits<T>::pack2(x[k + 6] * inv, x[k + 7] * inv));
            } else {
#pragma unroll
              for (int k = 0; k < 32; ++k) out[k] = from_float<T>(x[k] * inv);
            }
          } else if (live) {
            float* po = a.part_o + (pc.id * (MB * 128) + blk * 128 + r) * D + c;
#pragma unroll
            for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4*>(po + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
          }
        }
        if (live && !pc.whole) a.part_ml[pc.id * (MB * 128) + blk * 128 + r] = make_float2(m1, l1);
      }
      tc_fence_before();
      if (!(ok = meet())) break;                            // the next strip's queries may go in
    }
  } else if (warp == 8) {
    // ================================ MMA issuer =============================================================
    {
      // The whole warp walks the loop and one lane issues: operands that are the same in all lanes stay in uniform
      // registers, where the MMA wants them.  (One thread alone moved them there for every MMA and spent twice the time
      // of the MMA on it.)
      const bool lead = elect();
      constexpr uint32_t F = TypeTraits<M>::kFmt;
      constexpr uint32_t id_s = (1u << 4) | (F << 7) | (F << 10) | ((TK >> 3) << 17) | ((128u >> 4) << 24);
      constexpr uint32_t id_o = (1u << 4) | (F << 7) | (F << 10) | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
      const uint64_t dq = smem_desc(base + S::Q, 16, 1024), dk = smem_desc(base + S::K, 16, 1024), dv = smem_desc(base + S::V, BOX, 1024);
      uint32_t q_phase = 0, p_phase = 0;                    // p_phase: bit w
      int seen = 0;
      bool ok = true;
      auto waits = [&](uint32_t bar, uint32_t parity, int role) {
        if (__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag))) return true;
        if (lane == 0) report(a.status, XKV_ERR_TIMEOUT, role, pc.b, pc.h, pc.begin);
        return false;
      };
      while (ok && next_piece(a, walk, pc)) {
        const Span sp = span_of(p, pc.b);
        const int items = __shfl_sync(0xffffffffu, tiles_of(pc, sp.len), 0) * MB;
        // The issuer arrives too, so that the softmax warps never get two strips ahead: over strips without tiles nothing else
        // holds them, and a phase that has turned twice looks like one that has not.
        if (lead) mbar_arrive(bar_q);
        __syncwarp();
        if (!(ok = waits(bar_q, q_phase, 60))) break;
        q_phase ^= 1u;
        tc_fence_after();
        auto scores = [&](int j) {
          const int tile = seen + j / MB, stage = tile % STAGES, w = j & 1;
          if (!waits(bar_kfull(stage), (uint32_t)(tile / STAGES) & 1u, 61)) return false;
          tc_fence_after();
          const uint64_t q = desc_advance(dq, MB == 2 ? (uint32_t)(w * S::TILE) : 0u), k = desc_advance(dk, (uint32_t)(stage * S::TILE));
          const uint32_t d = tmem + (uint32_t)w * 128u;
          if (lead) {
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
              tc_mma(d, desc_advance(q, (s >> 2) * BOX + (s & 3) * 32), desc_advance(k, (s >> 2) * BOX + (s & 3) * 32), id_s, s ? 1u : 0u);
            tc_commit(bar_s(w));
            if (MB == 1 || w == 1) tc_commit(bar_kempty(stage));
          }
          __syncwarp();
          return true;
        };
        for (int j = 0; j < 2 && j < items; ++j)
          if (!(ok = scores(j))) break;
        for (int j = 0; ok && j < items; ++j) {
          const int tile = seen + j / MB, stage = tile % STAGES, w = j & 1;
          if (!(ok = waits(bar_p(w), (p_phase >> w) & 1u, 62))) break;
          p_phase ^= 1u << w;
          if (!(ok = waits(bar_vfull(stage), (uint32_t)(tile / STAGES) & 1u, 63))) break;
          tc_fence_after();
          const uint64_t v = desc_advance(dv, (uint32_t)(stage * S::TILE));
          const uint32_t o = tmem + 256u + (uint32_t)w * 128u, pt = tmem + (uint32_t)w * 128u, first = j < 2 ? 0u : 1u;
          if (lead) {
            tc_mma_ts(o, pt, v, id_o, first);
#pragma unroll
            for (int s = 1; s < TK / 16; ++s) tc_mma_ts(o, pt + s * 8, desc_advance(v, s * 2048), id_o, 1u);
            if (MB == 1 || w == 1) tc_commit(bar_vempty(stage));
            if (j + 2 >= items) tc_commit(bar_s(w));        // the group's last P.V
          }
          __syncwarp();
          if (j + 2 < items) ok = scores(j + 2);
        }
        seen += items / MB;
      }
    }
    __syncwarp();
  } else if constexpr (!Q8) {
    // ================================ tiles by TMA ============================================================
    if (warp == 9 && lane == 0) {
      int seen = 0;
      bool ok = true;
      while (ok && next_piece(a, walk, pc)) {
        const Span sp = span_of(p, pc.b);
        const int ntiles = tiles_of(pc, sp.len);
        for (int i = 0; ok && i < ntiles; ++i, ++seen) {
          const int stage = seen % STAGES, at = (pc.begin + i) * TK;
          const uint32_t parity = ((uint32_t)(seen / STAGES) & 1u) ^ 1u;
#pragma unroll
          for (int x = 0; x < 2 && ok; ++x) {
            const uint32_t full = x ? bar_vfull(stage) : bar_kfull(stage);
            if (!(ok = mbar_wait(x ? bar_vempty(stage) : bar_kempty(stage), parity, abort_flag))) {
              report(a.status, XKV_ERR_TIMEOUT, 70 + x, pc.b, pc.h, at);
              break;
            }
            mbar_expect_tx(full, S::TILE);
#pragma unroll
            for (int c = 0; c < S::HALVES; ++c)
              tma_load_4d(base + (x ? S::V : S::K) + stage * S::TILE + c * BOX, x ? &tmV : &tmK, c * 64, pc.h * a.map_h[x], at, pc.b * a.map_b[x], full);
          }
        }
      }
    }
    __syncwarp();
  } else if (warp >= 12) {
    // ================================ codes widened into tiles ===============================================
    constexpr int ROWS = TK / WIDENERS;                          // of a tile, per warp
    constexpr int CH = D / 16, RPI = 32 / CH, N = ROWS / RPI;    // 16-byte pieces of a row; rows per access of the warp; accesses
    const int c4 = warp - 12, r0 = lane / CH, c = lane % CH;      // this warp's tokens of a tile start at ROWS c4
    int seen = 0;
    bool ok = true;
    uint4 kr[N], vr[N];
    float ksr = 0.f, vsr = 0.f;
    // a tile that is not known yet is loaded when its turn comes; within a strip loads run one tile ahead
    auto load = [&](uint4 (&x)[N], const void* codes, int64_t sb, int64_t sh, int64_t sl, int t0, int len) {
      const uint8_t* src = static_cast<const uint8_t*>(codes) + (int64_t)pc.b * sb + (int64_t)pc.h * sh + c * 16;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = t0 + c4 * ROWS + i * RPI + r0;
        x[i] = make_uint4(0, 0, 0, 0);
        if (at < len) x[i] = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)at * sl));
      }
    };
    auto store = [&](const uint4 (&x)[N], uint32_t dst) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = c4 * ROWS + i * RPI + r0;
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t y = CODE == XKV_CACHE_INT8 ? w[k] ^ 0x80808080u : w[k];
          h[2 * k] = widen<CODE>(y, 0);
          h[2 * k + 1] = widen<CODE>(y, 1);
        }
        uint8_t* to = sm + dst + (c >> 2) * BOX + row * 128;
        *reinterpret_cast<uint4*>(to + ((((c & 3) * 2) ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(to + ((((c & 3) * 2 + 1) ^ (row & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
    };
    auto wait = [&](uint32_t bar, uint32_t parity, int role) {
      if (__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag))) return true;
      if (lane == 0) report(a.status, XKV_ERR_TIMEOUT, role, pc.b, pc.h, pc.begin);
      return false;
    };
    while (ok && next_piece(a, walk, pc)) {
      const Span sp = span_of(p, pc.b);
      const int ntiles = tiles_of(pc, sp.len);
      const float* ksg = p.k_scales + (int64_t)pc.b * p.ks_sb + (int64_t)pc.h * p.ks_sh;
      const float* vsg = p.v_scales + (int64_t)pc.b * p.vs_sb + (int64_t)pc.h * p.vs_sh;
      auto load_k = [&](int i) {
        const int t0 = (pc.begin + i) * TK, at = t0 + c4 * ROWS + lane;
        load(kr, p.k, p.k_sb, p.k_sh, p.k_sl, t0, sp.len);
        ksr = lane < ROWS && at < sp.len ? __ldg(ksg + at) : 0.f;
      };
      auto load_v = [&](int i) {
        const int t0 = (pc.begin + i) * TK, at = t0 + c4 * ROWS + lane;
        load(vr, p.v, p.v_sb, p.v_sh, p.v_sl, t0, sp.len);
        vsr = lane < ROWS && at < sp.len ? __ldg(vsg + at) : 0.f;
      };
      if (ntiles > 0) { load_k(0); load_v(0); }
      for (int i = 0; i < ntiles; ++i, ++seen) {
        const int stage = seen % STAGES;
        const uint32_t parity = ((uint32_t)(seen / STAGES) & 1u) ^ 1u;
        float* ks = reinterpret_cast<float*>(sm + S::SCALES + stage * 3 * TK * 4);
        if (!(ok = wait(bar_kempty(stage), parity, 70))) break;
        store(kr, S::K + stage * S::TILE);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_kfull(stage));
        const float k_scale = ksr;
        if (i + 1 < ntiles) load_k(i + 1);
        if (!(ok = wait(bar_vempty(stage), parity, 71))) break;
        store(vr, S::V + stage * S::TILE);
        if (lane < ROWS) {
          ks[c4 * ROWS + lane] = k_scale;
          ks[TK + c4 * ROWS + lane] = vsr;
          ks[2 * TK + c4 * ROWS + lane] = log2_size(vsr);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_vfull(stage));
        if (i + 1 < ntiles) load_v(i + 1);
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);        // copies in flight land
  }
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <typename T, int CODE, int D, int MB>
int launch(const CUtensorMap& tK, const CUtensorMap& tV, const Args& a, cudaStream_t st) {
  auto kern = tree_tc_kernel<T, CODE, D, MB>;
  static_assert(Smem<D, MB>::BYTES <= 232448, "shared memory budget exceeded");
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D, MB>::BYTES) != cudaSuccess) {
    cudaGetLastError();
    return XKV_ERR_LAUNCH;
  }
  kern<<<(unsigned)a.grid, threads<CODE>(), Smem<D, MB>::BYTES, st>>>(tK, tV, a);
  return cudaGetLastError() == cudaSuccess ? XKV_OK : XKV_ERR_LAUNCH;
}
template <typename T, int CODE>
int by_shape(const CUtensorMap& tK, const CUtensorMap& tV, const Args& a, cudaStream_t st) {
  if (a.p.head_dim == 128)
    return a.block_rows == 128 ? launch<T, CODE, 128, 1>(tK, tV, a, st) : launch<T, CODE, 128, 2>(tK, tV, a, st);
  return a.block_rows == 128 ? launch<T, CODE, 64, 1>(tK, tV, a, st) : launch<T, CODE, 64, 2>(tK, tV, a, st);
}
template <typename T>
int by_code(const CUtensorMap& tK, const CUtensorMap& tV, const Args& a, cudaStream_t st) {
  if (a.p.cache_code == XKV_CACHE_DENSE) return by_shape<T, XKV_CACHE_DENSE>(tK, tV, a, st);
  return a.p.cache_code == XKV_CACHE_INT8 ? by_shape<T, XKV_CACHE_INT8>(tK, tV, a, st) : by_shape<T, XKV_CACHE_E4M3>(tK, tV, a, st);
}

bool encode(CUtensorMap* m, const xkv_tree_params& p, const void* ptr, int64_t sb, int64_t sh, int64_t sl, int* map_b, int* map_h) {
  *map_b = sb != 0;
  *map_h = sh != 0;
  const int nb = sb ? p.batch : 1, nh = sh ? p.num_kv_heads : 1;
  const cuuint64_t dims[4] = {(cuuint64_t)p.head_dim, (cuuint64_t)nh, (cuuint64_t)p.kv_len, (cuuint64_t)nb};
  // a dimension of one element may have any stride: its place in the map takes a legal one
  const cuuint64_t strides[3] = {(cuuint64_t)(nh > 1 ? sh : p.head_dim) * 2, (cuuint64_t)sl * 2, (cuuint64_t)(nb > 1 ? sb : p.head_dim) * 2};
  const cuuint32_t box[4] = {64, 1, TK, 1};
  return encode_tiled_16bit(m, p.dtype, 4, ptr, dims, strides, box);
}
// what a tensor map takes: 16-byte rows, strides below 2^40 bytes; 0 (one cache for all) only across sequences and heads
bool map_ok(const void* ptr, int64_t stride, int n, bool zero = true) {
  return aligned16(ptr) && (n == 1 || (zero && stride == 0) || (stride_ok(stride) && stride < (int64_t(1) << 39)));
}

}  // namespace
}  // namespace tree

bool tree_tc_supported(const xkv_tree_params& p, int rows) {
  using namespace tree;
  if (p.dtype == XKV_F32 || rows <= 16 || p.num_tokens > MAX_T) return false;
  // The stream kernel reads the cache once per 16 rows, this one once, but it takes some 8 us longer to set up (tensor
  // memory, operands in shared memory, three meetings per strip): SETUP bytes of reading.  R = 24 over 8 heads of 1023
  // 16-bit rows (4 MB): 17 us there, 25 here; R = 104 over 8 x 16384 rows (537 MB): 405 us there, 125 here.
  constexpr double SETUP = 48e6;
  const double bytes = 2.0 * p.batch * p.num_kv_heads * p.kv_len * p.head_dim * (p.cache_code == XKV_CACHE_DENSE ? 2 : 1);
  if ((p.flags & XKV_FLAG_TREE_MMA_SYNC) || (!(p.flags & XKV_FLAG_TREE_TCGEN05) && bytes * (ceil_div(rows, 16) - 1) < SETUP)) return false;
  if (p.cache_code != XKV_CACHE_DENSE) return true;      // beyond what tree_stream_supported() has checked
  return map_ok(p.k, p.k_sb, p.batch) && map_ok(p.k, p.k_sh, p.num_kv_heads) && map_ok(p.k, p.k_sl, 2, false) &&
         map_ok(p.v, p.v_sb, p.batch) && map_ok(p.v, p.v_sh, p.num_kv_heads) && map_ok(p.v, p.v_sl, 2, false);
}

void tree_tc_plan(const xkv_tree_params&, TreePlan* pl) {
  pl->kernel = TreePlan::kTc;
  pl->name = "tree_tc";
  pl->block_rows = pl->rows <= 128 ? 128 : 256;
  pl->unit_tokens = tree::TK;
  pl->slots = device_sm_count();
}

int tree_tc_decode(const tree::Args& args, cudaStream_t st) {
  using namespace tree;
  Args a = args;
  CUtensorMap tK = {}, tV = {};
  const xkv_tree_params& p = a.p;
  if (p.cache_code == XKV_CACHE_DENSE && (!encode(&tK, p, p.k, p.k_sb, p.k_sh, p.k_sl, &a.map_b[0], &a.map_h[0]) ||
                                          !encode(&tV, p, p.v, p.v_sb, p.v_sh, p.v_sl, &a.map_b[1], &a.map_h[1])))
    return XKV_ERR_NO_DEVICE;
  return p.dtype == XKV_BF16 ? by_code<__nv_bfloat16>(tK, tV, a, st) : by_code<__half>(tK, tV, a, st);
}

}  // namespace xkv
