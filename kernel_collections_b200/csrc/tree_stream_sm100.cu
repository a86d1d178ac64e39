// Tree / decode attention for few query rows: the cache streams once through registers and mma.sync.
//
// Up to 16 query rows (heads of a KV head x drafted tokens) share one pass, so the arithmetic is far below the tensor
// rate and the pass is bound by HBM as long as the instructions per cache byte stay low.  Hence:
//  * Every warp is on its own: it copies its 4 KB of K and of V (32 tokens of 128 codes, 16 of 128 halves) into a private
//    two-stage ring with cp.async and meets the other warps only at the end of a piece.  No block barrier in the loop,
//    nothing to wait for but its own copies.  Eight warps in one block per SM, one tile ahead: twelve warps, or eight with
//    two tiles ahead, have more bytes in flight and reach less of HBM (4 x 131071 rows of 8 heads: 189 us against 200).
//  * With at most 8 query rows the tokens (and, for P.V, the dims) are the 16 rows of the MMA and the queries its 8 columns:
//    half the MMAs, accumulators and exponentials of the 16-row form, which pads the queries to 16.  The weights then
//    turn from accumulator to operand layout by movmatrix.
//  * 8-bit codes are widened in registers on their way into the MMA and never written back.  The contraction index of
//    Q.K^T may be permuted freely, so a thread takes 16 consecutive codes of a token (one 16-byte read) and Q is laid
//    out to match.  For P.V the two tokens of an operand register are interleaved by byte permutes.  int8: the code
//    with its sign bit flipped under the exponent byte 0x64 is the half 1024 + 128 + code, less 1152 (exactly; taken off
//    the score instead, the offset's roundings are as large as the scores of keys whose scale one channel has set); e4m3
//    converts in pairs.
//    Widened codes are exact in fp16 (8 significant bits), so the products run in fp16 whatever the query type.
//  * Scales never touch the codes: the key scale multiplies the score, the value scale the weight.
//  * fp16 ranges: a query row is multiplied by a power of two that brings its largest element to 2^14..2^15, and divided
//    out of the scores in fp32: elements below 2^-28 of the largest lose bits, others none.  Weights carry the factor 2^6
//    (it cancels in O / l) and go into the product times their value scale, relative to the largest such product: those down
//    to 2^-20 of it keep all 11 bits, however large the scale of a row without weight may be.
//  * fp32 queries: Q and P in two fp16 terms each (22 bits), two MMAs instead of one.
//  * Over 8-bit caches the reference of the exponents is checked on the products themselves, after they are formed (the few
//    tiles that move it form them again): no maximum over scores or scales, no exchange between lanes, in the others.
// Calls queued back to back: 4 x 131071 rows of 8 heads (e4m3, 8 query rows per head, 1.1 GB) 168 to 179 us, 6.2 to 6.6 TB/s, GPU to GPU; the
// same in int8 168, with fp32 queries 175 to 179, with 16 query rows 199.  16 ragged sequences of up to 16384 int8 rows (0.42 GB):
// 74 to 81 us.  One sequence of 777 rows: 13 us, the host's time for the call.
#include "tree_common.cuh"
#include "sm100_common.cuh"
#include <type_traits>

namespace xkv {
namespace tree {
using namespace sm100;
namespace {

constexpr int NW = 8, NT = NW * 32, STAGES = 2, HALF = 4096;   // HALF: bytes of K (or V) per warp and stage

template <typename T> __device__ __forceinline__ float to_float(T v) { return TypeTraits<T>::to_f(v); }
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v) { return TypeTraits<T>::from_f(v); }
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
// 2^x, relative error below 2^-22; 0 for -inf
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

// Two halves from the bytes `sel` picks of x: int8 codes (sign bits flipped beforehand), e4m3 codes.
__device__ __forceinline__ uint32_t widen_int8(uint32_t x, uint32_t sel) {
  const uint32_t y = __byte_perm(x, 0x64646464u, sel);         // {code + 128, 0x64, code' + 128, 0x64}
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&y), __half2half2(__ushort_as_half(0x6480)));   // - 1152
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t widen_e4m3(uint32_t x, int high) {
  uint32_t r;
  const uint16_t two = (uint16_t)(high ? x >> 16 : x);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
  return r;
}
// 8 x 8 transpose of 16-bit elements across the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// bytes 0, 1 of x (high = 0) or 2, 3 as two halves
template <int CODE> __device__ __forceinline__ uint32_t widen(uint32_t x, int high) {
  return CODE == XKV_CACHE_INT8 ? widen_int8(x, high ? 0x4342u : 0x4140u) : widen_e4m3(x, high);
}

template <typename T, int CODE, int D>
struct Shape {
  static constexpr int ES = CODE == XKV_CACHE_DENSE ? 2 : 1;
  static constexpr int ROWB = D * ES;              // bytes of a cache row
  static constexpr int CH = ROWB / 16;             // its 16-byte pieces
  static constexpr int TOK = HALF / ROWB;          // tokens per warp and stage
  static constexpr int UNIT = NW * TOK;            // tokens per block and stage
  static constexpr int SCALES = ES == 1 ? TOK * 8 : 0;
  static constexpr int STAGE = 2 * HALF + SCALES;
  static constexpr int FRAGS = D / 16 * 512;       // bytes of one term of the queries as MMA operands
  static_assert(16 * D * 4 <= STAGE, "the second stage of the first warp holds the staged queries");
  // pieces of a row are permuted by the row so that the reads below touch every bank once
  static __device__ __forceinline__ int at(int row, int c) { return row * ROWB + ((c ^ (CH >= 8 ? row & 7 : (row >> 1) & 3)) << 4); }
  // piece i (of CH / 4) that lane t of a quad reads of its token, and the first of the four dims of k-step s
  static __device__ __forceinline__ int piece(int i, int t) { return CH >= 8 ? t * 2 + (i & 1) + 8 * (i >> 1) : t; }
  static constexpr int KPC = 4 / ES;               // k-steps per piece
  static __device__ __forceinline__ int dim0(int s, int t) { return piece(s / KPC, t) * (16 / ES) + (s % KPC) * 4; }
};

// RB query rows per strip.  A thread's two rows and its tokens of every 8: RB == 16: rows g, g + 8 and tokens 2t, 2t + 1;
// RB == 8: rows 2t, 2t + 1 and token g.
template <typename T, int CODE, int D, int TERMS, int RB>
__global__ void __launch_bounds__(NT, 1) stream_kernel(const Args a) {
  using S = Shape<T, CODE, D>;
  constexpr bool Q8 = CODE != XKV_CACHE_DENSE, WIDE = RB == 16;
  using M = typename std::conditional<Q8, __half, typename std::conditional<std::is_same<T, float>::value, __half, T>::type>::type;
  constexpr int TOK = S::TOK, NS = TOK / 8, KS = D / 16, NO = D / 8;
  constexpr int E = WIDE ? 2 : 1;                  // tokens of every 8 that a thread scores, for each of its rows
  constexpr int QV = WIDE ? 1 : 2;                 // k-steps per 16 bytes of query operand
  // weights are 2^(score - reference + LIFT); the reference follows the maximum when it is passed by more than SLACK
  constexpr float LIFT = std::is_same<M, __half>::value ? 6.f : -12.f, SLACK = std::is_same<M, __half>::value ? 9.f : 20.f;
  extern __shared__ __align__(128) uint8_t smem[];
  const xkv_tree_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;");
  if (blockIdx.x == 0 && threadIdx.x < 8) a.status[threadIdx.x] = 0;       // nothing here waits: the status is always good
  Walk walk = walk_of(a, lane);
  Piece pc;
  while (next_piece(a, walk, pc)) {
    const int b = pc.b, h = pc.h, rb = pc.rb;
    const Span sp = span_of(p, b);
    const int mult = a.unit_tokens / S::UNIT;        // tiles of all warps per unit of the line
    const int begin = pc.begin * mult, end = min(pc.end * mult, (sp.len + S::UNIT - 1) / S::UNIT);

    uint8_t* const ring = smem + warp * (STAGES * S::STAGE);
    const uint32_t ring_a = smem_u32(ring);
    const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + ((int64_t)b * p.k_sb + (int64_t)h * p.k_sh) * S::ES;
    const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + ((int64_t)b * p.v_sb + (int64_t)h * p.v_sh) * S::ES;
    const float* ksc = Q8 ? p.k_scales + (int64_t)b * p.ks_sb + (int64_t)h * p.ks_sh : nullptr;
    const float* vsc = Q8 ? p.v_scales + (int64_t)b * p.vs_sb + (int64_t)h * p.vs_sh : nullptr;
    const int64_t k_pitch = p.k_sl * S::ES, v_pitch = p.v_sl * S::ES;
    auto fetch = [&](int u, int stage) {        // this warp's tokens of unit u; rows past the length arrive as zeros
      if (u < end) {
        const int t0 = u * S::UNIT + warp * TOK;
        const uint32_t dst = ring_a + stage * S::STAGE;
        constexpr int RPI = 32 / S::CH;         // rows per iteration of the warp (CH <= 16)
        const int r0 = lane / S::CH, c = lane % S::CH;
        if (t0 + TOK <= sp.len) {
          const uint8_t* ks = kbase + (int64_t)(t0 + r0) * k_pitch + c * 16;
          const uint8_t* vs = vbase + (int64_t)(t0 + r0) * v_pitch + c * 16;
#pragma unroll
          for (int i = 0; i < TOK / RPI; ++i) {
            const uint32_t at = dst + S::at(i * RPI + r0, c);
            cp16(at, ks);
            cp16(at + HALF, vs);
            ks += RPI * k_pitch;
            vs += RPI * v_pitch;
          }
          if (Q8) {
#pragma unroll
            for (int i = 0; i < TOK; i += 32) {
              cp4(dst + 2 * HALF + (i + lane) * 4, ksc + t0 + i + lane, true);
              cp4(dst + 2 * HALF + TOK * 4 + (i + lane) * 4, vsc + t0 + i + lane, true);
            }
          }
        } else {
          for (int i = 0; i < TOK / RPI; ++i) {
            const int row = i * RPI + r0;
            const bool live = t0 + row < sp.len;
            const int64_t at = live ? t0 + row : 0;
            cp16_or_zero(dst + S::at(row, c), kbase + at * k_pitch + c * 16, live);
            cp16_or_zero(dst + HALF + S::at(row, c), vbase + at * v_pitch + c * 16, live);
          }
          if (Q8) {
            for (int i = 0; i < TOK; i += 32) {
              const int row = i + lane;
              const bool live = t0 + row < sp.len;
              cp4(dst + 2 * HALF + row * 4, ksc + (live ? t0 + row : 0), live);
              cp4(dst + 2 * HALF + TOK * 4 + row * 4, vsc + (live ? t0 + row : 0), live);
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(begin, 0);

    // ---- queries: scaled rows as fp32 in the free second stage, then as MMA operands --------------------------------
    float* qs = reinterpret_cast<float*>(smem + S::STAGE);                         // [row][D]
    uint4* qfrag = reinterpret_cast<uint4*>(smem + NW * STAGES * S::STAGE);        // [term][k-step / QV][lane]
    float* qrow = reinterpret_cast<float*>(qfrag + TERMS * S::FRAGS / 16);         // [row]: row_scale
    const int T_ = p.num_tokens, G = p.num_heads / p.num_kv_heads;
    for (int r = warp; r < RB; r += NW) {
      const int row = rb * RB + r;
      const T* q = static_cast<const T*>(p.q) + (int64_t)b * p.q_sb + (int64_t)(h * G + row / T_) * p.q_sh + (int64_t)(row % T_) * p.q_st;
      float x[D / 32], top = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        x[i] = row < a.rows ? to_float(q[i * 32 + lane]) : 0.f;
        top = fmaxf(top, fabsf(x[i]));
      }
      top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
      // the sign of the scale goes to the queries, so that the largest product is the largest score; a scale of zero too
      float up = a.scale_log2 < 0.f ? -1.f : 1.f, scale = fmaxf(fabsf(a.scale_log2), 1.17549435e-38f);
      if (a.scale_log2 == 0.f) {
        up = 0.f;
        scale = 1.f;
      } else if (Q8 && top > 0.f && top < CUDART_INF_F) {
        const int e = min(max(14 - (int)(((__float_as_uint(top) >> 23) & 255u)) + 127, -120), 120);
        up *= __uint_as_float((uint32_t)(e + 127) << 23);
        scale = fmaxf(scale * __uint_as_float((uint32_t)(127 - e) << 23), 1.17549435e-38f);
      }
#pragma unroll
      for (int i = 0; i < D / 32; ++i) qs[r * D + i * 32 + lane] = x[i] * up;
      if (lane == 0) qrow[r] = scale;
    }
    __syncthreads();
    for (int s = warp; s < KS; s += NW) {
      uint32_t f[TERMS][2 * E];         // WIDE: (row g, dims 0 1), (g + 8, 0 1), (g, 2 3), (g + 8, 2 3); else (g, 0 1), (g, 2 3)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int r = 0; r < E; ++r) {
          const float* q = qs + (g + r * 8) * D + S::dim0(s, t) + 2 * k;
          f[0][r + E * k] = TypeTraits<M>::pack2(q[0], q[1]);
          if (TERMS == 2) {
            const float2 z = TypeTraits<M>::unpack2(f[0][r + E * k]);
            f[TERMS - 1][r + E * k] = TypeTraits<M>::pack2(q[0] - z.x, q[1] - z.y);
          }
        }
#pragma unroll
      for (int x = 0; x < TERMS; ++x) {
        if constexpr (WIDE) qfrag[(x * KS + s) * 32 + lane] = make_uint4(f[x][0], f[x][1], f[x][2], f[x][3]);
        else reinterpret_cast<uint2*>(qfrag)[((x * KS + s) / 2 * 32 + lane) * 2 + (s & 1)] = make_uint2(f[x][0], f[x][1]);
      }
    }
    float row_scale[2];       // score = accumulator * row_scale (* key scale), row_scale > 0
#pragma unroll
    for (int r = 0; r < 2; ++r) row_scale[r] = qrow[WIDE ? g + 8 * r : 2 * t + r];
    __syncthreads();

    float ref[2] = {-CUDART_INF_F, -CUDART_INF_F};                        // of the scores; 8-bit caches: of the products
    float2 l[2] = {{0.f, 0.f}, {0.f, 0.f}};                               // WIDE: [row]{token}; else [0]{row}
    // WIDE: [n]: rows g, g + 8 x columns 2t, 2t + 1 of 8 dims n.  Else [n / 2]: columns g of dims n, n + 1 x rows 2t, 2t + 1
    float o[NO * E / 2][4];
#pragma unroll
    for (int n = 0; n < NO * E / 2; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    // the largest over the lanes that share a thread's rows
    auto across = [](float x) {
      if (WIDE) {
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
      }
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
      return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
    };
    const int tok0 = WIDE ? 2 * t : g;          // + 8n + e: this thread's tokens
    // query row and dim of o[n][i]; 8-bit caches deal NO consecutive dims to each of the eight columns
    auto row_of = [&](int i) { return WIDE ? g + 8 * (i >> 1) : 2 * t + (i & 1); };
    auto dim_of = [&](int n, int i) {
      const int col = WIDE ? 2 * t + (i & 1) : g, tile = WIDE ? n : 2 * n + (i >> 1);
      return Q8 ? col * NO + tile : tile * 8 + col;
    };

    int stage = 0;
    for (int u = begin; u < end; ++u) {
      const int nxt = stage + STAGES - 1;
      fetch(u + STAGES - 1, nxt >= STAGES ? nxt - STAGES : nxt);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
      const int t0 = u * S::UNIT + warp * TOK;
      const uint8_t* const sk = ring + stage * S::STAGE;
      const uint8_t* const sv = sk + HALF;
      const float* const kss = reinterpret_cast<const float*>(sv + HALF);      // key scales, then value scales
      if (++stage == STAGES) stage = 0;
      if (t0 >= sp.len) continue;
      const bool plain = t0 + TOK <= sp.first;     // every row sees every token of this step

      // ---- scores ---------------------------------------------------------------------------------------------
      // WIDE: sc[n][2r + e], token 8n + 2t + e of row g + 8r; else sc[n / 2][2 (n & 1) + r], token 8n + g of row 2t + r
      float sc[NS * E / 2][4];
#pragma unroll
      for (int n = 0; n < NS * E / 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][i] = 0.f;
#pragma unroll
      for (int i = 0; i < S::CH / 4; ++i) {
        uint4 qf[TERMS][S::KPC / QV];
#pragma unroll
        for (int x = 0; x < TERMS; ++x)
#pragma unroll
          for (int k = 0; k < S::KPC / QV; ++k) qf[x][k] = qfrag[(x * KS + i * S::KPC) / QV * 32 + k * 32 + lane];
#pragma unroll
        for (int n = 0; n < NS; n += 2 / E) {
          uint32_t w[2 / E][4];
#pragma unroll
          for (int m = 0; m < 2 / E; ++m) {
            const uint4 w4 = *reinterpret_cast<const uint4*>(sk + S::at((n + m) * 8 + g, S::piece(i, t)));
            w[m][0] = w4.x; w[m][1] = w4.y; w[m][2] = w4.z; w[m][3] = w4.w;
          }
#pragma unroll
          for (int k = 0; k < S::KPC; ++k) {
            uint32_t f[2 / E][2];         // tokens of tile n + m, dims 0 1 and 2 3
#pragma unroll
            for (int m = 0; m < 2 / E; ++m) {
              if (Q8) {
                const uint32_t x = CODE == XKV_CACHE_INT8 ? w[m][k] ^ 0x80808080u : w[m][k];
                f[m][0] = widen<CODE>(x, 0);
                f[m][1] = widen<CODE>(x, 1);
              } else {
                f[m][0] = w[m][(2 * k) & 3];
                f[m][1] = w[m][(2 * k + 1) & 3];
              }
            }
#pragma unroll
            for (int x = 0; x < TERMS; ++x) {
              const uint4 q = qf[x][k / QV];
              if constexpr (WIDE) {
                const uint32_t qa[4] = {q.x, q.y, q.z, q.w};
                TypeTraits<M>::mma(sc[n], qa, f[0][0], f[0][1]);
              } else {
                const uint32_t ka[4] = {f[0][0], f[1][0], f[0][1], f[1][1]};
                TypeTraits<M>::mma(sc[n / 2], ka, k & 1 ? q.z : q.x, k & 1 ? q.w : q.y);
              }
            }
          }
        }
      }
      auto score = [&](int n, int r, int e) -> float& { return WIDE ? sc[n][2 * r + e] : sc[n / 2][2 * (n & 1) + r]; };
      // ---- key scales and hidden tokens (scores still without row_scale) -------------------------------------------------
      uint32_t vis[2] = {0xffffffffu, 0xffffffffu};        // bit E n + e: row sees token 8n + tok0 + e
      if (Q8) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          float2 k;
          if (WIDE) k = *reinterpret_cast<const float2*>(kss + n * 8 + tok0);
          else k.x = k.y = kss[n * 8 + tok0];
#pragma unroll
          for (int r = 0; r < E; ++r) {
            float* x = WIDE ? &sc[n][2 * r] : &sc[n / 2][2 * (n & 1)];
            const float2 y = mul2(make_float2(x[0], x[1]), k);
            x[0] = y.x;
            x[1] = y.y;
          }
        }
      }
      if (!plain) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int tok = min(rb * RB + (WIDE ? g + 8 * r : 2 * t + r), a.rows - 1) % T_;
#pragma unroll
          for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const int at = t0 + n * 8 + tok0 + e;
              if (at >= sp.len || !sees(p, b, tok, at, sp.first)) {
                vis[r] &= ~(1u << (E * n + e));
                score(n, r, e) = -CUDART_INF_F;
              }
            }
        }
      }
      // the largest score of each row of the thread in this tile, over all lanes that share the row
      auto largest = [&](float (&mx)[2]) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          mx[r] = -CUDART_INF_F;
#pragma unroll
          for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int e = 0; e < E; ++e) mx[r] = fmaxf(mx[r], score(n, r, e));
          mx[r] = across(mx[r]) * row_scale[r];
        }
      };
      // to new references (by a row's own scores: rows stay independent), by the factors f
      auto rescale = [&](const float (&f)[2]) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (WIDE) l[r] = mul2(l[r], make_float2(f[r], f[r]));
        if (!WIDE) l[0] = mul2(l[0], make_float2(f[0], f[1]));
#pragma unroll
        for (int n = 0; n < NO * E / 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][i] *= f[WIDE ? i >> 1 : i & 1];
      };
      // weights of tile n: WIDE: a row's two tokens; else a token's two rows
      auto weight = [&](int n, int r) {
        const float* s2 = WIDE ? &sc[n][2 * r] : &sc[n / 2][2 * (n & 1)];
        auto two = [&](auto of) { return WIDE ? make_float2(of(r), of(r)) : make_float2(of(0), of(1)); };
        const float2 x = fma2(make_float2(s2[0], s2[1]), two([&](int i) { return row_scale[i]; }),
                              two([&](int i) { return ref[i] == -CUDART_INF_F ? 0.f : LIFT - ref[i]; }));
        return make_float2(ex2(x.x), ex2(x.y));
      };
      float2 pw[NS][E];            // what P.V multiplies with
      if constexpr (Q8) {
        // The products are formed against the reference as it is and show by themselves whether it has to move: few do.
#pragma unroll 1
        for (bool again = false;; again = true) {
          float2 sum[2] = {l[0], l[1]};
          float top = 0.f;
#pragma unroll
          for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int r = 0; r < E; ++r) {
              float2 w = weight(n, r), v;
              sum[r] = add2(sum[r], w);
              if (WIDE) v = *reinterpret_cast<const float2*>(kss + TOK + n * 8 + tok0);
              else v.x = v.y = kss[TOK + n * 8 + tok0];
              w = mul2(w, v);
              if (!plain) {                    // a hidden token's scale may be anything
                if (!(vis[WIDE ? r : 0] >> (E * n) & 1)) w.x = 0.f;
                if (!(vis[WIDE ? r : 1] >> (E * n + E - 1) & 1)) w.y = 0.f;
              }
              top = fmaxf(top, fmaxf(fabsf(w.x), fabsf(w.y)));
              pw[n][r] = w;
            }
          bool move = top > LARGEST_PRODUCT || ref[0] == -CUDART_INF_F || ref[1] == -CUDART_INF_F;
#pragma unroll
          for (int r = 0; r < E; ++r) move |= fmaxf(sum[r].x, sum[r].y) >= LARGEST_SUM;
          if (again || !__any_sync(0xffffffffu, move)) {
            l[0] = sum[0];
            l[1] = sum[1];
            break;
          }
          float mx[2], f[2];
          largest(mx);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float px = -CUDART_INF_F;          // the largest score + log2 |value scale|; hidden tokens' scores are -infinity
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
              for (int e = 0; e < E; ++e) px = fmaxf(px, fmaf(score(n, r, e), row_scale[r], log2_size(kss[TOK + n * 8 + tok0 + e])));
            px = ceilf(fmaxf(across(px), mx[r] - FLOOR));
            const float to = px > ref[r] + SLACK ? px : ref[r];
            f[r] = moved(ref[r], to);
            ref[r] = to;
          }
          rescale(f);
        }
      } else {
        float mx[2], f[2];
        largest(mx);
        if (__any_sync(0xffffffffu, mx[0] > ref[0] + SLACK || mx[1] > ref[1] + SLACK)) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float to = mx[r] > ref[r] + SLACK ? mx[r] : ref[r];
            f[r] = to == -CUDART_INF_F ? 1.f : exp2f(ref[r] - to);
            ref[r] = to;
          }
          rescale(f);
        }
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int r = 0; r < E; ++r) pw[n][r] = weight(n, r);
      }
      // ---- as operands: WIDE [term][n][r] tokens 8n + 2t, + 1 of row g + 8r; else [term][n][0] the same of row g --------------
      uint32_t pf[TERMS][NS][E];
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int r = 0; r < E; ++r) {
          const float2 w = pw[n][r];
          const uint32_t hi = TypeTraits<M>::pack2(w.x, w.y);
          const float2 f = TypeTraits<M>::unpack2(hi);
          if (!Q8) l[r] = add2(l[r], f);      // the sum of what P.V multiplies with: the rounding cancels
          pf[0][n][r] = WIDE ? hi : transpose8(hi);
          if (TERMS == 2) {
            const uint32_t lo = TypeTraits<M>::pack2(w.x - f.x, w.y - f.y);
            pf[TERMS - 1][n][r] = WIDE ? lo : transpose8(lo);
          }
        }
      // Drafted rows may be hidden from some query rows only, and 0 * NaN is NaN: elements that are not finite are taken
      // out of the value tile here and added after the product, to the rows that see their token.
      uint64_t bad = 0;
      if (!plain && CODE != XKV_CACHE_INT8) {
        for (int i = lane; i < TOK * S::CH; i += 32) {
          const int row = i / S::CH;
          uint4* ad = reinterpret_cast<uint4*>(const_cast<uint8_t*>(sv) + S::at(row, i % S::CH));
          const uint4 v4 = *ad;
          uint32_t v[4] = {v4.x, v4.y, v4.z, v4.w};
          bool hit = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (Q8) {
#pragma unroll
              for (int e = 0; e < 32; e += 8)
                if ((v[k] >> e & 0x7fu) == 0x7fu) { v[k] &= ~(0xffu << e); hit = true; }
            } else {
              constexpr uint32_t EXP = std::is_same<M, __half>::value ? 0x7c00u : 0x7f80u;
#pragma unroll
              for (int e = 0; e < 32; e += 16)
                if ((v[k] >> e & EXP) == EXP) { v[k] &= ~(0xffffu << e); hit = true; }
            }
          }
          if (hit) {
            bad |= 1ull << row;
            *ad = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
        const uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)bad), hi = __reduce_or_sync(0xffffffffu, (uint32_t)(bad >> 32));
        bad = (uint64_t)hi << 32 | lo;
        __syncwarp();
      }
      // ---- O += P.V ------------------------------------------------------------------------------------------------
#pragma unroll
      for (int kk = 0; kk < TOK / 16; ++kk) {
        // values of dims n (f[0], f[1]: tokens 2t, + 1 and 2t + 8, + 9 of column g) and n + 1 (f[2], f[3])
        auto product = [&](int n, const uint32_t (&f)[4]) {
#pragma unroll
          for (int x = 0; x < TERMS; ++x) {
            if constexpr (WIDE) {
              const uint32_t pa[4] = {pf[x][2 * kk][0], pf[x][2 * kk][E - 1], pf[x][2 * kk + 1][0], pf[x][2 * kk + 1][E - 1]};
              TypeTraits<M>::mma(o[n], pa, f[0], f[1]);
              TypeTraits<M>::mma(o[n + 1], pa, f[2], f[3]);
            } else {
              const uint32_t va[4] = {f[0], f[2], f[1], f[3]};
              TypeTraits<M>::mma(o[n / 2], va, pf[x][2 * kk][0], pf[x][2 * kk + 1][0]);
            }
          }
        };
        if constexpr (Q8) {
          constexpr int WORDS = D / 32;           // words of four dims per token that a thread widens
          uint32_t w[4][WORDS];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = kk * 16 + (j >> 1) * 8 + 2 * t + (j & 1);
            if constexpr (WORDS == 4) {
              const uint4 v = *reinterpret_cast<const uint4*>(sv + S::at(row, g));
              w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(sv + S::at(row, g >> 1) + (g & 1) * 8);
              w[j][0] = v.x; w[j][1] = v.y;
            }
            if (CODE == XKV_CACHE_INT8)
#pragma unroll
              for (int i = 0; i < WORDS; ++i) w[j][i] ^= 0x80808080u;
          }
#pragma unroll
          for (int i = 0; i < WORDS; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {        // dims 4i + 2k, + 1: bytes of two tokens side by side
              const uint32_t x = __byte_perm(w[0][i], w[1][i], k ? 0x7362u : 0x5140u);
              const uint32_t y = __byte_perm(w[2][i], w[3][i], k ? 0x7362u : 0x5140u);
              product(4 * i + 2 * k, {widen<CODE>(x, 0), widen<CODE>(y, 0), widen<CODE>(x, 1), widen<CODE>(y, 1)});
            }
        } else {
          const int mi = lane >> 3, r = lane & 7;
          const int row = kk * 16 + (mi & 1) * 8 + r;
#pragma unroll
          for (int n = 0; n < NO; n += 2) {
            uint32_t v[4];
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                         : "r"(smem_u32(sv) + S::at(row, n + (mi >> 1))) : "memory");
            product(n, v);
          }
        }
      }
      while (bad) {
        const int tok = __ffsll((long long)bad) - 1;
        bad &= bad - 1;
        const uint8_t* vr = vbase + (int64_t)(t0 + tok) * v_pitch;
#pragma unroll
        for (int n = 0; n < NO * E / 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = rb * RB + row_of(i), d = dim_of(n, i);
            const float x = Q8 ? __half2float(__half(__nv_cvt_fp8_to_halfraw(vr[d], __NV_E4M3)))
                               : to_float(reinterpret_cast<const M*>(vr)[d]);
            if (!(fabsf(x) < CUDART_INF_F) && row < a.rows && sees(p, b, row % T_, t0 + tok, sp.first)) o[n][i] += x;
          }
      }
      __syncwarp();       // every lane is done with the stage before the next copies into it
    }

    // ---- join the eight warps ------------------------------------------------------------------------------------------
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    constexpr int OS = D + 4;
    float* acc = reinterpret_cast<float*>(smem);               // [warp][row][OS]
    float2* ml = reinterpret_cast<float2*>(qfrag);             // [warp][row]
    static_assert(NW * RB * OS * 4 <= NW * STAGES * S::STAGE, "the ring holds the partial outputs");
    float f_o[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float sum = WIDE ? l[r].x + l[r].y : r ? l[0].y : l[0].x, m = ref[r] == -CUDART_INF_F ? ref[r] : ref[r] - LIFT;
#pragma unroll
      for (int o = WIDE ? 1 : 4; o < (WIDE ? 4 : 32); o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      f_o[r] = Q8 ? settle_sum(m, sum) : 1.f;
      if ((WIDE ? t : g) == 0) ml[warp * RB + (WIDE ? g + 8 * r : 2 * t + r)] = make_float2(m, sum);
    }
#pragma unroll
    for (int n = 0; n < NO * E / 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[(warp * RB + row_of(i)) * OS + dim_of(n, i)] = Q8 ? o[n][i] * f_o[WIDE ? i >> 1 : i & 1] : o[n][i];
    __syncthreads();
    const int live = min(RB, a.rows - rb * RB);
    for (int i = threadIdx.x; i < live * (D / 4); i += NT) {
      const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
      float m = -CUDART_INF_F;
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, ml[w * RB + r].x);
      const float use = m == -CUDART_INF_F ? 0.f : m;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float2 e = ml[w * RB + r];
        const float f = exp2f(e.x - use);
        const float4 y = *reinterpret_cast<const float4*>(acc + (w * RB + r) * OS + d);
        x.x = fmaf(f, y.x, x.x); x.y = fmaf(f, y.y, x.y); x.z = fmaf(f, y.z, x.z); x.w = fmaf(f, y.w, x.w);
        sum = fmaf(f, e.y, sum);
      }
      if (pc.whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int64_t out_row = (int64_t)h * a.rows + rb * RB + r;
        T* out = static_cast<T*>(p.out) + (int64_t)b * p.o_sb + out_row * p.o_sr + d;
        out[0] = from_float<T>(x.x * inv); out[1] = from_float<T>(x.y * inv);
        out[2] = from_float<T>(x.z * inv); out[3] = from_float<T>(x.w * inv);
      } else {
        *reinterpret_cast<float4*>(a.part_o + (pc.id * RB + r) * D + d) = x;
        if (d == 0) a.part_ml[pc.id * RB + r] = make_float2(m, sum);
      }
    }
    __syncthreads();       // the ring is free for the next piece
  }
}

template <typename T, int CODE, int D, int TERMS, int RB>
int launch(const Args& a, cudaStream_t st) {
  auto kern = stream_kernel<T, CODE, D, TERMS, RB>;
  constexpr int smem = NW * STAGES * Shape<T, CODE, D>::STAGE + TERMS * Shape<T, CODE, D>::FRAGS + 16 * (int)sizeof(float);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return XKV_ERR_LAUNCH;
  }
  kern<<<(unsigned)a.grid, NT, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? XKV_OK : XKV_ERR_LAUNCH;
}
template <typename T, int CODE, int TERMS>
int by_shape(const Args& a, cudaStream_t st) {
  if (a.p.head_dim == 128) return a.block_rows == 8 ? launch<T, CODE, 128, TERMS, 8>(a, st) : launch<T, CODE, 128, TERMS, 16>(a, st);
  return a.block_rows == 8 ? launch<T, CODE, 64, TERMS, 8>(a, st) : launch<T, CODE, 64, TERMS, 16>(a, st);
}
template <typename T, int TERMS>
int by_code(const Args& a, cudaStream_t st) {
  return a.p.cache_code == XKV_CACHE_INT8 ? by_shape<T, XKV_CACHE_INT8, TERMS>(a, st) : by_shape<T, XKV_CACHE_E4M3, TERMS>(a, st);
}

bool rows_aligned(const void* ptr, int64_t sb, int64_t sh, int64_t sl, int es) {
  return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0 && sb * es % 16 == 0 && sh * es % 16 == 0 && sl * es % 16 == 0;
}

}  // namespace

}  // namespace tree

bool tree_stream_supported(const xkv_tree_params& p) {
  if (p.head_dim != 128 && p.head_dim != 64) return false;
  const int es = p.cache_code == XKV_CACHE_DENSE ? 2 : 1;
  if (p.cache_code == XKV_CACHE_DENSE && p.dtype == XKV_F32) return false;
  if (!tree::rows_aligned(p.k, p.k_sb, p.k_sh, p.k_sl, es) || !tree::rows_aligned(p.v, p.v_sb, p.v_sh, p.v_sl, es)) return false;
  if (p.cache_code != XKV_CACHE_DENSE &&
      ((reinterpret_cast<uintptr_t>(p.k_scales) & 3u) || (reinterpret_cast<uintptr_t>(p.v_scales) & 3u)))
    return false;
  return true;
}

void tree_stream_plan(const xkv_tree_params& p, TreePlan* pl) {
  pl->kernel = TreePlan::kStream;
  pl->name = "stream";
  pl->block_rows = pl->rows <= 8 ? 8 : 16;
  pl->unit_tokens = tree::NW * tree::HALF / (p.head_dim * (p.cache_code == XKV_CACHE_DENSE ? 2 : 1));
  pl->slots = device_sm_count();
  // A short cache is one unit, so that no strip is cut and nothing has to be merged: up to LAUNCH tiles in a row cost a
  // block about what the merge and its launch cost the call (777 int8 rows, 4 tiles: 18.4 -> 15.2 us per queued call; 1023
  // bf16 rows, 8 tiles: 17.0 -> 14.4; a call that is waited for, 30 -> 33).
  constexpr int LAUNCH = 8;
  const int tiles = ceil_div(p.kv_len, pl->unit_tokens);
  const int64_t strips = (int64_t)p.batch * p.num_kv_heads * ceil_div(pl->rows, pl->block_rows);
  if (tiles <= LAUNCH && strips <= pl->slots && p.num_splits == 0) pl->unit_tokens *= tiles;
}

int tree_stream_decode(const tree::Args& a, cudaStream_t st) {
  using namespace tree;
  if (a.p.cache_code == XKV_CACHE_DENSE)
    return a.p.dtype == XKV_BF16 ? by_shape<__nv_bfloat16, XKV_CACHE_DENSE, 1>(a, st) : by_shape<__half, XKV_CACHE_DENSE, 1>(a, st);
  if (a.p.dtype == XKV_BF16) return by_code<__nv_bfloat16, 1>(a, st);
  if (a.p.dtype == XKV_F16) return by_code<__half, 1>(a, st);
  return by_code<float, 2>(a, st);
}

}  // namespace xkv
