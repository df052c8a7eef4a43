// kv4.cu -- the 4-bit key/value cache (include/ork_b200.h): rows into it and back, and attention of the last
// tokens of each sequence over it.
//
// A value is code * step + lowest with one (step, lowest) pair of fp16 for each 64 dims of a token's head.
#include <cuda_runtime.h>

#define ORK_F16_AS_U16  // nvcc cannot compile expressions of the header's _Float16; the ABI is the same

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "elem.cuh"
#include "errword.cuh"
#include "ork_internal.h"
#include "ork_structs.h"
#include "sm100.cuh"

namespace orkb {

__device__ unsigned int g_kv4_error = 0;

namespace {

constexpr int kGroup = 64;  // dims that share a step and a lowest value

__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

__device__ __forceinline__ void kv4_error() {
  atomicOr(&g_kv4_error, 1u);
  err_word_set();
}

// ---- rows into the cache and back ------------------------------------------------------------------------------
// A storing thread handles 16 consecutive dims of k or of v of one row and head, two 32-bit words of codes: a group's 4
// threads find its lowest and largest value with two shuffles, and dk / 8 threads read and write a token's k and v of a
// head whole; its next row is on the way as it lies in memory. A reading-back thread handles one word, four rows at a
// time. A warp keeps its heads and steps through the rows of its sequence (blockIdx.y).
// The division by the step, which has to be the IEEE one for the codes to be the definition's, is a product with the
// step's reciprocal wherever that is sure to round to the same code, and is done again where it is not (a quotient within
// 1e-5 of the middle between two codes; the product is off by 6e-6 at most).
// 49145 rows of 8 heads of 128 bf16 dims: the store reads 201 MB and writes 57 MB in 70 us, 3.7 TB/s, bound by its
// instructions (75 % of the issue slots: lowest, largest, quotients); the load back 46 us, 5.5 TB/s, bound by memory.
constexpr int kRowThreads = 256;
constexpr int kStoreWords = 2;  // words of codes that a storing thread makes; one: 84 us instead of 70

struct Rows {
  int nseq, Hkv, cap, rows;
  long long ts, hs;
  const int *start, *pos;
};

// eight values at p, with 16-byte accesses where the caller found them aligned
__device__ __forceinline__ float2 widen2(uint32_t w, const __half *) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ float2 widen2(uint32_t w, const __nv_bfloat16 *) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t narrow2(float x, float y, const __half *) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t narrow2(float x, float y, const __nv_bfloat16 *) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <class E>
struct Raw8 {  // eight values as they lie in memory
  uint32_t w[2 * sizeof(E)];
};
template <class E>
__device__ __forceinline__ void load8(const E *p, bool vec, Raw8<E> &x) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; i++) {
      const uint4 a = reinterpret_cast<const uint4 *>(p)[i];
      x.w[4 * i] = a.x, x.w[4 * i + 1] = a.y, x.w[4 * i + 2] = a.z, x.w[4 * i + 3] = a.w;
    }
  } else if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int i = 0; i < 8; i++) x.w[i] = __float_as_uint(p[i]);
  } else {
    const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
    for (int i = 0; i < 4; i++) x.w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
  }
}
template <class E>
__device__ __forceinline__ void widen8(const Raw8<E> &r, float *x) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(E) * 2; i++) {
    if constexpr (sizeof(E) == 4) {
      x[i] = __uint_as_float(r.w[i]);
    } else {
      const float2 f = widen2(r.w[i], (const E *)nullptr);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}
template <class E>
__device__ __forceinline__ void load8(const E *p, bool vec, float (&x)[8]) {
  Raw8<E> r;
  load8(p, vec, r);
  widen8(r, x);
}
template <class E>
__device__ __forceinline__ void store8(E *p, bool vec, const float (&x)[8]) {
  if (vec) {
    if constexpr (sizeof(E) == 4) {
      *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<uint4 *>(p) = make_uint4(narrow2(x[0], x[1], p), narrow2(x[2], x[3], p), narrow2(x[4], x[5], p),
                                                 narrow2(x[6], x[7], p));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) p[i] = from_f32<E>(x[i]);
  }
}

__device__ __forceinline__ float min_nan(float a, float b, float c) {  // NaN if any is
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <class E, int DK, bool STORE, bool VEC>
__global__ void __launch_bounds__(kRowThreads, STORE ? 4 : 1) kv4_rows_kernel(Rows r, E *k, E *v, uint32_t *kc, uint32_t *vc,
                                                               __half2 *kp, __half2 *vp) {
  constexpr int WORDS = DK / 8, NW = STORE ? kStoreWords : 1;  // words of a row, of a thread
  constexpr int LANES = 2 * WORDS / NW;                             // threads of a (row, head): k's, then v's
  const int s = blockIdx.y, lane = threadIdx.x & 31;
  const int row0 = r.start ? r.start[s] : s * r.rows;
  const int n = r.start ? r.start[s + 1] - row0 : r.rows;
  const int slot0 = r.pos ? r.pos[s] : 0;
  // teams of LANES threads: team i takes head i % Hkv and every `step`-th row from i / Hkv on
  const int teams = gridDim.x * (kRowThreads / LANES), step = teams / r.Hkv;
  const int team = (blockIdx.x * kRowThreads + threadIdx.x) / LANES, h = team % r.Hkv, t0 = team / r.Hkv;
  const int at = threadIdx.x % LANES, w = at * NW % WORDS;
  const bool is_v = at * NW >= WORDS;
  if (t0 >= step) return;  // whole teams; a group's threads stay together
  if (n < 0 || row0 < 0) {  // offsets that decrease, or begin before the rows
    if (at == 0) kv4_error();
    return;
  }
  // the rows whose slots the cache has
  const long long first = slot0 < 0 ? -(long long)slot0 : 0, end = (long long)r.cap - slot0;
  const int last = (int)max(0LL, min((long long)n, end));
  if (at == 0 && (t0 < min((long long)n, first) || n > last)) kv4_error();
  int t = t0;
  if (t < first) t += (int)((min(first, (long long)n) - t + step - 1) / step) * step;
  const long long hop = (long long)step * r.ts;
  E *row = (is_v ? v : k) + ((long long)row0 + t) * r.ts + (long long)h * r.hs + 8 * w;
  const size_t tok = ((size_t)s * r.Hkv + h) * r.cap + (size_t)((long long)slot0 + t);
  uint32_t *code = (is_v ? vc : kc) + tok * WORDS + w;
  __half2 *par = (is_v ? vp : kp) + tok * (DK / kGroup) + w / 8;
  constexpr int GROUP = 8 / NW;  // threads of a group of 64 dims
  const unsigned mask = ((1u << GROUP) - 1) << (lane & ~(GROUP - 1));
  Raw8<E> next[NW];
  if constexpr (!STORE) {  // four rows at a time on their way: a row is little to ask for
    for (; t < last; t += 4 * step, row += 4 * hop, code += 4 * step * WORDS, par += 4 * step * (DK / kGroup)) {
      uint32_t c[4];
      __half2 p[4];
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (t + u * step < last) c[u] = code[(long long)u * step * WORDS], p[u] = par[(long long)u * step * (DK / kGroup)];
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (t + u * step < last) {
          const float2 f = __half22float2(p[u]);
          float x[8];
          // code * step is exact in fp32: one rounding either way
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = fmaf(__uint_as_float(0x4b000000u | ((c[u] >> (4 * i)) & 15u)) - 8388608.0f, f.x, f.y);
          store8<E>(row + u * hop, VEC, x);
        }
    }
    return;
  }
  if (STORE && t < last)
#pragma unroll
    for (int u = 0; u < NW; u++) load8<E>(row + 8 * u, VEC, next[u]);
  for (; t < last; t += step, row += hop, code += step * WORDS, par += step * (DK / kGroup)) {
    float x[NW][8];
    if constexpr (STORE) {
      widen8(next[0], x[0]);
      float lo = x[0][0], hi = lo;
#pragma unroll
      for (int u = 0; u < NW; u++) {
        if (u) widen8(next[u], x[u]);
        if (t + step < last) load8<E>(row + hop + 8 * u, VEC, next[u]);
#pragma unroll
        for (int i = 0; i < 8; i += 2) lo = min_nan(lo, x[u][i], x[u][i + 1]), hi = max_nan(hi, x[u][i], x[u][i + 1]);
      }
#pragma unroll
      for (int o = 1; o < GROUP; o <<= 1) {
        const float l2 = __shfl_xor_sync(mask, lo, o), h2 = __shfl_xor_sync(mask, hi, o);
        lo = min_nan(lo, l2, l2);
        hi = max_nan(hi, h2, h2);
      }
      // every operation rounds on its own, so that any IEEE implementation of the formulas gives these bits
      __half step2 = __float2half_rn(fminf(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f), 65504.0f));
      __half low = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
      if (!(fabsf(lo) <= 3.402823466e38f && fabsf(hi) <= 3.402823466e38f)) step2 = low = __ushort_as_half((unsigned short)0x7fff);
      const float sf = __half2float(step2), lf = __half2float(low);
      float inv = 0.0f;  // no step, no codes
      if (sf > 0.0f) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(sf * 15.0f));
      uint32_t c[NW];
#pragma unroll
      for (int u = 0; u < NW; u++) {
        using namespace sm100;
        const float2 two23 = both(8388608.0f);
        float off = 0.0f, r4[8];
        float2 m[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          // the quotient over 15 clamped to [0, 1]; m: the code plus 2^23, rounded to an integer by that addition
          const float2 d = add2(make_float2(x[u][2 * i], x[u][2 * i + 1]), both(-lf));
          const float2 q = make_float2(__saturatef(d.x * inv), __saturatef(d.y * inv));
          m[i] = fma2(q, both(15.0f), two23);
          const float2 z = add2(m[i], both(-8388608.0f));
          const float2 e = fma2(q, both(-15.0f), z);
          off = fmaxf(off, fmaxf(fabsf(e.x), fabsf(e.y)));
          r4[2 * i] = z.x, r4[2 * i + 1] = z.y;
        }
        // four codes side by side in the low bits of 2^23 + c0 + 16 c1 + 256 c2 + 4096 c3
        const float a = fmaf(r4[3], 4096.0f, fmaf(r4[2], 256.0f, fmaf(r4[1], 16.0f, m[0].x)));
        const float b = fmaf(r4[7], 4096.0f, fmaf(r4[6], 256.0f, fmaf(r4[5], 16.0f, m[2].x)));
        c[u] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x5410);
        if (off > 0.49999f) {
          c[u] = 0;
#pragma unroll 1
          for (int i = 0; i < 8; i++) {
            float y = x[u][0];
#pragma unroll
            for (int j = 1; j < 8; j++) y = i == j ? x[u][j] : y;
            c[u] |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(y, lf), sf)), 0.0f), 15.0f) << (4 * i);
          }
        }
      }
      if constexpr (NW == 2) *reinterpret_cast<uint2 *>(code) = make_uint2(c[0], c[1]);
      else *code = c[0];
      if ((w & 7) == 0) *par = __halves2half2(step2, low);
    }
  }
}

// ---- attention over the cache ----------------------------------------------------------------------------------
// With s_j, b_j the step and lowest value of token j (per 64 dims g) and c_j its codes,
//   q . k_j = sum_g s_jg (q_g . c_jg) + b_jg sum(q_g),   out = sum_j p_j v_j = sum_j (p_j s_jg) c_jg + sum_j p_j b_jg,
// so the codes enter the matrix instructions as integers and are never dequantized. They are the 16-row operand of
// the instructions (16 tokens of k, then 16 dims of v) and the query rows the 8 columns: a decode step has no more
// rows than that per kv head, and the other way round half of each product would be padding.
// First product, mma.m16n8k32 of 8-bit integers: an AND takes four codes out of a word. q is scaled per row to
// integers below 2^21 and split into three signed bytes; the three products run one after another, the sums shifted
// left by eight between them, and stay below 2^31: the logits carry q's 21 bits and no other error. fp32 queries have a
// fourth byte, summed by itself: 29 bits, so that a dim keeps fp32's digits next to one 32 times larger, and 22 bits
// next to one 128 times larger (a dim of 200 among dims of 1.6: outputs off by 3e-6, 4e-5 with three bytes). (A code in the
// low bits of an fp16 is an exact subnormal too, and one instruction fewer; but the tensor cores align what they add
// by the nominal exponents, and the leading zeros cost 6 to 10 of their 24 bits: logits were off by 2^-15.)
// Second product, mma.m16n8k16 of fp16: the output has no more than 11 bits either. A shift and two ANDs put two nibbles
// of each 16-bit half into the mantissa, as the subnormals code * 2^-22 and code * 2^-18, and the scales are taken out of
// the sums at the end. (Left where the byte has them, a shift less, 131071 tokens came out off by 6e-4 instead of
// 2.7e-4.) p * step, rounded to fp16, is transposed between the products with movmatrix. For fp32 queries (SPLIT) it is
// split into an fp16 and the fp16 of what that leaves, 22 bits together, the product runs twice, and every code is shifted
// to the top of the mantissa, code * 2^-18.
// What keeps p * step in fp16's range: the steps of each group of 64 dims are scaled by a power of two, the one that
// brings the largest of the warp's first stage to 1 at least and less than 2; and a row's p is 2^(x - m) for an m that
// follows not the largest logit but the largest p * step, the logit plus the exponent of the token's larger scaled step.
// So the row's largest p * step lies between 2^(kTop - 6) and 2^15 in one group at least. What is 2^-16 of it, and more,
// is rounded to 11 bits (what is 2^-5 of it, and more, to 22), and smaller ones to 2^-27 of it: a token of large steps
// that has no weight costs the others no digits, nor does a group of large steps the other group. With one scale of both
// groups, by the largest step of the warp's tokens, a group of steps 10^4 times smaller was off by 6e-4 instead of 3e-7
// (fp32 queries), and 32768 tokens 19 nats below another one by 7e-2 instead of 3e-6.
// The codes of v are not negative although v has no sign: their sum would grow far above the output that it is to
// leave after the lowest values' share is added, and the tensor cores truncate what they add. So each stage ends
// with 8 * sum(p * step) taken out again (the sum by a product with ones, so that it holds the rounded p * step), and
// v is (c - 8) s + (b + 8 s). For fp32 queries the truncation shows all the same: it makes every unit's sum a little
// smaller. There every other unit counts down, with -p * step and codes 15 - c, so that what one unit loses the next
// brings back, and 7.5, the middle of the codes, is taken out: 131071 tokens came out off by 1.5e-6 to 2e-6 without,
// 0.8e-6 to 1.1e-6 with it, 4000 tokens by 0.7e-6 and 0.5e-6. (16-bit queries would lose 5 % of their speed to it.)
//
// Bound by the instructions on the codes: 17.9 a token and kv head, issue slots 60 % and the tensor pipe 37 % used, at
// 5.0 to 5.3 TB/s of cache (55 x 8 heads of 16384 bf16 tokens, 8 rows each: 196 us; the copies alone run at 6.4 TB/s).
// fp32 queries, 32 sequences of 8192 tokens, 64/8 heads of 128: 96 us.
// Stages are requested by one elected lane at addresses that are the same in a warp by construction (uniform
// registers): 13 % faster than a lane picked by its number.
//
// A warp owns a run of 16-token units and brings kStageUnits of them at a time into its own ring of shared memory
// with bulk copies (codes and parameters of k and v, contiguous); no other warp waits on it. The parameters are
// widened to fp32 once per stage (each token's are needed by four lanes). Softmax is kept online per stage. The warps
// of a CTA, then the CTAs of a (sequence, kv head, row tile) -- its tokens are split over gridDim.x -- are joined in a
// fixed order, so results do not depend on timing.
//
// Lane layout (r = lane / 4, c = lane % 4). First product: row m of a unit is token (m & 7) / 2 + 4 (m & 1) + 8 (m / 8),
// contraction quadruples are the dims (e, e + 2, e + 4, e + 6) that one AND leaves, column r is query row r of q's
// fragment; the accumulators are rows 2 c and 2 c + 1 at the tokens of m = r and r + 8. Second product: contraction pairs are the
// tokens (c, c + 4) and (c + 8, c + 12), put side by side by a byte permutation; row r of a tile (g, j) is dim
// 64 g + 8 r + 2 j, row r + 8 the dim after it. This order of the tokens keeps both reads of codes to two-way bank
// conflicts (64-byte rows; four consecutive tokens where the plain order would read every other one).
constexpr int kWarps = 4;   // per CTA
constexpr int kUnit = 16;   // tokens
constexpr int kStageUnits = 3;
constexpr int kStageTok = kUnit * kStageUnits;
constexpr int kRows = 8;    // query rows of a column tile
// m only follows the running maximum of p * step (log2) once that is kTop + kRise above it, and then to kTop below it:
// most stages raise the maximum of some of the eight rows a little, and scaling the accumulators for that was a fifth of
// the instructions.
constexpr float kTop = 8.0f, kRise = 5.0f;
// Scaled steps between these count as 1 in the maximum, and nearly all are: a stage of none but those takes the maximum of
// the logits alone (0.6 % of the time of a full batch went to the test, 7 % to the exact maximum in every stage). With them
// p * step reaches 2^(kTop + kRise) * 4 = 2^15.
constexpr float kOddBelow = 0x1p-6f, kOddAbove = 4.0f;
constexpr int kNoStep = -60;  // log2 of the step that a token of smaller steps counts as, so that p stays finite

struct Attn4 {
  const uint8_t *kc, *vc;
  const __half *kp, *vp;
  int nseq, Hkv, cap, H, T, window, sinks, max_len;
  int row_T, late;  // rows of q and out from one sequence to the next; tokens held that come after the T ones
  long long q_ts, q_hs;
  const int *len;
  float scale;
  float *wsum;
  int splits, tiles, prow;  // token splits; row tiles, and their rows in all
  bool qvec;          // q's rows are 16-byte aligned
  bool join;          // the last CTA of an item joins its splits
  unsigned int *done; // [nseq * Hkv * tiles] counts of finished splits, zero between launches
  int vis;            // most tokens that a row range can see, a multiple of kUnit (x's row stride)
  float *po;          // partial outputs [nseq][Hkv][prow][splits][dk], normalised by nothing
  float2 *pml;        // their maxima (log2 units) and sums [nseq][Hkv][prow][splits]
  float *stat;        // m + log2(sum) of every row [nseq][Hkv][prow], for wsum
  float *x;           // logits in log2 units [nseq][Hkv][prow][vis], kept for wsum
};

// The visible tokens of a sequence as 16-token units: su units of sinks from token 0 on, then the window's.
struct Units {
  int n, su, lo, all;  // tokens held; sink units; first unit of the window; units in all
};
__device__ __forceinline__ Units units_of(const Attn4 &a, int n) {
  Units u;
  u.n = n;
  const int first = a.window && n - a.T - a.window + 1 > 0 ? n - a.T - a.window + 1 : 0;
  u.lo = first / kUnit;
  u.su = min((a.sinks + kUnit - 1) / kUnit, u.lo);
  u.all = u.su + (n + kUnit - 1) / kUnit - u.lo;
  return u;
}
__device__ __forceinline__ int token_of(const Units &u, int unit) {
  return (unit < u.su ? unit : unit - u.su + u.lo) * kUnit;
}

// the number of tokens of sequence s up to the last of T; 0 (reported) where it cannot be
__device__ __forceinline__ int seq_len(const Attn4 &a, int s) {
  const int n = a.len[s];
  if (n >= 0 && n <= a.max_len) return max(n - a.late, 0);
  if (threadIdx.x == 0) kv4_error();
  return 0;
}
__device__ __forceinline__ bool visible(const Attn4 &a, int p, int j) {
  return j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
}

// d += a b: fp16, 16 x 8 x 16; mma0: d = a b. mma_i8: unsigned times signed bytes, 16 x 8 x 32
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_i8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_i80(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
// byte i of each of four words
__device__ __forceinline__ uint32_t bytes_of(const int (&w)[4], int i) {
  const uint32_t sel = (uint32_t)(i | (i + 4) << 4);
  return __byte_perm(__byte_perm((uint32_t)w[0], (uint32_t)w[1], sel), __byte_perm((uint32_t)w[2], (uint32_t)w[3], sel), 0x5410);
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // an 8 x 8 tile of 16-bit values
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// x as fp16 pairs: the rounded values, and what they leave
__device__ __forceinline__ void split2(float2 x, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __float22half2_rn(x);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x.x - f.x, x.y - f.y);
  hi = *reinterpret_cast<const uint32_t *>(&h);
  lo = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ float quad_max(float v) {  // over c
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float col_max(float v) {  // over r
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float col_sum(float v) {
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// the power of two 2^e
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

template <int DK>
struct Stage {  // one ring slot of a warp
  uint8_t k[kStageTok * DK / 2], v[kStageTok * DK / 2];
  __half2 kp[kStageTok * (DK / kGroup)], vp[kStageTok * (DK / kGroup)];
};
// A stage's parameters in fp32: of each token the steps of its groups, then the lowest values (k), or the scaled steps
// and b + kMid s (v).
template <int DK>
struct Wide {
  float k[kStageTok][2 * (DK / kGroup)], v[kStageTok][2 * (DK / kGroup)];
};
template <int DK>
constexpr int kStages = DK == 128 ? 2 : 4;
// CTAs that an SM holds: with both halves of p * step, or two column tiles, the registers of three would spill
template <class E, int DK, int NT>
constexpr int kCtas = DK == 128 && (NT == 2 || sizeof(E) == 4) ? 2 : 3;
// q of a CTA: its bytes in the order the first product takes them, and the scales and sums of its rows
template <class E>
constexpr int kDigits = sizeof(E) == 4 ? 4 : 3;
template <class E, int DK, int NT>
struct Query {
  uint4 d[NT][kDigits<E>][DK / kGroup][32];
  float f[NT * kRows], sum[DK / kGroup][NT * kRows];
};
template <class E, int DK, int NT>
constexpr int kAttnSmem = kWarps * (kStages<DK> * ((int)sizeof(Stage<DK>) + 8) + (int)sizeof(Wide<DK>)) + (int)sizeof(Query<E, DK, NT>);

template <int N>
__device__ __forceinline__ void load_pars(const float *p, float (&x)[N]) {
  if constexpr (N == 4) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const float2 v = *reinterpret_cast<const float2 *>(p);
    x[0] = v.x, x[1] = v.y;
  }
}
template <int N>
__device__ __forceinline__ void store_pars(float *p, const float (&x)[N]) {
  if constexpr (N == 4) *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
  else *reinterpret_cast<float2 *>(p) = make_float2(x[0], x[1]);
}
// the NG parameter pairs (step, lowest) of a token
template <int NG>
__device__ __forceinline__ void token_pars(const __half2 *p, float2 (&x)[NG]) {
  if constexpr (NG == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    x[0] = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
    x[1] = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
  } else {
    x[0] = __half22float2(*p);
  }
}

template <int DK>
__device__ __forceinline__ void load_stage(const Attn4 &a, size_t base, const Units &u, int unit, int cnt, Stage<DK> *st,
                                           uint32_t bar) {
  constexpr int NG = DK / kGroup;
  const size_t tok = base + (size_t)token_of(u, unit);
  const uint32_t cb = (uint32_t)cnt * kUnit * (DK / 2), pb = (uint32_t)cnt * kUnit * NG * 4;
  if (sm100::elect_one()) {
    sm100::bar_expect(bar, 2 * cb + 2 * pb);
    sm100::bulk_load(sm100::smem_addr(st->k), a.kc + tok * (DK / 2), cb, bar);
    sm100::bulk_load(sm100::smem_addr(st->kp), a.kp + tok * NG * 2, pb, bar);
    sm100::bulk_load(sm100::smem_addr(st->v), a.vc + tok * (DK / 2), cb, bar);
    sm100::bulk_load(sm100::smem_addr(st->vp), a.vp + tok * NG * 2, pb, bar);
  }
  __syncwarp();
}

// NT column tiles of kRows query rows share every operand made from the codes.
template <class E, int DK, int NT, bool WS>
__global__ void __launch_bounds__(32 * kWarps, kCtas<E, DK, NT>) kv4_attn_kernel(const Attn4 a, const E *__restrict__ q, E *__restrict__ out) {
  constexpr int NG = DK / kGroup, NST = kStages<DK>, TR = NT * kRows;
  constexpr bool SPLIT = sizeof(E) == 4;
  constexpr int ND = kDigits<E>;
  constexpr float kMid = SPLIT ? 7.5f : 8.0f;  // what the codes of v are taken from
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // known to be the same for the whole warp
  const int split = blockIdx.x % a.splits, th = blockIdx.x / a.splits, kvh = th / a.tiles, tile = th % a.tiles;
  const int s = blockIdx.y, G = a.H / a.Hkv, rows = a.T * G;
  Stage<DK> *ring = reinterpret_cast<Stage<DK> *>(smem) + warp * NST;
  Wide<DK> *wide = reinterpret_cast<Wide<DK> *>(smem + kWarps * NST * sizeof(Stage<DK>)) + warp;
  Query<E, DK, NT> *qm = reinterpret_cast<Query<E, DK, NT> *>(smem + kWarps * (NST * sizeof(Stage<DK>) + sizeof(Wide<DK>)));
  const uint32_t bars = sm100::smem_addr(qm + 1) + warp * NST * 8;
  // q of row r of tile y, by warp y: on its way while the sequence's length is read
  float qx[NG][16];
  if (warp < NT) {
    const int row = tile * TR + warp * kRows + r;
    const E *qr = q + ((long long)s * a.row_T + row / G) * a.q_ts + (long long)(kvh * G + row % G) * a.q_hs + 16 * c;
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
      for (int i = 0; i < 16; i++) qx[g][i] = 0.0f;
    if (row < rows) {
      auto load = [&](auto vec) {
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
          for (int i = 0; i < 16; i += 8) load8<E>(qr + 64 * g + i, decltype(vec)::value, *reinterpret_cast<float(*)[8]>(&qx[g][i]));
      };
      if (a.qvec) load(std::true_type());
      else load(std::false_type());
    }
  }
  if (lane < NST) sm100::bar_init(bars + 8 * lane, 1);
  sm100::bar_init_fence();
  __syncwarp();

  const int n = sm100::uniform(seq_len(a, s));
  const Units u = units_of(a, n);
  const int cu0 = (int)((long long)u.all * split / a.splits), cu1 = (int)((long long)u.all * (split + 1) / a.splits);
  const int u0 = cu0 + (cu1 - cu0) * warp / kWarps, u1 = cu0 + (cu1 - cu0) * (warp + 1) / kWarps;
  const size_t base = ((size_t)s * a.Hkv + kvh) * a.cap;
  // a stage ends at the jump from the sinks to the window
  auto count = [&](int unit) { return min(min(kStageUnits, u1 - unit), unit < u.su ? u.su - unit : kStageUnits); };
  int next = u0;  // first unit not yet requested
#pragma unroll
  for (int i = 0; i < NST; i++)
    if (next < u1) {
      const int cnt = count(next);
      load_stage<DK>(a, base, u, next, cnt, ring + i, bars + 8 * i);
      next += cnt;
    }

  // as integers: byte ND - 1 - d of those of the lane's words, even dims then odd ones
  if (warp < NT) {
    const int y = warp;
    float mx = 0.0f;
    bool fin = true;
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        mx = fmaxf(mx, fabsf(qx[g][i]));
        fin = fin && fabsf(qx[g][i]) <= 3.402823466e38f;
      }
    mx = quad_max(mx);
    const unsigned quad = 15u << (lane & 28);
    fin = (__ballot_sync(0xffffffffu, fin) & quad) == quad;
    const int e = fin ? min(100, 123 + 8 * ND - (int)(__float_as_uint(mx) >> 23)) : 0;  // -107 at least
    const float up = pow2(e), f = fin ? a.scale * 1.4426950408889634f * pow2(-e) : __int_as_float(0x7fc00000);
    if (c == 0) qm->f[y * kRows + r] = f;
#pragma unroll
    for (int g = 0; g < NG; g++) {
      int w[16];
      std::conditional_t<SPLIT, long long, int> sum = 0;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        w[i] = fin ? __float2int_rn(qx[g][i] * up) : 0;
        sum += w[i];
        w[i] = (int)((uint32_t)w[i] + (ND == 4 ? 0x80808080u : 0x808080u));  // bytes of 128 + digit
      }
      const float total = quad_sum((float)sum) * f;
      if (c == 0) qm->sum[g][y * kRows + r] = total;
#pragma unroll
      for (int d = 0; d < ND; d++) {
        auto digit = [&](int i) {
          const int w4[4] = {w[i], w[i + 2], w[i + 4], w[i + 6]};
          return bytes_of(w4, ND - 1 - d) ^ 0x80808080u;
        };
        qm->d[y][d][g][lane] = make_uint4(digit(0), digit(1), digit(8), digit(9));
      }
    }
  }
  __syncthreads();
  float fs[NT][2], qs[NT][NG][2];  // of the rows 2 c and 2 c + 1 that the accumulators hold
#pragma unroll
  for (int y = 0; y < NT; y++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      fs[y][i] = qm->f[y * kRows + 2 * c + i];
#pragma unroll
      for (int g = 0; g < NG; g++) qs[y][g][i] = qm->sum[g][y * kRows + 2 * c + i];
    }

  const uint32_t qaddr = sm100::smem_addr(&qm->d[0][0][0][lane]);
  float o[NT][NG][4][4], z[NT][NG][2], l[NT][2], mrow[NT][2];
#pragma unroll
  for (int y = 0; y < NT; y++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      l[y][i] = 0.0f, mrow[y][i] = -INFINITY;
#pragma unroll
      for (int g = 0; g < NG; g++) {
        z[y][g][i] = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) o[y][g][j][i] = o[y][g][j][i + 2] = 0.0f;
      }
    }
  float vs[NG];  // scales of the groups' steps; 0 until a stage has any
  bool unset = true;
  uint32_t flip = 0;  // all ones: units of even number count down (see above)
#pragma unroll
  for (int g = 0; g < NG; g++) vs[g] = 0.0f;
  bool ok = true;
  int slot = 0;
  uint32_t parity = 0;
  for (int unit = u0; unit < u1;) {
    const int cnt = count(unit), tok0 = token_of(u, unit), tok1 = tok0 + cnt * kUnit;
    const Stage<DK> *st = ring + slot;
    ok = sm100::bar_wait(bars + 8 * slot, parity);
    if (!ok) break;
    // every token of the stage visible to every row?
    const bool whole = cnt == kStageUnits && tok1 <= n - a.T + 1 && (a.window == 0 || tok0 > n - 1 - a.window || tok1 <= a.sinks);
    constexpr int PT = (kStageTok + 31) / 32;
    float vpar[PT][2 * NG];  // of the tokens that this lane widens
#pragma unroll
    for (int i = 0; i < PT; i++) {
      const int tk = lane + 32 * i, j = tok0 + tk;
      if (kStageTok % 32 == 0 || tk < kStageTok) {
        float2 kf[NG], vf[NG];
        token_pars<NG>(st->kp + tk * NG, kf);
        token_pars<NG>(st->vp + tk * NG, vf);
        if (!whole) {
          const bool seen = tk < cnt * kUnit && j < n && (a.window == 0 || j > n - a.T - a.window || j < a.sinks);
#pragma unroll
          for (int g = 0; g < NG; g++)
            if (!seen) kf[g] = vf[g] = make_float2(0.0f, 0.0f);
          // values that are not numbers reach the rows that see the token by the sums of the lowest values: 0 * NaN
          // would reach them all
          const unsigned lanes = kStageTok % 32 == 0 || i + 1 < PT ? 0xffffffffu : (1u << kStageTok % 32) - 1;
#pragma unroll
          for (int g = 0; g < NG; g++) {
            const bool bad = !(fabsf(vf[g].x) <= 1e6f && fabsf(vf[g].y) <= 1e6f);
            if (bad) vf[g] = both(0.0f);
#pragma unroll 1
            for (unsigned at = __ballot_sync(lanes, bad); at; at &= at - 1)
#pragma unroll
              for (int y = 0; y < NT; y++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                  if (visible(a, n - a.T + (tile * TR + y * kRows + 2 * c + h) / G, tok0 + 32 * i + __ffs(at) - 1))
                    z[y][g][h] = __int_as_float(0x7fc00000);
          }
        }
        float kpar[2 * NG];
#pragma unroll
        for (int g = 0; g < NG; g++) {
          kpar[g] = kf[g].x, kpar[NG + g] = kf[g].y;
          vpar[i][g] = vf[g].x, vpar[i][NG + g] = fmaf(kMid, vf[g].x, vf[g].y);
        }
        store_pars(wide->k[tk], kpar);
      }
    }
    if (unset) {
      unset = false;
#pragma unroll
      for (int g = 0; g < NG; g++)
        if (vs[g] == 0.0f) {
          float top = 0.0f;
#pragma unroll
          for (int i = 0; i < PT; i++)
            if (kStageTok % 32 == 0 || lane + 32 * i < kStageTok) top = fmaxf(top, fabsf(vpar[i][g]));
          const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
          if (bits && bits < 0x7f800000u) vs[g] = pow2(127 - (int)(bits >> 23));
          else unset = true;
        }
    }
    const uint32_t down = SPLIT ? (flip ^ (lane & 16 ? ~0u : 0u)) & 0x80000000u : 0u;  // the sign of the lane's tokens' units
    float top[PT];  // the tokens' larger steps
#pragma unroll
    for (int i = 0; i < PT; i++) {
      const int tk = lane + 32 * i;
      top[i] = top[0];
      if (kStageTok % 32 == 0 || tk < kStageTok) {
#pragma unroll
        for (int g = 0; g < NG; g++) vpar[i][g] *= __uint_as_float(__float_as_uint(vs[g]) ^ down);
        store_pars(wide->v[tk], vpar[i]);
        top[i] = fmaxf(fabsf(vpar[i][0]), fabsf(vpar[i][NG - 1]));
      }
    }
    float most = top[0], least = top[0];
#pragma unroll
    for (int i = 1; i < PT; i++) most = fmaxf(most, top[i]), least = fminf(least, top[i]);
    bool odd = most > kOddAbove || least < kOddBelow;
    if (!whole) {  // of the tokens that the stage has
      odd = false;
#pragma unroll
      for (int i = 0; i < PT; i++) {
        const int tk = lane + 32 * i;
        odd = odd || (tk < cnt * kUnit && tok0 + tk < n && !(top[i] >= kOddBelow && top[i] <= kOddAbove));
      }
    }
    __syncwarp();

    float x[NT][kStageUnits][4];  // logits of row 2 c + i % 2 at the token of m = r + 8 (i / 2), in log2 units
    const int mt = (r >> 1) + 4 * (r & 1);
#pragma unroll
    for (int w = 0; w < kStageUnits; w++) {  // units past cnt hold old codes, and steps of zero
      int acc[NT][NG][4], low[SPLIT ? NT : 1][NG][4];  // of the first three digits; of the fourth
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const uint8_t *kr = st->k + (kUnit * w + mt) * (DK / 2) + g * 32 + c * 8;
        const uint2 k0 = *reinterpret_cast<const uint2 *>(kr), k1 = *reinterpret_cast<const uint2 *>(kr + 8 * (DK / 2));
        const uint32_t af[2][4] = {
            {k0.x & 0x0f0f0f0fu, k1.x & 0x0f0f0f0fu, (k0.x >> 4) & 0x0f0f0f0fu, (k1.x >> 4) & 0x0f0f0f0fu},
            {k0.y & 0x0f0f0f0fu, k1.y & 0x0f0f0f0fu, (k0.y >> 4) & 0x0f0f0f0fu, (k1.y >> 4) & 0x0f0f0f0fu}};
#pragma unroll
        for (int y = 0; y < NT; y++)
#pragma unroll
          for (int d = 0; d < ND; d++) {
            uint32_t qb[4];  // kept in shared memory, the registers are full
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(qb[0]), "=r"(qb[1]), "=r"(qb[2]), "=r"(qb[3])
                         : "r"(qaddr + (uint32_t)(((y * ND + d) * NG + g) * 512)));
            if (d == 3) {
              mma_i80(low[SPLIT ? y : 0][g], af[0], qb[0], qb[1]);
              mma_i8(low[SPLIT ? y : 0][g], af[1], qb[2], qb[3]);
              continue;
            }
            if (d == 0) mma_i80(acc[y][g], af[0], qb[0], qb[1]);
            else {
#pragma unroll
              for (int i = 0; i < 4; i++) acc[y][g][i] <<= 8;
              mma_i8(acc[y][g], af[0], qb[0], qb[1]);
            }
            mma_i8(acc[y][g], af[1], qb[2], qb[3]);
          }
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float par[2 * NG];
        load_pars(wide->k[kUnit * w + 8 * h + mt], par);
#pragma unroll
        for (int y = 0; y < NT; y++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            auto dot = [&](int g) {  // q . codes
              const float top = (float)acc[y][g][2 * h + i];
              return SPLIT ? fmaf(top, 256.0f, (float)low[SPLIT ? y : 0][g][2 * h + i]) : top;
            };
            float d = dot(0) * par[0], b = par[NG] * qs[y][0][i];
            if constexpr (NG == 2) {
              d = fmaf(dot(1), par[1], d);
              b = fmaf(par[NG + 1], qs[y][1][i], b);
            }
            x[y][w][2 * h + i] = fmaf(d, fs[y][i], b);
          }
      }
    }
    if (!whole) {
#pragma unroll
      for (int y = 0; y < NT; y++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int p = n - a.T + (tile * TR + y * kRows + 2 * c + i) / G;  // the row's position
#pragma unroll
          for (int w = 0; w < kStageUnits; w++)
#pragma unroll
            for (int h = 0; h < 2; h++)
              if (w >= cnt || !visible(a, p, tok0 + kUnit * w + 8 * h + mt)) x[y][w][2 * h + i] = -INFINITY;
        }
    }
    if constexpr (WS) {
#pragma unroll
      for (int y = 0; y < NT; y++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float *xr = a.x + (((size_t)s * a.Hkv + kvh) * a.prow + tile * TR + y * kRows + 2 * c + i) * a.vis +
                      (size_t)unit * kUnit + mt;
#pragma unroll
          for (int w = 0; w < kStageUnits; w++)
            if (w < cnt) xr[kUnit * w] = x[y][w][i], xr[kUnit * w + 8] = x[y][w][2 + i];
        }
    }
    float mx[NT][2];
    bool rise = false;
    if (!__any_sync(0xffffffffu, odd)) {
#pragma unroll
      for (int y = 0; y < NT; y++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          mx[y][i] = fmaxf(x[y][0][i], x[y][0][2 + i]);
#pragma unroll
          for (int w = 1; w < kStageUnits; w++) mx[y][i] = fmaxf(mx[y][i], fmaxf(x[y][w][i], x[y][w][2 + i]));
        }
    } else {
#pragma unroll
      for (int w = 0; w < kStageUnits; w++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float par[2 * NG];
          load_pars(wide->v[kUnit * w + 8 * h + mt], par);
          const int e = (int)(__float_as_uint(fmaxf(fabsf(par[0]), fabsf(par[NG - 1]))) >> 23);
          const float lt = e < 255 ? (float)max(e - 127, kNoStep) : (float)kNoStep;
#pragma unroll
          for (int y = 0; y < NT; y++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const float v = x[y][w][2 * h + i] + lt;
              mx[y][i] = w + h ? fmaxf(mx[y][i], v) : v;
            }
        }
    }
#pragma unroll
    for (int y = 0; y < NT; y++)
#pragma unroll
      for (int i = 0; i < 2; i++) rise = rise || mx[y][i] > mrow[y][i] + (kTop + kRise);
    if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
      for (int y = 0; y < NT; y++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const float m = fmaxf(mrow[y][i], col_max(mx[y][i]) - kTop), k = mrow[y][i] == m ? 1.0f : sm100::ex2(mrow[y][i] - m);
          mrow[y][i] = m;
          l[y][i] *= k;
#pragma unroll
          for (int g = 0; g < NG; g++) {
            z[y][g][i] *= k;
#pragma unroll
            for (int j = 0; j < 4; j++) o[y][g][j][i] *= k, o[y][g][j][i + 2] *= k;
          }
        }
    }
    float sum[NT][NG][4];  // of p * step, rows 2 c and 2 c + 1 (twice)
    float mu[NT][2];
#pragma unroll
    for (int y = 0; y < NT; y++)
#pragma unroll
      for (int i = 0; i < 2; i++) mu[y][i] = mrow[y][i] == -INFINITY ? 0.0f : mrow[y][i];
#pragma unroll
    for (int w = 0; w < kStageUnits; w++) {
      uint32_t ph[NT][NG][2], pl[SPLIT ? NT : 1][NG][2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float par[2 * NG];
        load_pars(wide->v[kUnit * w + 8 * h + mt], par);
#pragma unroll
        for (int y = 0; y < NT; y++) {
          float e[2], ps[NG][2];
#pragma unroll
          for (int i = 0; i < 2; i++) {
            e[i] = sm100::ex2(x[y][w][2 * h + i] - mu[y][i]);
            l[y][i] += e[i];
#pragma unroll
            for (int g = 0; g < NG; g++) {
              ps[g][i] = e[i] * par[g];
              z[y][g][i] = fmaf(e[i], par[NG + g], z[y][g][i]);
            }
          }
#pragma unroll
          for (int g = 0; g < NG; g++) {
            if constexpr (SPLIT) {
              uint32_t lo;
              split2(make_float2(ps[g][0], ps[g][1]), ph[y][g][h], lo);
              pl[y][g][h] = transpose8(lo);
            } else {
              const __half2 hp = __floats2half2_rn(ps[g][0], ps[g][1]);
              ph[y][g][h] = *reinterpret_cast<const uint32_t *>(&hp);
            }
            ph[y][g][h] = transpose8(ph[y][g][h]);
          }
        }
      }
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const uint32_t one[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
        for (int y = 0; y < NT; y++) {
          if (w == 0) mma0(sum[y][g], one, ph[y][g][0], ph[y][g][1]);
          else mma(sum[y][g], one, ph[y][g][0], ph[y][g][1]);
          if constexpr (SPLIT) mma(sum[y][g], one, pl[y][g][0], pl[y][g][1]);
        }
        uint32_t wv[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
          wv[k] = *reinterpret_cast<const uint32_t *>(st->v + (kUnit * w + 4 * k + c) * (DK / 2) + g * 32 + r * 4);
#pragma unroll
        for (int j = 0; j < 4; j++) {  // dims 2 j and 2 j + 1 of the lane's eight
          const uint32_t sel = j & 2 ? 0x7632u : 0x5410u;
          const uint32_t b0 = __byte_perm(wv[0], wv[1], sel), b1 = __byte_perm(wv[2], wv[3], sel);
          uint32_t af[4];
          if constexpr (SPLIT) {  // to bits 6 .. 9
            const uint32_t f = w & 1 ? ~flip : flip;
            af[0] = ((j & 1 ? b0 >> 2 : b0 << 6) ^ f) & 0x03c003c0u, af[1] = ((j & 1 ? b0 >> 6 : b0 << 2) ^ f) & 0x03c003c0u;
            af[2] = ((j & 1 ? b1 >> 2 : b1 << 6) ^ f) & 0x03c003c0u, af[3] = ((j & 1 ? b1 >> 6 : b1 << 2) ^ f) & 0x03c003c0u;
          } else {
            const uint32_t s0 = j & 1 ? b0 >> 6 : b0 << 2, s1 = j & 1 ? b1 >> 6 : b1 << 2;
            af[0] = s0 & 0x003c003cu, af[1] = s0 & 0x03c003c0u, af[2] = s1 & 0x003c003cu, af[3] = s1 & 0x03c003c0u;
          }
#pragma unroll
          for (int y = 0; y < NT; y++) {
            mma(o[y][g][j], af, ph[y][g][0], ph[y][g][1]);
            if constexpr (SPLIT) mma(o[y][g][j], af, pl[y][g][0], pl[y][g][1]);
          }
        }
      }
    }
    // take kMid * sum(p * step) out again, in the codes' units
#pragma unroll
    for (int y = 0; y < NT; y++)
#pragma unroll
      for (int g = 0; g < NG; g++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[y][g][j][i] = fmaf(sum[y][g][i & 1], -kMid * (SPLIT || i & 2 ? 0x1p-18f : 0x1p-22f), o[y][g][j][i]);
    unit += cnt;
    if constexpr (SPLIT) flip = ~flip;  // an odd number of units a stage
    __syncwarp();  // every lane has read the slot
    if (next < u1) {
      const int more = count(next);
      load_stage<DK>(a, base, u, next, more, ring + slot, bars + 8 * slot);
      next += more;
    }
    if (++slot == NST) slot = 0, parity ^= 1;
  }
  if (!ok) {
    if (lane == 0) kv4_error();
#pragma unroll 1
    for (int i = 0; i < NST; i++) {  // copies still on their way land before the rings are used again, if they ever do
      sm100::bar_wait(bars + 8 * slot, parity);
      if (++slot == NST) slot = 0, parity ^= 1;
    }
  }

  // ---- the warps' results, then the CTA's
  sm100::dependents_launch();
  constexpr int LDO = DK + 4;
  float *so = reinterpret_cast<float *>(smem);                        // [kWarps][TR][LDO]
  float2 *sml = reinterpret_cast<float2 *>(so + kWarps * TR * LDO);   // [kWarps][TR]
  static_assert(kWarps * TR * (LDO * 4 + 8) + 4 <= kWarps * NST * (int)sizeof(Stage<DK>), "the rings hold it");
  __syncthreads();  // the rings are idle (a warp whose wait gave up has reported it)
  float back[NG], back1[NG];  // of the even and odd dims of the codes
#pragma unroll
  for (int g = 0; g < NG; g++) {
    back[g] = vs[g] == 0.0f ? 0.0f : (SPLIT ? 0x1p18f : 0x1p22f) / vs[g];
    back1[g] = SPLIT ? back[g] : back[g] * 0.0625f;
  }
#pragma unroll
  for (int y = 0; y < NT; y++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int rr = warp * TR + y * kRows + 2 * c + i;
      const float ls = col_sum(l[y][i]);
      if (r == 0) sml[rr] = make_float2(mrow[y][i], ls);
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const float zz = col_sum(z[y][g][i]);
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; j++)
          v[2 * j] = fmaf(o[y][g][j][i], back[g], zz), v[2 * j + 1] = fmaf(o[y][g][j][i + 2], back1[g], zz);
        float4 *dst = reinterpret_cast<float4 *>(so + rr * LDO + 64 * g + 8 * r);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
  __syncthreads();
  constexpr int PER = 8;  // consecutive dims of one row
  auto write_row = [&](int row, int d0, float m, float sum, const float (&v)[PER]) {
    E *dst = out + (((long long)s * a.row_T + row / G) * a.H + kvh * G + row % G) * DK + d0;
#pragma unroll
    for (int i = 0; i < PER; i++) dst[i] = from_f32<E>(sum == 0.0f ? 0.0f : v[i] / sum);
    if (WS && d0 == 0) a.stat[((size_t)s * a.Hkv + kvh) * a.prow + row] = m == -INFINITY ? sum : m + log2f(sum);
  };
  for (int at = threadIdx.x; at < TR * DK / PER; at += 32 * kWarps) {
    const int rr = at * PER / DK, d0 = at * PER % DK, row = tile * TR + rr;
    if (row >= rows) break;
    float m = -INFINITY, sum = 0.0f, v[PER] = {};
#pragma unroll
    for (int w = 0; w < kWarps; w++) m = fmaxf(m, sml[w * TR + rr].x);
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      const float2 ml = sml[w * TR + rr];
      const float k = ml.x == -INFINITY && ml.y == 0.0f ? 0.0f : sm100::ex2(ml.x - m);
      sum = fmaf(k, ml.y, sum);
      if (k != 0.0f)
#pragma unroll
        for (int i = 0; i < PER; i++) v[i] = fmaf(k, so[(w * TR + rr) * LDO + d0 + i], v[i]);
    }
    const size_t pr = (((size_t)s * a.Hkv + kvh) * a.prow + row) * a.splits + split;
    if (a.splits > 1 && d0 == 0) a.pml[pr] = make_float2(m, sum);
    if (a.splits > 1) {
      float4 *dst = reinterpret_cast<float4 *>(a.po + pr * DK + d0);
      dst[0] = make_float4(v[0], v[1], v[2], v[3]);
      dst[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      write_row(row, d0, m, sum, v);
    }
  }
  if (!a.join && !(WS && a.splits > 1)) return;
  // few splits: the last CTA to finish joins them, in their order (more go to kv4_after_kernel, a CTA per row)
  unsigned int *flag = reinterpret_cast<unsigned int *>(sml + kWarps * TR);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *flag = atomicInc(a.done + ((size_t)s * a.Hkv + kvh) * a.tiles + tile, a.splits - 1);
  __syncthreads();
  if (*flag != (unsigned int)a.splits - 1) return;
  __threadfence();
  if (!a.join) {  // the rows' statistics, so that the weights need not wait for the join
    for (int row = tile * TR + warp; row < min(rows, (tile + 1) * TR); row += kWarps) {
      const size_t at = ((size_t)s * a.Hkv + kvh) * a.prow + row;
      float m = -INFINITY, sum = 0.0f;
      for (int i = lane; i < a.splits; i += 32) m = fmaxf(m, __ldcg(&a.pml[at * a.splits + i].x));
      for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
      for (int i = lane; i < a.splits; i += 32) {
        const float2 ml = __ldcg(a.pml + at * a.splits + i);
        sum += ml.x == -INFINITY && ml.y == 0.0f ? 0.0f : sm100::ex2(ml.x - m) * ml.y;
      }
      for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (lane == 0) a.stat[at] = m == -INFINITY ? sum : m + log2f(sum);
    }
    return;
  }
  for (int at = threadIdx.x; at < TR * DK / PER; at += 32 * kWarps) {
    const int rr = at * PER / DK, d0 = at * PER % DK, row = tile * TR + rr;
    if (row >= rows) break;
    const size_t pr = (((size_t)s * a.Hkv + kvh) * a.prow + row) * a.splits;
    float m = -INFINITY, sum = 0.0f, v[PER] = {};
    for (int i = 0; i < a.splits; i++) m = fmaxf(m, __ldcg(&a.pml[pr + i].x));
#pragma unroll 4
    for (int i = 0; i < a.splits; i++) {
      const float2 ml = __ldcg(a.pml + pr + i);
      const float4 *po = reinterpret_cast<const float4 *>(a.po + (pr + i) * DK + d0);
      const float4 p0 = __ldcg(po), p1 = __ldcg(po + 1);
      const float k = ml.x == -INFINITY && ml.y == 0.0f ? 0.0f : sm100::ex2(ml.x - m);
      sum = fmaf(k, ml.y, sum);
      if (k != 0.0f) {
        v[0] = fmaf(k, p0.x, v[0]), v[1] = fmaf(k, p0.y, v[1]), v[2] = fmaf(k, p0.z, v[2]), v[3] = fmaf(k, p0.w, v[3]);
        v[4] = fmaf(k, p1.x, v[4]), v[5] = fmaf(k, p1.y, v[5]), v[6] = fmaf(k, p1.z, v[6]), v[7] = fmaf(k, p1.w, v[7]);
      }
    }
    write_row(row, d0, m, sum, v);
  }
}

// After the attention: the first `joins` CTAs of a sequence join the splits of a row each, the others add to wsum,
// kSumTok tokens of a kv head each: wsum[j] += sum over the rows of 2^(x_j - stat), four tokens a thread, four rows on
// their way at once (64 rows of 131071 logits, the whole pass: 53 us; eight rows and fewer CTAs an SM 55, one 57).
constexpr int kAfter = 128, kSumTok = 4 * kAfter;

template <class E, int DK>
__device__ __forceinline__ void join_row(const Attn4 &a, E *__restrict__ out) {
  constexpr int NW = kAfter / 32, PER = DK / 32;
  __shared__ float2 sml[NW];
  __shared__ float so[NW][DK];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.H / a.Hkv, rows = a.T * G, s = blockIdx.y;
  const int kvh = blockIdx.x / rows, row = blockIdx.x % rows;
  const size_t pr = (((size_t)s * a.Hkv + kvh) * a.prow + row) * a.splits;
  float m = -INFINITY, l = 0.0f, v[PER] = {};
  const int i0 = a.splits * warp / NW, i1 = a.splits * (warp + 1) / NW;  // the warp's splits, 32 at a time
  for (int i = i0; i < i1; i += 32) {
    const float2 ml = i + lane < i1 ? a.pml[pr + i + lane] : make_float2(-INFINITY, 0.0f);
    float mn = ml.x;
    for (int off = 16; off; off >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, off));
    mn = fmaxf(mn, m);
    const float was = m == mn ? 1.0f : sm100::ex2(m - mn);
    const float k = ml.x == -INFINITY && ml.y == 0.0f ? 0.0f : sm100::ex2(ml.x - mn);
    m = mn;
    l = fmaf(k, ml.y, l * was);
#pragma unroll
    for (int d = 0; d < PER; d++) v[d] *= was;
    const int cnt = min(32, i1 - i);
#pragma unroll 16
    for (int j = 0; j < cnt; j++) {
      const float kj = __shfl_sync(0xffffffffu, k, j);
      const float *po = a.po + (pr + i + j) * DK + PER * lane;
#pragma unroll
      for (int d = 0; d < PER; d++) {
        const float x = po[d];
        if (kj != 0.0f) v[d] = fmaf(kj, x, v[d]);
      }
    }
  }
  for (int off = 16; off; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  if (lane == 0) sml[warp] = make_float2(m, l);
#pragma unroll
  for (int d = 0; d < PER; d++) so[warp][PER * lane + d] = v[d];
  __syncthreads();
  if ((int)threadIdx.x >= DK) return;
  float mm = -INFINITY, sum = 0.0f, x = 0.0f;
#pragma unroll
  for (int w = 0; w < NW; w++) mm = fmaxf(mm, sml[w].x);
#pragma unroll
  for (int w = 0; w < NW; w++) {
    const float k = sml[w].x == -INFINITY && sml[w].y == 0.0f ? 0.0f : sm100::ex2(sml[w].x - mm);
    sum = fmaf(k, sml[w].y, sum);
    if (k != 0.0f) x = fmaf(k, so[w][threadIdx.x], x);
  }
  out[(((long long)s * a.row_T + row / G) * a.H + kvh * G + row % G) * DK + threadIdx.x] = from_f32<E>(sum == 0.0f ? 0.0f : x / sum);
}

__device__ __forceinline__ void sum_weights(const Attn4 &a, int block) {
  constexpr int CH = 256;  // rows at a time
  __shared__ float stat[CH];
  const int kvh = block % a.Hkv, s = blockIdx.y, rows = a.T * (a.H / a.Hkv);
  const Units u = units_of(a, seq_len(a, s));
  const int i0 = block / a.Hkv * kSumTok, live = u.all * kUnit, i = i0 + 4 * threadIdx.x;
  if (i0 >= live) return;
  const size_t pr = ((size_t)s * a.Hkv + kvh) * a.prow;
  const int j = i < live ? token_of(u, i / kUnit) + i % kUnit : u.n;
  float *w = a.wsum + ((size_t)s * a.Hkv + kvh) * a.cap + j;
  float old[4], sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < 4; e++) old[e] = j + e < u.n ? w[e] : 0.0f;
  for (int r0 = 0; r0 < rows; r0 += CH) {
    const int r1 = min(rows, r0 + CH);
    if (r0) __syncthreads();
    for (int row = r0 + threadIdx.x; row < r1; row += kAfter) stat[row - r0] = a.stat[pr + row];
    for (int b = r0; b < r1; b += 4) {  // four rows on their way at once
      const float *x = a.x + (pr + b) * a.vis + i;
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (b + k < r1 && i < live) v[k] = __ldcs(reinterpret_cast<const float4 *>(x + (size_t)k * a.vis));
      if (b == r0) __syncthreads();
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if (b + k >= r1 || i >= live) break;
        const float st = stat[b + k - r0], y[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
        for (int e = 0; e < 4; e++) {  // a place that is not visible holds -inf
          if (st == st) sum[e] += sm100::ex2(y[e] - st);
          else if (y[e] != -INFINITY) sum[e] = st;  // a row that sees a NaN: so are its weights, of what it sees
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (j + e < u.n) w[e] = old[e] + sum[e];
}

template <class E, int DK>
__global__ void __launch_bounds__(kAfter) kv4_after_kernel(const Attn4 a, E *__restrict__ out, int joins) {
  sm100::dependency_wait();
  if ((int)blockIdx.x < joins) join_row<E, DK>(a, out);
  else sum_weights(a, blockIdx.x - joins);
}

// Up to this many splits are joined by the last CTA of an item, in the launch itself; more by a CTA a row.
constexpr int kJoinSplits = 16;

// Token splits: the fewest waves of resident CTAs times what one takes, its units and about 45 units' worth (9 us) of
// setting up and joining. Measured: 440 items of 1024 units 197, 203, 210, 215 us in 1 to 4 splits, 231 in 8; 296 items
// 142, 159, 143, 149 us in 1 to 4, 160 in 6; 144 items 104, 79, 76, 95 us in 1 to 4; 8 items of 8192 units 69 us in 18
// splits, 58 in 37 and 55, 66 in 74. It picks 1, 3, 3 and 55.
// Two units a warp at least.
int choose_splits(const Attn4 &a, int ctas) {
  const long long items = (long long)a.nseq * a.Hkv * a.tiles, units = a.vis / kUnit, slots = 148LL * ctas;
  long long best = 1, least = 0;
  for (long long s = 1; s == 1 || (s <= units / (2 * kWarps) && s <= 128); s++) {
    const long long cost = (items * s + slots - 1) / slots * ((units + s - 1) / s + 45);
    if (s == 1 || cost < least) best = s, least = cost;
  }
  return (int)best;
}

template <class E, int DK, bool WS>
cudaError_t launch_attn_ws(const Attn4 &a, const E *q, E *out, cudaStream_t st, uint64_t *launches) {
  auto kern = a.prow / a.tiles == kRows ? kv4_attn_kernel<E, DK, 1, WS> : kv4_attn_kernel<E, DK, 2, WS>;
  const int smem = a.prow / a.tiles == kRows ? kAttnSmem<E, DK, 1> : kAttnSmem<E, DK, 2>;
  cudaError_t e = smem_attr((const void *)kern, smem);
  if (e != cudaSuccess) return e;
  kern<<<dim3(a.splits * a.tiles * a.Hkv, a.nseq), 32 * kWarps, smem, st>>>(a, q, out);
  *launches += 1;
  e = cudaGetLastError();
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const int joins = a.splits > 1 && !a.join ? a.Hkv * a.T * (a.H / a.Hkv) : 0;
  if (e == cudaSuccess && (WS || joins)) {
    cfg.gridDim = dim3(joins + (WS ? (a.vis + kSumTok - 1) / kSumTok * a.Hkv : 0), a.nseq);
    cfg.blockDim = dim3(kAfter);
    *launches += 1;
    e = cudaLaunchKernelEx(&cfg, kv4_after_kernel<E, DK>, a, out, joins);
  }
  return e;
}
template <class E>
cudaError_t launch_attn(const Attn4 &a, int dk, const E *q, E *out, cudaStream_t st, uint64_t *launches) {
  if (dk == 64) return a.wsum ? launch_attn_ws<E, 64, true>(a, q, out, st, launches) : launch_attn_ws<E, 64, false>(a, q, out, st, launches);
  return a.wsum ? launch_attn_ws<E, 128, true>(a, q, out, st, launches) : launch_attn_ws<E, 128, false>(a, q, out, st, launches);
}

}  // namespace

unsigned int kv4_error_flag(bool reset) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_kv4_error, sizeof v);
  if (reset && v) {
    const unsigned int z = 0;
    cudaMemcpyToSymbol(g_kv4_error, &z, sizeof z);
  }
  return v;
}

ORKB_ERR_WORD_SETTER(kv4_set_err_word)

}  // namespace orkb

using namespace orkb;

static int refuse(const char *name, const char *why) {
  fprintf(stderr, "[ork] ERROR %s: %s\n", name, why);
  return -1;
}

static const char *cache_wrong(const ork_b200_kv4 *c) {
  if (!c->k || !c->v || !c->kp || !c->vp) return "a cache array is NULL";
  if (c->dk != 64 && c->dk != 128) return "dk is 64 or 128";
  if (c->nseq < 1 || c->Hkv < 1 || c->cap < 64 || c->cap % 64) return "nseq, Hkv >= 1 and cap a multiple of 64";
  if ((long long)c->nseq * c->Hkv > 65535) return "nseq * Hkv is at most 65535";
  if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->kp | (uintptr_t)c->vp) % 16) return "cache arrays are 16-byte aligned";
  return nullptr;
}

static int kv4_rows(ork_npu *c, const ork_b200_kv4 *kv, const void *k, const void *v, int type, int rows, long long ts,
                    long long hs, const int *start, const int *pos, bool store, const char *name) {
  if (!c || !kv || !k || !v) return -1;
  if (const char *why = cache_wrong(kv)) return refuse(name, why);
  if (type < ORK_B200_F32 || type > ORK_B200_BF16) return refuse(name, "unknown element type");
  if (rows < 0 || (!start && (long long)kv->nseq * rows > 0x7fffffff)) return refuse(name, "bad number of rows");
  if (ts < kv->dk || hs < kv->dk) return refuse(name, "a row stride below dk");
  const size_t es = elem_bytes(type);
  if (((uintptr_t)k | (uintptr_t)v) % es) return refuse(name, "rows are aligned to their type");
  if (((uintptr_t)start | (uintptr_t)pos) % 4) return refuse(name, "start and pos are 4-byte aligned");
  DeviceGuard dg(c->device);
  if (!device_ptrs_ok(c, name, {kv->k, kv->v, kv->kp, kv->vp, k, v, start, pos})) return -1;
  if (rows == 0) return 0;
  const bool vec = ((uintptr_t)k | (uintptr_t)v | (size_t)ts * es | (size_t)hs * es) % 16 == 0;
  const Rows r = {kv->nseq, kv->Hkv, kv->cap, rows, ts, hs, start, pos};
  // Teams of a (row, head): a multiple of Hkv, so that every thread has a head; as many rows for each as it has on their
  // way at once, and 12 blocks an SM at most (three waves of a store: 8 are 1 to 4 % slower, one row for each 15 to 30 %
  // on 4000 rows of 64 dims).
  const long long per = kRowThreads / (kv->dk / 4 / (store ? kStoreWords : 1)), each = store ? 2 : 4;
  const long long want = ((rows + each - 1) / each * kv->Hkv + per - 1) / per;
  const long long most = std::max<long long>(148LL * 12 / kv->nseq, (kv->Hkv + per - 1) / per);
  const dim3 grid((unsigned)std::min(want, most), kv->nseq);
  const cudaError_t e = with_elem(type, [&](auto *t) {
    using E = std::remove_pointer_t<decltype(t)>;
    auto go = [&](auto aligned) {
      constexpr bool V = decltype(aligned)::value;
      auto kern = kv->dk == 64 ? (store ? kv4_rows_kernel<E, 64, true, V> : kv4_rows_kernel<E, 64, false, V>)
                               : (store ? kv4_rows_kernel<E, 128, true, V> : kv4_rows_kernel<E, 128, false, V>);
      kern<<<grid, kRowThreads, 0, c->stream>>>(r, (E *)k, (E *)v, (uint32_t *)kv->k, (uint32_t *)kv->v, (__half2 *)kv->kp,
                                                (__half2 *)kv->vp);
    };
    if (vec) go(std::true_type());
    else go(std::false_type());
    return cudaGetLastError();
  });
  c->launches += 1;
  if (e != cudaSuccess) {
    log_err(name, e);
    return -1;
  }
  return 0;
}

// What a launch for the tokens t0 .. t0 + T - 1 of the call's T takes, and where in the workspace (from 0 on).
struct Plan4 {
  Attn4 k;
  size_t ml, po, stat, need;  // bytes of partial maxima, outputs, statistics; of all
  size_t counts;
};
static Plan4 kv4_plan(const ork_b200_kv4 *kv, const ork_b200_kv4_attn *a, int t0, int T) {
  Plan4 p = {};
  Attn4 &k = p.k;
  k.kc = kv->k, k.vc = kv->v, k.kp = (const __half *)kv->kp, k.vp = (const __half *)kv->vp;
  k.nseq = kv->nseq, k.Hkv = kv->Hkv, k.cap = kv->cap, k.H = a->H, k.T = T, k.row_T = a->T, k.late = a->T - t0 - T;
  k.window = a->window < a->max_len ? a->window : 0;  // a window over everything is none
  k.sinks = std::min(a->sinks, a->max_len);
  k.max_len = a->max_len, k.q_ts = a->q_ts, k.q_hs = a->q_hs, k.len = a->len, k.scale = a->scale, k.wsum = a->wsum;
  const int rows = T * (a->H / kv->Hkv), tr = rows > kRows ? 2 * kRows : kRows;
  k.tiles = (rows + tr - 1) / tr;
  k.prow = k.tiles * tr;
  // sinks and window, whole units of each
  long long vis = (std::max(a->max_len - k.late, 1) + kUnit - 1) / kUnit * kUnit;
  if (k.window) vis = std::min<long long>(vis, (long long)k.window + k.T + k.sinks + 3 * kUnit);
  k.vis = (int)(vis / kUnit * kUnit);
  k.splits = choose_splits(k, kv->dk == 128 && (tr > kRows || a->type == ORK_B200_F32) ? 2 : 3);
  k.qvec = ((uintptr_t)a->q | (size_t)a->q_ts * elem_bytes(a->type) | (size_t)a->q_hs * elem_bytes(a->type)) % 16 == 0;
  k.join = k.splits > 1 && k.splits <= kJoinSplits;
  auto whole = [](size_t b) { return (b + 255) / 256 * 256; };
  const size_t prows = (size_t)k.nseq * k.Hkv * k.prow, parts = k.splits > 1 ? prows * k.splits : 0;
  p.ml = whole(parts * sizeof(float2)), p.po = whole(parts * kv->dk * 4), p.stat = a->wsum ? whole(prows * 4) : 0;
  p.need = p.ml + p.po + p.stat + (a->wsum ? prows * k.vis * 4 : 0);
  if (k.join || (a->wsum && k.splits > 1)) p.counts = (size_t)k.nseq * k.Hkv * k.tiles;
  return p;
}

// Logits that a call with weights to add up keeps at a time, in bytes: a call of more goes through its tokens in several
// passes (2500 tokens of 16 heads after 60000: 9.6 GB otherwise). Decode steps and drafts need one.
constexpr long long kLogits = 4ll << 30;

extern "C" {

int ork_b200_kv4_store_async(ork_npu *c, const ork_b200_kv4 *kv, const void *k, const void *v, int type, int rows,
                             long long ts, long long hs, const int *start, const int *pos) {
  return kv4_rows(c, kv, k, v, type, rows, ts, hs, start, pos, true, "ork_b200_kv4_store_async");
}

int ork_b200_kv4_load_async(ork_npu *c, const ork_b200_kv4 *kv, void *k, void *v, int type, int rows, long long ts,
                            long long hs, const int *start, const int *pos) {
  return kv4_rows(c, kv, k, v, type, rows, ts, hs, start, pos, false, "ork_b200_kv4_load_async");
}

int ork_b200_kv4_attn_async(ork_npu *c, const ork_b200_kv4 *kv, const ork_b200_kv4_attn *a) {
  const char *name = "ork_b200_kv4_attn_async";
  if (!c || !kv || !a || !a->q || !a->out || !a->len) return -1;
  if (const char *why = cache_wrong(kv)) return refuse(name, why);
  if (a->type < ORK_B200_F32 || a->type > ORK_B200_BF16) return refuse(name, "unknown element type");
  if (a->H < 1 || a->H % kv->Hkv) return refuse(name, "H is a multiple of Hkv");
  if (a->T < 1 || a->T > kv->cap || (long long)kv->nseq * a->T * a->H > 0x7fffffff) return refuse(name, "bad number of rows");
  if (a->q_ts < kv->dk || a->q_hs < kv->dk) return refuse(name, "a row stride below dk");
  if (a->max_len < 0 || a->max_len > kv->cap) return refuse(name, "max_len is 0 .. cap");
  if (a->window < 0 || a->sinks < 0) return refuse(name, "window and sinks are not negative");
  if (((uintptr_t)a->q | (uintptr_t)a->out) % elem_bytes(a->type)) return refuse(name, "rows are aligned to their type");
  if (((uintptr_t)a->len | (uintptr_t)a->wsum) % 4) return refuse(name, "len and wsum are 4-byte aligned");
  DeviceGuard dg(c->device);
  if (!device_ptrs_ok(c, name, {kv->k, kv->v, kv->kp, kv->vp, a->q, a->out, a->len, a->wsum})) return -1;
  if (a->max_len == 0) {
    const cudaError_t e = cudaMemsetAsync(a->out, 0, (size_t)kv->nseq * a->T * a->H * kv->dk * elem_bytes(a->type), c->stream);
    if (e != cudaSuccess) log_err(name, e);
    return e == cudaSuccess ? 0 : -1;
  }
  int step = a->T;  // tokens a pass
  if (a->wsum) {
    const long long span = a->window ? std::min<long long>(a->max_len, (long long)a->window + a->T + a->sinks + 3 * kUnit) : a->max_len;
    int unit = 1;  // tokens of whole column tiles
    while (unit < 2 * kRows && (a->H / kv->Hkv) * unit % (2 * kRows)) unit *= 2;
    step = (int)std::min<long long>(step, std::max(kLogits / 4 / span / ((long long)kv->nseq * a->H) / unit, 1ll) * unit);
  }
  Plan4 p = kv4_plan(kv, a, 0, step);
  size_t need = p.need, counts = p.counts;
  for (int t = step; t < a->T; t += step) {  // whatever is refused is refused before the first pass
    const Plan4 q = kv4_plan(kv, a, t, std::min(step, a->T - t));
    need = std::max(need, q.need), counts = std::max(counts, q.counts);
  }
  if (need && !work_block(c, name, &c->work, need)) return -1;
  unsigned int *done = nullptr;
  if (counts && !(done = zeroed_counts(c, name, counts))) return -1;
  for (int t = 0; t < a->T; t += step) {
    if (t) p = kv4_plan(kv, a, t, std::min(step, a->T - t));
    uint8_t *ws = (uint8_t *)c->work.p;
    p.k.pml = (float2 *)ws, p.k.po = (float *)(ws + p.ml), p.k.stat = (float *)(ws + p.ml + p.po);
    p.k.x = (float *)(ws + p.ml + p.po + p.stat);
    p.k.done = done + kAttnCounts;
    const cudaError_t e = with_elem(a->type, [&](auto *x) {
      using E = std::remove_pointer_t<decltype(x)>;
      return launch_attn<E>(p.k, kv->dk, (const E *)a->q + t * a->q_ts, (E *)a->out + (long long)t * a->H * kv->dk, c->stream, &c->launches);
    });
    if (e != cudaSuccess) {
      log_err(name, e);
      return -1;
    }
  }
  return 0;
}

}  // extern "C"
