// attn.cu -- attention of packed rows (prompts, or chunks after a cached prefix) with a sliding window and sink
// keys (include/ork_b200.h: ork_b200_attn_async), on the 5th-generation tensor cores.
//
// A CTA owns two tiles of 128 query rows of one kv head and streams the keys that any of them sees, 128 at a time:
//   S = Q K^T     128 x 128 x dk, both operands in shared memory, S in tensor memory (fp32)
//   P = 2^(S sc - m)  online softmax, a thread per row; P goes back to tensor memory in 16 bits, over S
//   O += P V      128 x dk x 128, P from tensor memory, V in shared memory as it lies (N-major), O in tensor memory
// The two tiles alternate: while one is in its softmax the tensor cores work for the other. A row of a tile is a
// (token, head) pair, `pack` heads of the group (its largest power of two, at most 8) side by side, so that few tokens
// still fill a tile, and the tile's tokens, whose windows end at different keys, are few.
// Roles (320 threads): warps 0-3 and 4-7 the softmax and output of tile 0 and 1, warp 8 issues the products, warp 9
// the TMA loads into a ring of 128 x dk slots that K and V tiles share. A row of S is read twice, for its maximum and
// for its weights, 32 columns at a time: tensor memory has bandwidth to spare, and a whole row in registers spills.
// The running maximum follows only when it rises by more than 2^8, so that O is seldom scaled; weights stay below 256.
// Masks are applied to the tiles that hold an edge; tiles that no row sees are not visited.
// A value of V that is not finite reaches rows that do not see it (0 * inf): a row whose result is not finite is
// computed again, from its visible keys alone, by its warp. Rows of V past the sequence are cleared in shared memory.
//
// Every wait is bounded; one that expires records an error and the roles fall through to the common exit.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>

#include "elem.cuh"
#include "errword.cuh"
#include "ork_internal.h"
#include "ork_structs.h"
#include "sm100.cuh"

namespace orkb {

__device__ unsigned int g_attn_error = 0;

namespace {

// The row ranges of sequence s, or false (reported) where they do not lie in the tensors or pass the maxima that
// sized the launch.
struct Seq {
  int q0, tq, k0, tk;
};
__device__ __forceinline__ bool seq_of(const ork_b200_attn &a, int s, Seq *o) {
  o->q0 = a.q_start[s], o->k0 = a.k_start[s];
  const int q1 = a.q_start[s + 1], k1 = a.k_start[s + 1];
  const bool ok = o->q0 >= 0 && q1 >= o->q0 && q1 <= a.q_rows && q1 - o->q0 <= a.max_q && o->k0 >= 0 && k1 >= o->k0 &&
                  k1 <= a.k_rows && k1 - o->k0 <= a.max_k;
  o->tq = ok ? q1 - o->q0 : 0;
  o->tk = ok ? k1 - o->k0 : 0;
  if (!ok && threadIdx.x == 0) {
    atomicOr(&g_attn_error, 1u);
    err_word_set();
  }
  return ok;
}

constexpr int kTile = 128;    // query rows of a tile, keys of a step
constexpr int kThreads = 320;
constexpr float kRise = 8.0f;  // log2 of the rise of a maximum that O is scaled for

__device__ __forceinline__ void attn_failed() {
  atomicOr(&g_attn_error, 1u);
  err_word_set();
}

// Shared-memory matrix descriptors of tiles of 64 x 16-bit columns with 128-byte swizzle, 1024-byte aligned: K-major
// (the contraction along the 128 bytes; 8-row groups 1024 bytes apart), and MN-major (the contraction along the rows;
// `chunk` bytes from one 64-column block to the next).
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t chunk) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(chunk >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
template <class E>
constexpr uint32_t inst_desc(int n, bool b_mn) {
  const uint32_t f = sizeof(E) == 2 && !std::is_same<E, __half>::value ? 1u : 0u;  // fp16 0, bf16 1
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

__device__ __forceinline__ uint32_t pack2(float x, float y, const __half *) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, const __nv_bfloat16 *) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <int DK>
struct Smem {
  static constexpr int kSlots = DK == 128 ? 5 : 8;
  static constexpr int kTileBytes = kTile * DK * 2, kChunk = kTile * 128;  // a 64-column block of a tile
  static constexpr int kBars = 1 + 2 * kSlots + 6;
  static constexpr int kBytes = 1024 + (2 + kSlots) * kTileBytes + kBars * 8 + 16;
};
static_assert(Smem<128>::kBytes <= 232448 && Smem<64>::kBytes <= 232448, "shared memory");

// The key tiles of query positions p0 .. p1 (p1 >= 0): ns tiles of sinks from 0 on, then lo .. hi.
struct Steps {
  int ns, lo, hi;
  __device__ __forceinline__ int count() const { return ns + hi - lo + 1; }
  __device__ __forceinline__ int tile(int i) const { return i < ns ? i : i - ns + lo; }
  __device__ __forceinline__ bool has(int t) const { return t <= hi && (t >= lo || t < ns); }
};
__device__ __forceinline__ Steps steps_of(int p0, int p1, int window, int sinks) {
  Steps s;
  s.lo = window && p0 - window + 1 > 0 ? (p0 - window + 1) / kTile : 0;
  s.hi = p1 >= 0 ? p1 / kTile : -1;
  s.ns = min((sinks + kTile - 1) / kTile, s.lo);
  if (p1 < 0) s.ns = s.lo = 0;
  return s;
}

// One row from its visible keys alone, by a warp: lane l holds dims l + 32 u.
template <class E, int DK>
__device__ __noinline__ void slow_row(const ork_b200_attn &a, const Seq &s, int tok, int h) {
  constexpr int PER = DK / 32;
  const int lane = threadIdx.x & 31, kvh = h / (a.H / a.Hkv), p = s.tk - s.tq + tok;
  const E *q = (const E *)a.q + (s.q0 + tok) * a.q_ts + h * a.q_hs;
  E *out = (E *)a.out + (s.q0 + tok) * a.o_ts + h * a.o_hs;
  float qv[PER], o[PER] = {}, m = -INFINITY, l = 0.0f;
  for (int u = 0; u < PER; u++) qv[u] = to_f32(q[lane + 32 * u]) * a.scale;
  for (int j = 0; j <= p; j++) {
    if (a.window && j <= p - a.window && j >= a.sinks) j = p - a.window + 1;
    const E *k = (const E *)a.k + (s.k0 + j) * a.k_ts + kvh * a.k_hs, *v = (const E *)a.v + (s.k0 + j) * a.v_ts + kvh * a.v_hs;
    float x = 0.0f;
    for (int u = 0; u < PER; u++) x += qv[u] * to_f32(k[lane + 32 * u]);
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    const float mn = fmaxf(m, x), c = m == mn ? 1.0f : expf(m - mn), w = expf(x - (mn == -INFINITY ? 0.0f : mn));
    l = l * c + w;
    for (int u = 0; u < PER; u++) o[u] = o[u] * c + w * to_f32(v[lane + 32 * u]);
    m = mn;
  }
  for (int u = 0; u < PER; u++) out[lane + 32 * u] = from_f32<E>(l == 0.0f ? 0.0f : o[u] / l);
}

template <class E, int DK>
__global__ void __launch_bounds__(kThreads, 1)
    attn_kernel(const ork_b200_attn a, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                const __grid_constant__ CUtensorMap mv, int pack, int groups) {
  using M = Smem<DK>;
  constexpr int SLOTS = M::kSlots, CH = DK / 64;
  extern __shared__ uint8_t raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sq = sm100::smem_addr(smem), sring = sq + 2 * M::kTileBytes, bars = sring + SLOTS * M::kTileBytes;
  const uint32_t qfull = bars, full = bars + 8, empty = full + 8 * SLOTS, sfull = empty + 8 * SLOTS, pfull = sfull + 16,
                 ofull = pfull + 16;
  uint32_t *slot = (uint32_t *)(smem + (2 + SLOTS) * M::kTileBytes + M::kBars * 8);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  // the item: a head group of a sequence, and a pair of tiles of its tokens, the last ones first (they see most)
  const int hg = blockIdx.x % groups, kvh = hg * pack / (a.H / a.Hkv), h0 = hg * pack;
  const int per = kTile / pack, tok0 = (gridDim.x / groups - 1 - blockIdx.x / groups) * 2 * per;
  Seq s;
  if (!seq_of(a, blockIdx.y, &s) || tok0 >= s.tq) return;
  const int back = s.tk - s.tq;  // position of token 0
  Steps st[2], all;
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int t0 = tok0 + t * per, t1 = min(t0 + per, s.tq) - 1;
    st[t] = steps_of(back + t0, t0 <= t1 ? back + t1 : -1, a.window, a.sinks);
  }
  all = steps_of(back + tok0, back + min(tok0 + 2 * per, s.tq) - 1, a.window, a.sinks);

  if (threadIdx.x == 0) {
    sm100::bar_init(qfull, 1);
    for (int i = 0; i < SLOTS; i++) sm100::bar_init(full + 8 * i, 1), sm100::bar_init(empty + 8 * i, 1);
    for (int t = 0; t < 2; t++) sm100::bar_init(sfull + 8 * t, 1), sm100::bar_init(pfull + 8 * t, 4), sm100::bar_init(ofull + 8 * t, 1);
    sm100::bar_init_fence();
  }
  if (warp == 8) sm100::tmem_alloc(sm100::smem_addr(slot), 512);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *slot;
  const int steps = all.count();

  if (warp == 9) {  // ---- loads
    if (lane == 0 && steps > 0) {
      sm100::bar_expect(qfull, 2 * M::kTileBytes);
      for (int t = 0; t < 2; t++)
        for (int c = 0; c < CH; c++)
          sm100::tma_load_3d(sq + t * M::kTileBytes + c * M::kChunk, &mq, 64 * c, h0, s.q0 + tok0 + t * per, qfull);
      for (int i = 0; i < 2 * steps; i++) {  // K of step 0, V of step 0, K of step 1, ...
        const int sl = i % SLOTS;
        if (i >= SLOTS && !sm100::bar_wait(empty + 8 * sl, (i / SLOTS - 1) & 1)) {
          attn_failed();
          break;
        }
        sm100::bar_expect(full + 8 * sl, M::kTileBytes);
        for (int c = 0; c < CH; c++)
          sm100::tma_load_3d(sring + sl * M::kTileBytes + c * M::kChunk, i & 1 ? (const void *)&mv : (const void *)&mk, 64 * c, kvh,
                             s.k0 + all.tile(i >> 1) * kTile, full + 8 * sl);
      }
    }
  } else if (warp == 8) {  // ---- products
    constexpr uint32_t ids = inst_desc<E>(kTile, false), ido = inst_desc<E>(DK, true);
    bool ok = steps == 0 || sm100::bar_wait(qfull, 0);
    int np[2] = {0, 0};  // P tiles consumed
    // S of tile t at step i from the K in slot sl
    auto score = [&](int t, int sl) {
      const uint64_t qa = desc_k(sq + t * M::kTileBytes), kb = desc_k(sring + sl * M::kTileBytes);
#pragma unroll
      for (int c = 0; c < CH; c++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          sm100::tc_mma(tmem + t * kTile, qa + (uint64_t)(c * (M::kChunk >> 4) + 2 * k), kb + (uint64_t)(c * (M::kChunk >> 4) + 2 * k),
                        ids, c | k ? 1u : 0u);
      sm100::tc_commit(sfull + 8 * t);
    };
    auto wait_full = [&](int i) { return sm100::bar_wait(full + 8 * (i % SLOTS), (i / SLOTS) & 1); };
    if (steps > 0 && ok) {
      ok = wait_full(0);
      sm100::tc_fence_after();
      if (ok && lane == 0) {
        for (int t = 0; t < 2; t++)
          if (st[t].has(all.tile(0))) score(t, 0);
        sm100::tc_commit(empty);
      }
    }
    for (int i = 0; i < steps && ok; i++) {
      const int kt = all.tile(i), vi = 2 * i + 1, ki = 2 * i + 2;
      ok = wait_full(vi) && (i + 1 == steps || wait_full(ki));
      if (!ok) break;
      const uint32_t sv = sring + vi % SLOTS * M::kTileBytes;
      if (kt * kTile + kTile > s.tk) {  // rows past the sequence: zeros
        for (int at = (s.tk - kt * kTile) * 8 + lane; at < kTile * 8; at += 32)
#pragma unroll
          for (int c = 0; c < CH; c++)
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(sv + c * M::kChunk + at * 16), "r"(0) : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
#pragma unroll
      for (int t = 0; t < 2; t++) {
        if (st[t].has(kt)) {
          ok = ok && sm100::bar_wait(pfull + 8 * t, np[t] & 1);
          if (!ok) break;
          sm100::tc_fence_after();
          if (lane == 0) {
            const uint64_t vb = desc_mn(sv, M::kChunk);
#pragma unroll
            for (int k = 0; k < kTile / 16; k++)
              sm100::tc_mma_ts(tmem + 256 + t * 128, tmem + t * kTile + 8 * k, vb + (uint64_t)(k * (2048 >> 4)), ido,
                               np[t] || k ? 1u : 0u);
          }
          np[t]++;
        }
        if (lane == 0 && i + 1 < steps && st[t].has(all.tile(i + 1))) score(t, ki % SLOTS);
        __syncwarp();
      }
      if (ok && lane == 0) {
        sm100::tc_commit(empty + 8 * (vi % SLOTS));
        if (i + 1 < steps) sm100::tc_commit(empty + 8 * (ki % SLOTS));
      }
      __syncwarp();
    }
    if (!ok && lane == 0) attn_failed();
    if (ok && lane == 0)
      for (int t = 0; t < 2; t++)
        if (np[t]) sm100::tc_commit(ofull + 8 * t);
  } else if (warp < 8) {  // ---- softmax of tile t, a thread per row
    const int t = warp >> 2, row = threadIdx.x & 127, tok = tok0 + t * per + row / pack, h = h0 + row % pack;
    const int p = back + tok;
    // positions of the warp's rows, of those that are rows of the sequence
    const int w0 = back + tok0 + t * per + (warp & 3) * 32 / pack, w1 = back + tok0 + t * per + ((warp & 3) * 32 + 31) / pack;
    const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * kTile, to = ts - t * kTile + 256 + t * 128;
    const float sc = a.scale * 1.4426950408889634f;
    float m = -INFINITY, l = 0.0f;
    int n = 0;  // steps done
    bool ok = true;
    for (int i = 0; i < steps; i++) {
      const int kt = all.tile(i), j0 = kt * kTile;
      if (!st[t].has(kt)) continue;
      ok = sm100::bar_wait(sfull + 8 * t, n & 1);
      if (!ok) break;
      sm100::tc_fence_after();
      uint32_t x[2][32];
      const bool edge = !(j0 + kTile - 1 <= w0 && (a.window == 0 || j0 > w1 - a.window || j0 + kTile <= a.sinks));
      const int hi = p - j0, lo = a.window ? p - a.window - j0 : -1, sk = a.sinks - j0;
      auto mask = [&](int c, uint32_t (&v)[32]) {
#pragma unroll
        for (int e = 0; e < 32; e++) {
          const int j = 32 * c + e;
          if (!(j <= hi && (j > lo || j < sk))) v[e] = 0xff800000u;
        }
      };
      float mx[4];
      sm100::tmem_ld32(ts, x[0]);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        sm100::tmem_ld_wait(x[c & 1]);
        if (c < 3) sm100::tmem_ld32(ts + 32 * c + 32, x[(c + 1) & 1]);
        else sm100::tmem_ld32(ts, x[0]);
        if (edge) mask(c, x[c & 1]);
        mx[c] = __uint_as_float(x[c & 1][0]);
#pragma unroll
        for (int e = 1; e < 32; e++) mx[c] = fmaxf(mx[c], __uint_as_float(x[c & 1][e]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool rise = (top - m) * sc > kRise;
      if (__any_sync(0xffffffffu, rise)) {
        const float k = rise ? sm100::ex2((m - top) * sc) : 1.0f;
        if (rise) m = top;
        l *= k;
        if (n) {
#pragma unroll
          for (int c = 0; c < DK / 32; c++) {
            uint32_t o[32];
            sm100::tmem_ld32(to + 32 * c, o);
            sm100::tmem_ld_wait(o);
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * k);
            sm100::tmem_st32(to + 32 * c, o);
          }
        }
      }
      const float2 sc2 = make_float2(sc, sc), mu = m == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(-m * sc, -m * sc);
      float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
      for (int c = 0; c < 4; c++) {
        uint32_t pk[16];
        sm100::tmem_ld_wait(x[c & 1]);
        if (c < 3) sm100::tmem_ld32(ts + 32 * c + 32, x[(c + 1) & 1]);
        if (edge) mask(c, x[c & 1]);
#pragma unroll
        for (int e = 0; e < 16; e++) {
          float2 v = sm100::fma2(make_float2(__uint_as_float(x[c & 1][2 * e]), __uint_as_float(x[c & 1][2 * e + 1])), sc2, mu);
          v = make_float2(sm100::ex2(v.x), sm100::ex2(v.y));
          sum[e & 1] = sm100::add2(sum[e & 1], v);
          pk[e] = pack2(v.x, v.y, (const E *)nullptr);
        }
        sm100::tmem_st16(ts + 16 * c, pk);
      }
      sum[0] = sm100::add2(sum[0], sum[1]);
      l += sum[0].x + sum[0].y;
      sm100::tmem_st_wait();
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::bar_arrive(pfull + 8 * t);
      n++;
    }
    if (n && ok) {
      ok = sm100::bar_wait(ofull + 8 * t, 0);
      sm100::tc_fence_after();
    }
    if (!ok && lane == 0) attn_failed();
    const bool live = tok < s.tq && ok;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    E *out = (E *)a.out + (long long)(s.q0 + tok) * a.o_ts + (long long)h * a.o_hs;
    bool fin = true;
#pragma unroll
    for (int c = 0; c < DK / 32; c++) {
      uint32_t o[32];
      if (n) {
        sm100::tmem_ld32(to + 32 * c, o);
        sm100::tmem_ld_wait(o);
      } else {
#pragma unroll
        for (int e = 0; e < 32; e++) o[e] = 0;
      }
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
          v[k] = l == 0.0f ? 0.0f : __uint_as_float(o[e + k]) * inv;
          fin = fin && fabsf(v[k]) <= 3.402823466e38f;
        }
        if (live)
          *reinterpret_cast<uint4 *>(out + 32 * c + e) =
              make_uint4(pack2(v[0], v[1], out), pack2(v[2], v[3], out), pack2(v[4], v[5], out), pack2(v[6], v[7], out));
      }
    }
    for (unsigned bad = __ballot_sync(0xffffffffu, live && !fin); bad; bad &= bad - 1) {
      const int from = __ffs(bad) - 1;
      slow_row<E, DK>(a, s, __shfl_sync(0xffffffffu, tok, from), __shfl_sync(0xffffffffu, h, from));
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 8) sm100::tmem_free(tmem, 512);
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? (PFN_cuTensorMapEncodeTiled_v12000)p
               : nullptr;
  }();
  return fn;
}

// A map of rows [rows][heads][dk] with strides ts and hs, in boxes of 64 dims x nh heads x nr rows.
bool make_map(CUtensorMap *m, const ork_b200_attn &a, const void *p, int heads, int rows, long long ts, long long hs, int nh, int nr) {
  const cuuint64_t dims[3] = {(cuuint64_t)a.dk, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)hs * 2, (cuuint64_t)ts * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)nh, (cuuint32_t)nr}, one[3] = {1, 1, 1};
  return encoder()(m, a.type == ORK_B200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                   const_cast<void *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class E, int DK>
cudaError_t launch_attn(const ork_b200_attn &a, cudaStream_t st) {
  const int G = a.H / a.Hkv, pack = std::min(G & -G, 8), per = kTile / pack, groups = a.H / pack;
  CUtensorMap mq, mk, mv;
  if (!encoder() || !make_map(&mq, a, a.q, a.H, a.q_rows, a.q_ts, a.q_hs, pack, per)) return cudaErrorInvalidValue;
  mk = mv = mq;  // without keys nothing is loaded
  if (a.max_k && (!make_map(&mk, a, a.k, a.Hkv, a.k_rows, a.k_ts, a.k_hs, 1, kTile) ||
                  !make_map(&mv, a, a.v, a.Hkv, a.k_rows, a.v_ts, a.v_hs, 1, kTile)))
    return cudaErrorInvalidValue;
  const int smem = Smem<DK>::kBytes;
  const cudaError_t e = smem_attr((const void *)attn_kernel<E, DK>, smem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)((a.max_q + 2 * per - 1) / (2 * per) * groups), a.nseq);
  attn_kernel<E, DK><<<grid, kThreads, smem, st>>>(a, mq, mk, mv, pack, groups);
  return cudaGetLastError();
}

}  // namespace

unsigned int attn_error_flag(bool reset) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_attn_error, sizeof v);
  if (reset && v) {
    const unsigned int z = 0;
    cudaMemcpyToSymbol(g_attn_error, &z, sizeof z);
  }
  return v;
}

ORKB_ERR_WORD_SETTER(attn_set_err_word)

}  // namespace orkb

using namespace orkb;

static int refuse(const char *why) {
  fprintf(stderr, "[ork] ERROR ork_b200_attn_async: %s\n", why);
  return -1;
}

extern "C" int ork_b200_attn_async(ork_npu *c, const ork_b200_attn *a) {
  if (!c || !a || !a->q || !a->k || !a->v || !a->out || !a->q_start || !a->k_start) return -1;
  if (a->type != ORK_B200_F16 && a->type != ORK_B200_BF16) return refuse("type is ORK_B200_F16 or ORK_B200_BF16");
  if (a->dk != 64 && a->dk != 128) return refuse("dk is 64 or 128");
  if (a->nseq < 1 || a->nseq > 65535 || a->Hkv < 1 || a->H < 1 || a->H > 65535 || a->H % a->Hkv)
    return refuse("nseq >= 1 and H a multiple of Hkv, neither above 65535");
  if (a->q_rows < 0 || a->k_rows < 0 || a->max_q < 0 || a->max_q > a->q_rows || a->max_k < 0 || a->max_k > a->k_rows)
    return refuse("max_q is 0 .. q_rows, max_k 0 .. k_rows");
  if (a->window < 0 || a->sinks < 0) return refuse("window and sinks are not negative");
  if (!(a->scale > 0.0f)) return refuse("scale is positive");
  for (long long st : {a->q_ts, a->q_hs, a->k_ts, a->k_hs, a->v_ts, a->v_hs, a->o_ts, a->o_hs})
    if (st < a->dk || st % 8) return refuse("strides are multiples of 8, dk at least");
  if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) % 16)
    return refuse("q, k, v and out are 16-byte aligned");
  DeviceGuard dg(c->device);
  if (!device_ptrs_ok(c, "ork_b200_attn_async", {a->q, a->k, a->v, a->out, a->q_start, a->k_start})) return -1;
  if (a->max_q == 0) return 0;
  ork_b200_attn d = *a;
  d.window = d.window < d.max_k ? d.window : 0;  // a window over everything is none
  d.sinks = std::min(d.sinks, d.max_k);
  const cudaError_t e = d.type == ORK_B200_F16
                            ? (d.dk == 64 ? launch_attn<__half, 64>(d, c->stream) : launch_attn<__half, 128>(d, c->stream))
                            : (d.dk == 64 ? launch_attn<__nv_bfloat16, 64>(d, c->stream) : launch_attn<__nv_bfloat16, 128>(d, c->stream));
  c->launches += 1;
  if (e != cudaSuccess) {
    log_err("ork_b200_attn_async", e);
    return -1;
  }
  return 0;
}
