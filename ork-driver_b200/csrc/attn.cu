// attn.cu -- attention of packed rows (prompts, or chunks after a cached prefix) with a sliding window and sink
// keys (include/ork_b200.h: ork_b200_attn_async), on the 5th-generation tensor cores.
//
// One CTA per SM takes items, two tiles of 128 query rows of one kv head, and streams the keys that any of them sees, 128
// at a time; the loads and products of an item begin under the end of the one before:
//   S = Q K^T     128 x 128 x dk, both operands in shared memory, S in tensor memory (fp32)
//   P = 2^(S sc - m + top)  online softmax, a thread per row; P goes back to tensor memory in 16 bits, over S
//   O += P V      128 x dk x 128, P from tensor memory, V in shared memory as it lies (N-major), O in tensor memory
// The two tiles alternate: while one is in its softmax the tensor cores work for the other. A row of a tile is a
// (token, head) pair, `pack` heads of the group (its largest power of two, at most 8) side by side, so that few tokens
// still fill a tile, and the tile's tokens, whose windows end at different keys, are few.
// Roles (three warpgroups): 0 and 1 the softmax and output of tile 0 and 1; of the third, warp 8 issues the products and
// warp 9 the TMA loads into a ring of 128 x dk slots that K and V tiles share. It gives most of its registers to the
// others, whose threads hold a row of S each.
// The running maximum follows only when it rises by more than 2^8, so that O is seldom scaled; weights stay below 2^8 (fp16:
// 2^15, kTop).
// Masks are applied to the tiles that hold an edge; tiles that no row sees are not visited.
// A value of V that is not finite reaches rows that do not see it (0 * inf): a row whose result is not finite is
// computed again, from its visible keys alone, by its warp, once the CTA has no items left and nobody waits for it (in
// between, some hundred thousand keys would outlast the bounded waits). Such rows are listed in their own places in out.
// Rows of V past the sequence are cleared in shared memory.
//
// Bound by the chain softmax -> P V -> Q K^T of each tile: a step of two tiles and 128 keys of 128 dims takes 3900
// clocks, of which the tensor cores work 2050 to 2450 and the exponential unit 2050 (both 56 % active over the launch).
// 16384 tokens, all visible, 16 heads of 128, bf16: 0.86 to 1.04 ms, 1.05 to 1.27 PFLOP/s; 8192 tokens of 64 heads, window
// 1024: 370 to 410 us. Measured against: a step of 64 keys with two places for S, 1.58 ms; P handed over by halves, 1.02 ms;
// two threads a row, 0.93 to 1.02 ms.
//
// Every wait is bounded; one that expires records an error and the roles fall through to the common exit, which waits,
// bounded too, for the copies and products still on their way.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

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
  if (!ok) {
    atomicOr(&g_attn_error, 1u);
    err_word_set();
  }
  return ok;
}

constexpr int kTile = 128;    // query rows of a tile, keys of a step
constexpr int kThreads = 384;
constexpr float kRise = 8.0f;  // log2 of the rise of a maximum that O is scaled for
// log2 of the weight of the running maximum. With kRise it fills fp16's range to 2^15, so that a weight is lost to the
// second product below 2^-32 of the maximum's, not 2^-25: 131072 of those would be 0.4 % of a row. bf16 needs none of it.
template <class E>
constexpr float kTop = std::is_same<E, __half>::value ? 7.0f : 0.0f;

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

__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if any is
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Shared memory: the two Q tiles, the ring, 4 KB for each softmax warp's output, barriers, items, the tensor memory's
// address, each softmax warp's list of rows to compute again.
template <int DK>
struct Smem {
  static constexpr int kSlots = DK == 128 ? 4 : 8;
  static constexpr int kTileBytes = kTile * DK * 2, kChunk = kTile * 128;  // a 64-column block of a tile
  static constexpr int kStage = (2 + kSlots) * kTileBytes, kBar = kStage + 8 * 4096;
  static constexpr int kBars = 2 + 2 * kSlots + 6 + 4 + 2, kItem = kBar + kBars * 8;
  static constexpr int kList = kItem + 2 * 80 + 16, kBytes = 1024 + kList + 8 * 16;
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

// 16 bytes of a row as fp32
template <class E>
__device__ __forceinline__ void widen8(const uint4 &w, float (&x)[8]) {
  const E *e = reinterpret_cast<const E *>(&w);
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = to_f32(e[i]);
}

// Rows computed from their visible keys alone, by a warp, kAgain of them over the same keys: 32 keys at a time, a lane's
// own in the first product, its DK / 32 dims in the second. Row r has its query at q[r], its output at out[r] and the
// position p[r] (-1: no row); qs: room for their queries in shared memory. Where every row sees one infinite value, 16384
// tokens of 16 heads of 128 take 93 ms instead of 0.9; a row at a time 260 ms, eight rows 82.
constexpr int kAgain = 4;
template <class E, int DK>
__device__ __forceinline__ void exact_rows(const ork_b200_attn &a, const Seq &s, int kvh, const E *const (&q)[kAgain],
                                           E *const (&out)[kAgain], const int (&p)[kAgain], float *qs) {
  constexpr int PER = DK / 32;
  const int lane = threadIdx.x & 31;
  int first = 0x7fffffff, last = -1;
  float o[kAgain][PER], m[kAgain], l[kAgain];
  __syncwarp();
#pragma unroll
  for (int r = 0; r < kAgain; r++) {
    m[r] = -INFINITY, l[r] = 0.0f;
    if (p[r] >= 0) first = min(first, p[r]), last = max(last, p[r]);
#pragma unroll
    for (int u = 0; u < PER; u++) {
      o[r][u] = 0.0f;
      qs[r * DK + PER * lane + u] = p[r] >= 0 ? to_f32(q[r][PER * lane + u]) * a.scale : 0.0f;
    }
  }
  __syncwarp();
  // what any of them sees: ns sinks, then lo .. last
  const int lo = a.window ? max(0, first - a.window + 1) : 0, ns = min(a.sinks, lo), n = ns + last + 1 - lo;
  const uint32_t sq = sm100::smem_addr(qs);
  const E *kb = (const E *)a.k + s.k0 * a.k_ts + kvh * a.k_hs, *vb = (const E *)a.v + s.k0 * a.v_ts + kvh * a.v_hs + PER * lane;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = min(i0 + lane, n - 1), j = i < ns ? i : i - ns + lo;
    float w[kAgain] = {};
    uint4 kw[DK / 8];
#pragma unroll
    for (int d = 0; d < DK / 8; d++) kw[d] = reinterpret_cast<const uint4 *>(kb + j * a.k_ts)[d];
#pragma unroll
    for (int d = 0; d < DK / 8; d++) {
      float kd[8];
      widen8<E>(kw[d], kd);
#pragma unroll
      for (int r = 0; r < kAgain; r++) {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
          float4 f;  // read where it is used, there are more than registers hold
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
                       : "r"(sq + (r * DK + 8 * d + h) * 4)
                       : "memory");
          w[r] = fmaf(f.x, kd[h], fmaf(f.y, kd[h + 1], fmaf(f.z, kd[h + 2], fmaf(f.w, kd[h + 3], w[r]))));
        }
      }
    }
    bool done = true;
#pragma unroll
    for (int r = 0; r < kAgain; r++) {
      const bool see = i0 + lane < n && j <= p[r] && (a.window == 0 || j > p[r] - a.window || j < a.sinks);
      float mn = see ? w[r] : -INFINITY;
      for (int d = 16; d; d >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
      mn = fmaxf(m[r], mn);
      const float c = m[r] == mn ? 1.0f : expf(m[r] - mn), e = expf(w[r] - (mn == -INFINITY ? 0.0f : mn));
      float t = see ? e : 0.0f;
      for (int d = 16; d; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
      l[r] = l[r] * c + t;
      m[r] = mn;
#pragma unroll
      for (int u = 0; u < PER; u++) o[r][u] *= c;
      w[r] = see ? e : -1.0f;  // no weight: what the row does not see must not reach it
      done = done && (p[r] < 0 || l[r] != l[r]);
    }
    if (done) break;  // a logit that is a NaN or infinite makes its row NaN whatever follows
    const int cnt = min(32, n - i0);
#pragma unroll 8
    for (int y = 0; y < cnt; y++) {
      const E *v = vb + __shfl_sync(0xffffffffu, j, y) * a.v_ts;
      float x[PER];
#pragma unroll
      for (int u = 0; u < PER; u++) x[u] = to_f32(v[u]);
#pragma unroll
      for (int r = 0; r < kAgain; r++) {
        const float wy = __shfl_sync(0xffffffffu, w[r], y);
        if (!(wy < 0.0f))
#pragma unroll
          for (int u = 0; u < PER; u++) o[r][u] = fmaf(wy, x[u], o[r][u]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kAgain; r++)
    if (p[r] >= 0)
#pragma unroll
      for (int u = 0; u < PER; u++) out[r][PER * lane + u] = from_f32<E>(l[r] == 0.0f ? 0.0f : o[r][u] / l[r]);
}

// An item: a head group of a sequence, and a pair of tiles of its tokens.
struct Item {
  Seq s;
  int kvh, h0, tok0, back;  // first head and token; position of token 0
  Steps st[2], all;         // of the tiles, of either
  int end;                  // there are no more items
  int no;                   // its number
};
static_assert(sizeof(Item) <= 80, "an item's place");
// Items are numbered by tile pair (the last ones first: they see most), then sequence, then head group. False: nothing
// to do.
__device__ __forceinline__ bool item_of(const ork_b200_attn &a, int it, int pairs, int lp, int groups, Item *o) {
  const int hg = it % groups, sq = it / groups % a.nseq, pair = pairs - 1 - it / groups / a.nseq, per = kTile >> lp;
  o->h0 = hg << lp, o->kvh = o->h0 / (a.H / a.Hkv), o->tok0 = pair * 2 * per;
  if (!seq_of(a, sq, &o->s) || o->tok0 >= o->s.tq) return false;
  o->back = o->s.tk - o->s.tq;
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int t0 = o->tok0 + t * per, t1 = min(t0 + per, o->s.tq) - 1;
    o->st[t] = steps_of(o->back + t0, t0 <= t1 ? o->back + t1 : -1, a.window, a.sinks);
  }
  o->all = steps_of(o->back + o->tok0, o->back + min(o->tok0 + 2 * per, o->s.tq) - 1, a.window, a.sinks);
  o->end = 0;
  o->no = it;
  return true;
}

template <class E, int DK>
__global__ void __launch_bounds__(kThreads, 1)
    attn_kernel(const ork_b200_attn a, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                const __grid_constant__ CUtensorMap mv, int lp, int groups, int pairs, int items, unsigned int *count) {
  using M = Smem<DK>;
  constexpr int SLOTS = M::kSlots, CH = DK / 64;
  extern __shared__ uint8_t raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sq = sm100::smem_addr(smem), sring = sq + 2 * M::kTileBytes, bars = sq + M::kBar;
  const uint32_t qfull = bars, qempty = bars + 8, full = bars + 16, empty = full + 8 * SLOTS, sfull = empty + 8 * SLOTS,
                 pfull = sfull + 16, ofull = pfull + 16, ifull = ofull + 16, iempty = ifull + 16, done = iempty + 16;
  Item *place = (Item *)(smem + M::kItem);  // [2]
  uint32_t *slot = (uint32_t *)(smem + M::kItem + 2 * 80);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int per = kTile >> lp;

  if (warp == 9 && lane < 3)
    asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &mq : lane == 1 ? &mk : &mv) : "memory");
  if (threadIdx.x == 0) {
    sm100::bar_init(qfull, 1), sm100::bar_init(qempty, 1);
    for (int i = 0; i < SLOTS; i++) sm100::bar_init(full + 8 * i, 1), sm100::bar_init(empty + 8 * i, 1);
    for (int t = 0; t < 2; t++) {
      sm100::bar_init(sfull + 8 * t, 1), sm100::bar_init(pfull + 8 * t, 4);
      sm100::bar_init(ofull + 8 * t, 1), sm100::bar_init(ifull + 8 * t, 1), sm100::bar_init(iempty + 8 * t, 9);
    }
    sm100::bar_init(done, 1);
    sm100::bar_init_fence();
  }
  // the items of which the warp has rows to compute again: how many, the latest one's number and first such row. That row
  // in out holds their bits, and the number and first row of the item before.
  int4 *again = (int4 *)(smem + M::kList) + (warp & 7);
  if (warp < 8 && lane == 0) *again = make_int4(0, 0, 0, 0);
  if (warp == 8) sm100::tmem_alloc(sm100::smem_addr(slot), 512);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *slot;
  bool ok = true;
  Item w;
  // registers: 2 x 216 + 72 = 3 x 168, what the block was launched with
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 9 && lane == 0) {  // ---- items, and loads: Q, then K of step 0, V of step 0, K of step 1, ...
      int nq = 0, g = 0, k = 0;    // Q pairs, ring tiles, items so far
      for (int it = blockIdx.x; ok; it = (int)(gridDim.x + atomicAdd(count, 1u))) {
        w.end = it >= items;
        if (!w.end && !item_of(a, it, pairs, lp, groups, &w)) continue;
        ok = k < 2 || sm100::bar_wait(iempty + 8 * (k & 1), ((k >> 1) - 1) & 1);
        if (!ok) break;
        place[k & 1] = w;
        sm100::bar_arrive(ifull + 8 * (k & 1));
        k++;
        if (w.end) break;
        if (w.all.count() == 0) continue;
        ok = nq == 0 || sm100::bar_wait(qempty, (nq - 1) & 1);
        if (!ok) break;
        nq++;
        sm100::bar_expect(qfull, 2 * M::kTileBytes);
        for (int t = 0; t < 2; t++)
          for (int c = 0; c < CH; c++)
            sm100::tma_load_3d(sq + t * M::kTileBytes + c * M::kChunk, &mq, 64 * c, w.h0, w.s.q0 + w.tok0 + t * per, qfull);
        for (int i = 0; i < 2 * w.all.count(); i++, g++) {
          const int sl = g % SLOTS;
          ok = g < SLOTS || sm100::bar_wait(empty + 8 * sl, (g / SLOTS - 1) & 1);
          if (!ok) break;
          sm100::bar_expect(full + 8 * sl, M::kTileBytes);
          for (int c = 0; c < CH; c++)
            sm100::tma_load_3d(sring + sl * M::kTileBytes + c * M::kChunk, i & 1 ? (const void *)&mv : (const void *)&mk, 64 * c,
                               w.kvh, w.s.k0 + w.all.tile(i >> 1) * kTile, full + 8 * sl);
        }
      }
      if (!ok) attn_failed();
      // the last CTA to be done with the count leaves it zero for the next launch
      __threadfence();
      if (atomicInc(count + 1, gridDim.x - 1) == gridDim.x - 1) *count = 0;
      // no copy is on its way when the CTA ends, whoever gave up
      if (nq) sm100::bar_wait(qfull, (nq - 1) & 1);
      for (int i = max(0, g - SLOTS); i < g; i++) sm100::bar_wait(full + 8 * (i % SLOTS), (i / SLOTS) & 1);
    } else if (warp == 8) {  // ---- products, issued by one elected lane from operands the whole warp agrees on
      constexpr uint32_t ids = inst_desc<E>(kTile, false), ido = inst_desc<E>(DK, true);
      constexpr uint32_t kSlot = M::kTileBytes >> 4;
      const uint64_t qd = desc_k(sq), kd = desc_k(sring), vd = desc_mn(sring, M::kChunk);
      int nq = 0, g = 0, np[2] = {0, 0};  // Q pairs, ring slot of the next K, P tiles so far
      int gp = 0;                         // parity of the ring's round at g
      auto wait_full = [&](int off) {     // ring tile g + off, off < SLOTS
        const int sl = g + off < SLOTS ? g + off : g + off - SLOTS;
        return sm100::bar_wait(full + 8 * sl, g + off < SLOTS ? gp : gp ^ 1);
      };
      auto slot_of = [&](int off) { return (uint32_t)(g + off < SLOTS ? g + off : g + off - SLOTS); };
      // S of tile t from the K in slot sl
      auto score = [&](int t, uint32_t sl) {
        const uint64_t qa = qd + t * kSlot, kb = kd + sl * kSlot;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
          for (int k = 0; k < 4; k++)
            sm100::tc_mma(tmem + t * kTile, qa + (c * (M::kChunk >> 4) + 2 * k), kb + (c * (M::kChunk >> 4) + 2 * k), ids, c | k ? 1u : 0u);
        sm100::tc_commit(sfull + 8 * t);
      };
      for (int k = 0; ok; k++) {
        ok = sm100::bar_wait(ifull + 8 * (k & 1), (k >> 1) & 1);
        if (!ok) break;
        const Item *pl = place + (k & 1);
        auto steps_at = [&](const Steps &x) { return Steps{sm100::uniform(x.ns), sm100::uniform(x.lo), sm100::uniform(x.hi)}; };
        const Steps all = steps_at(pl->all), mine[2] = {steps_at(pl->st[0]), steps_at(pl->st[1])};
        const int tk = sm100::uniform(pl->s.tk), end = sm100::uniform(pl->end);
        if (lane == 0) sm100::bar_arrive(iempty + 8 * (k & 1));
        if (end) break;
        const int steps = all.count();
        if (steps == 0) continue;
        bool any[2] = {false, false};
        ok = sm100::bar_wait(qfull, nq & 1) && wait_full(0);
        if (!ok) break;
        nq++;
        sm100::tc_fence_after();
        if (sm100::elect_one()) {
#pragma unroll
          for (int t = 0; t < 2; t++)
            if (mine[t].has(all.tile(0))) score(t, (uint32_t)g);
          sm100::tc_commit(empty + 8 * g);
          if (steps == 1) sm100::tc_commit(qempty);
        }
        __syncwarp();
        for (int i = 0; i < steps && ok; i++) {
          const int kt = all.tile(i);
          const bool more = i + 1 < steps;
          const uint32_t vsl = slot_of(1), ksl = slot_of(2);
          ok = wait_full(1) && (!more || wait_full(2));
          if (!ok) break;
          if (kt * kTile + kTile > tk) {  // rows past the sequence: zeros
            const uint32_t sv = sring + vsl * M::kTileBytes;
            for (int at = (tk - kt * kTile) * 8 + lane; at < kTile * 8; at += 32)
#pragma unroll
              for (int c = 0; c < CH; c++)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(sv + c * M::kChunk + at * 16), "r"(0) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          const int next = more ? all.tile(i + 1) : 0;
#pragma unroll
          for (int t = 0; t < 2; t++) {
            const bool now = mine[t].has(kt), then = more && mine[t].has(next);
            if (now) {
              ok = ok && sm100::bar_wait(pfull + 8 * t, np[t] & 1);
              if (!ok) break;
              np[t]++;
              sm100::tc_fence_after();
            }
            if (sm100::elect_one()) {
              if (now) {
                const uint64_t vb = vd + vsl * kSlot;
#pragma unroll
                for (int e = 0; e < kTile / 16; e++)
                  sm100::tc_mma_ts(tmem + 256 + t * 128, tmem + t * kTile + 8 * e, vb + e * (2048 >> 4), ido, any[t] || e ? 1u : 0u);
              }
              if (then) score(t, ksl);
              if (t == 1) {
                sm100::tc_commit(empty + 8 * vsl);
                if (more) sm100::tc_commit(empty + 8 * ksl);
                if (i + 2 == steps) sm100::tc_commit(qempty);
              }
            }
            __syncwarp();
            any[t] = any[t] || now;
          }
          g += 2;
          if (g >= SLOTS) g -= SLOTS, gp ^= 1;
        }
        if (!ok) break;
        if (sm100::elect_one()) {
#pragma unroll
          for (int t = 0; t < 2; t++)
            if (any[t]) sm100::tc_commit(ofull + 8 * t);
        }
        __syncwarp();
      }
      if (!ok && lane == 0) attn_failed();
      if (sm100::elect_one()) sm100::tc_commit(done);  // nor a product
      __syncwarp();
      sm100::bar_wait(done, 0);
    }
  } else {  // ---- softmax of tile t, a thread per row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = warp >> 2, wrow = (warp & 3) * 32, row = wrow + lane;
    const uint32_t ts = tmem + ((uint32_t)wrow << 16) + t * kTile, to = ts - t * kTile + 256 + t * 128;
    const uint32_t stage = sq + M::kStage + warp * 4096;
    const float sc = a.scale * 1.4426950408889634f;
    const float2 sc2 = make_float2(sc, sc);
    int ns = 0, no = 0;  // steps and items with any so far
    for (int k = 0; ok; k++) {
      ok = sm100::bar_wait(ifull + 8 * (k & 1), (k >> 1) & 1);
      if (!ok) break;
      const Item *pl = place + (k & 1);
      if (sm100::uniform(pl->end)) break;
      const int tok0 = sm100::uniform(pl->tok0) + t * per, pos0 = sm100::uniform(pl->back) + tok0, p = pos0 + (row >> lp);
      // a tile of keys has no edge for the warp's rows if it begins at `inner` or before, and after `outer` or before the
      // sinks' end
      const int inner = pos0 + (wrow >> lp) - kTile + 1, outer = pos0 + ((wrow + 31) >> lp) - a.window;
      const int first = ns, sinks = sm100::uniform(pl->st[t].ns), lo = sm100::uniform(pl->st[t].lo), last = sm100::uniform(pl->st[t].hi);
      float m = -INFINITY, l = 0.0f;
      for (int kt = sinks ? 0 : lo; kt <= last; kt = kt + 1 == sinks ? lo : kt + 1) {
        const int j0 = kt * kTile;
        ok = sm100::bar_wait(sfull + 8 * t, ns & 1);
        if (!ok) break;
        sm100::tc_fence_after();
        const bool edge = !(j0 <= inner && (a.window == 0 || j0 > outer || j0 + kTile <= a.sinks));
        uint32_t x[4][32];
        float mx[4];
        auto load = [&](int c) { sm100::tmem_ld32(ts + 32 * c, x[c]); };
        auto mask_max = [&](int c) {
          if (edge) {  // the row's visible columns as bits: up to its position, after the window's begin or among the sinks
            auto below = [&](int n) { return n <= 32 * c ? 0u : n >= 32 * c + 32 ? 0xffffffffu : (1u << (n - 32 * c)) - 1u; };
            const uint32_t see = below(p - j0 + 1) & (~below(a.window ? p - a.window - j0 + 1 : 0) | below(a.sinks - j0));
#pragma unroll
            for (int e = 0; e < 32; e++)
              if (!(see >> e & 1u)) x[c][e] = 0xff800000u;
          }
#pragma unroll
          for (int q = 0; q < 4; q++) {
            auto f = [&](int e) { return __uint_as_float(x[c][e + q]); };
            mx[q] = max3(c ? mx[q] : f(0), f(0), f(4));
            mx[q] = max3(mx[q], f(8), f(12));
            mx[q] = max3(mx[q], f(16), f(20));
            mx[q] = max3(mx[q], f(24), f(28));
          }
        };
        float2 sum = make_float2(0.0f, 0.0f);
        auto weights = [&](int c, float2 mu) {
          uint32_t pk[16];
          float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int e = 0; e < 16; e++) {
            float2 v = sm100::fma2(make_float2(__uint_as_float(x[c][2 * e]), __uint_as_float(x[c][2 * e + 1])), sc2, mu);
            v = make_float2(sm100::ex2(v.x), sm100::ex2(v.y));
            if (e & 1) part = sm100::add2(part, v);
            else sum = sm100::add2(sum, v);
            pk[e] = pack2(v.x, v.y, (const E *)nullptr);
          }
          sum = sm100::add2(sum, part);
          sm100::tmem_st16(ts + 16 * c, pk);
        };
        load(0), load(1);
        sm100::tmem_ld_wait(x[0]), sm100::tmem_ld_wait(x[1]);
        load(2), load(3);
        mask_max(0), mask_max(1);
        sm100::tmem_ld_wait(x[2]), sm100::tmem_ld_wait(x[3]);
        mask_max(2), mask_max(3);
        const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
        if (!(top < INFINITY)) l = __int_as_float(0x7fc00000);  // an infinity or a NaN among the logits: see exact_rows
        const bool rise = (top - m) * sc > kRise;
        if (__any_sync(0xffffffffu, rise)) {
          const float k2 = rise ? sm100::ex2((m - top) * sc) : 1.0f;
          if (rise) m = top;
          l *= k2;
          if (ns > first) {
#pragma unroll 1
            for (int c = 0; c < DK / 32; c++) {
              uint32_t o[32];
              sm100::tmem_ld32(to + 32 * c, o);
              sm100::tmem_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * k2);
              sm100::tmem_st32(to + 32 * c, o);
            }
          }
        }
        const float off = m == -INFINITY ? 0.0f : fmaf(-m, sc, kTop<E>);
        const float2 mu = make_float2(off, off);
#pragma unroll
        for (int c = 0; c < 4; c++) weights(c, mu);
        l += sum.x + sum.y;
        sm100::tmem_st_wait();
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::bar_arrive(pfull + 8 * t);
        ns++;
      }
      if (!ok) break;
      if (ns > first) {
        ok = sm100::bar_wait(ofull + 8 * t, no & 1);
        if (!ok) break;
        no++;
        sm100::tc_fence_after();
      }
      // rows of 64 columns through shared memory, so that a store writes whole 128-byte lines
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      bool fin = true;
      const Seq seq = {sm100::uniform(pl->s.q0), sm100::uniform(pl->s.tq), sm100::uniform(pl->s.k0), sm100::uniform(pl->s.tk)};
      const int h0 = sm100::uniform(pl->h0), no = sm100::uniform(pl->no);
      __syncwarp();
      if (lane == 0) sm100::bar_arrive(iempty + 8 * (k & 1));
      E *const base = (E *)a.out + (long long)seq.q0 * a.o_ts + 8 * (lane & 7);
#pragma unroll 1
      for (int c = 0; c < CH; c++) {
#pragma unroll 1
        for (int hf = 0; hf < 2; hf++) {
          uint32_t o[32];
          if (ns > first) {
            sm100::tmem_ld32(to + 64 * c + 32 * hf, o);
            sm100::tmem_ld_wait(o);
          }
#pragma unroll
          for (int e = 0; e < 32; e++) {
            const float v = ns > first ? __uint_as_float(o[e]) * inv : 0.0f;
            fin = fin && fabsf(v) <= 3.402823466e38f;
            o[e] = __float_as_uint(v);
          }
#pragma unroll
          for (int e = 0; e < 4; e++) {
            auto two = [&](int q) { return pack2(__uint_as_float(o[8 * e + q]), __uint_as_float(o[8 * e + q + 1]), base); };
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + (((4 * hf + e) ^ (lane & 7)) << 4)),
                         "r"(two(0)), "r"(two(2)), "r"(two(4)), "r"(two(6))
                         : "memory");
          }
        }
        __syncwarp();
#pragma unroll 2
        for (int j = 0; j < 8; j++) {
          const int rr = 4 * j + (lane >> 3), tk = tok0 + ((wrow + rr) >> lp), h = h0 + ((wrow + rr) & ((1 << lp) - 1));
          uint4 v;
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(stage + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4)));
          if (tk < seq.tq) *reinterpret_cast<uint4 *>(base + (long long)tk * a.o_ts + (long long)h * a.o_hs + 64 * c) = v;
        }
        __syncwarp();
      }
      const int tok = tok0 + (row >> lp), h = h0 + (row & ((1 << lp) - 1));
      const unsigned bad = __ballot_sync(0xffffffffu, tok < seq.tq && !fin);
      if (bad && lane == __ffs(bad) - 1) {
        const int4 e = *again;
        *(int4 *)((E *)a.out + (long long)(seq.q0 + tok) * a.o_ts + (long long)h * a.o_hs) = make_int4((int)bad, e.y, e.z, 0);
        *again = make_int4(e.x + 1, no, lane, 0);
      }
    }
    __syncwarp();
    // whatever out may hold by now (rows that a caller laid over one another), every item and row is checked
    int4 e = *again;
    for (int left = ok ? e.x : 0; left && (unsigned)e.y < (unsigned)items && item_of(a, e.y, pairs, lp, groups, &w); left--) {
      auto token = [&](int rr) { return w.tok0 + t * per + ((wrow + rr) >> lp); };
      auto place_of = [&](int rr, long long ts, long long hs) {
        return (long long)(w.s.q0 + token(rr)) * ts + (long long)(w.h0 + ((wrow + rr) & ((1 << lp) - 1))) * hs;
      };
      if (token(e.z & 31) >= w.s.tq) break;
      e = *(const int4 *)((const E *)a.out + place_of(e.z & 31, a.o_ts, a.o_hs));
      for (unsigned bad = (unsigned)e.x; bad;) {
        const E *q[kAgain];
        E *out[kAgain];
        int p[kAgain];
#pragma unroll
        for (int r = 0; r < kAgain; r++) {
          const int rr = bad ? __ffs(bad) - 1 : 0;
          p[r] = bad && token(rr) < w.s.tq ? w.back + token(rr) : -1;
          q[r] = (const E *)a.q + place_of(rr, a.q_ts, a.q_hs), out[r] = (E *)a.out + place_of(rr, a.o_ts, a.o_hs);
          bad &= bad - 1;
        }
        exact_rows<E, DK>(a, w.s, w.kvh, q, out, p, (float *)(smem + M::kStage + warp * 4096));
      }
    }
    if (!ok && lane == 0) attn_failed();
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
cudaError_t launch_attn(const ork_b200_attn &a, unsigned int *count, cudaStream_t st) {
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
  const int pairs = (a.max_q + 2 * per - 1) / (2 * per);
  const long long items = (long long)pairs * groups * a.nseq;
  if (items > 0x7fffff00) return cudaErrorInvalidValue;
  attn_kernel<E, DK><<<(int)std::min<long long>(items, 148), kThreads, smem, st>>>(a, mq, mk, mv, __builtin_ctz(pack), groups, pairs, (int)items, count);
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
  if (((uintptr_t)a->q_start | (uintptr_t)a->k_start) % 4) return refuse("q_start and k_start are 4-byte aligned");
  DeviceGuard dg(c->device);
  if (!device_ptrs_ok(c, "ork_b200_attn_async", {a->q, a->k, a->v, a->out, a->q_start, a->k_start})) return -1;
  if (a->max_q == 0) return 0;
  ork_b200_attn d = *a;
  d.window = d.window < d.max_k ? d.window : 0;  // a window over everything is none
  d.sinks = std::min(d.sinks, d.max_k);
  unsigned int *count = zeroed_counts(c, "ork_b200_attn_async", 0);
  if (!count) return -1;
  const bool f16 = d.type == ORK_B200_F16, wide = d.dk == 128;
  const cudaError_t e = f16 ? (wide ? launch_attn<__half, 128>(d, count, c->stream) : launch_attn<__half, 64>(d, count, c->stream))
                            : (wide ? launch_attn<__nv_bfloat16, 128>(d, count, c->stream)
                                    : launch_attn<__nv_bfloat16, 64>(d, count, c->stream));
  c->launches += 1;
  if (e != cudaSuccess) {
    log_err("ork_b200_attn_async", e);
    return -1;
  }
  return 0;
}
