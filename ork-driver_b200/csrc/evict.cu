// evict.cu -- eviction from a cache by accumulated attention weight (include/ork_b200.h: ork_b200_evict_async).
//
// A token's key orders it: the first `sinks` and last `recent` tokens have the largest key, others their score's
// bits mapped to an unsigned word of the same order (a NaN's: minus infinity's). The kept ones are those above a threshold
// key, and of those equal to it the lowest slots. Two launches:
//   evict_pick  a cluster of CTAs per (sequence, kv head) finds the threshold in three digits of 11, 11 and 10 bits: each pass counts the
//               keys that share the bits found so far, every CTA of its part of the tokens, and adds the counts up through
//               distributed shared memory. Keys stay in shared memory between the passes when they fit. It ends with the
//               number of kept tokens, and of kept ones equal to the threshold, before each chunk of kChunk tokens.
//   evict_move  a CTA per chunk: the places of its kept tokens by a prefix sum over the chunk, then their rows, plane by
//               plane, with as many threads on a row as it has 16-byte (4-byte) words.
// The counts are integers, so no order of adding changes anything.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>

#include "errword.cuh"
#include "ork_internal.h"
#include "ork_structs.h"
#include "sm100.cuh"

namespace orkb {

__device__ unsigned int g_evict_error = 0;

namespace {

constexpr int kThreads = 1024;  // of evict_pick
constexpr int kChunk = 512;     // tokens of a CTA of evict_move, one a thread
// Words that a thread of evict_move has on their way: two, and four CTAs an SM, whose 32 registers a thread leave no more.
// 16 x 8 heads of up to 32768 4-bit tokens, moved and read back: 239 us; four words and three CTAs 242, eight and two 258.
constexpr int kMoves = 2;
constexpr int kCluster = 8;     // CTAs that pick together, at most
constexpr int kHeld = 24576;    // keys that a CTA of evict_pick holds
constexpr int kDigits = 2048;   // of a pass, two a thread: 11, 11 and 10 bits
static_assert(kDigits == 2 * kThreads);

// What evict_pick leaves for evict_move, per (sequence, kv head): the threshold, how many of those equal to it are kept,
// and per chunk the kept tokens above it and those equal to it before the chunk.
struct Picked {
  uint32_t threshold;
  int equal, n, pad;
};

__device__ __forceinline__ uint32_t key_of(float score, int j, int n, int sinks, int recent) {
  if (j < sinks || j >= n - recent) return 0xffffffffu;
  const uint32_t b = __float_as_uint(isnan(score) ? -INFINITY : score + 0.0f);  // -0 counts as 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ int held_len(const ork_b200_evict &e, int s) {  // 0 (reported) where it cannot be
  const int n = e.len[s];
  if (n >= 0 && n <= e.max_len) return n;
  if (threadIdx.x == 0) {
    atomicOr(&g_evict_error, 1u);
    err_word_set();
  }
  return 0;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int2 remote_int2(const int *p, uint32_t rank) {
  uint32_t at;
  int2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(sm100::smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ int remote_int(const int *p, uint32_t rank) {
  uint32_t at;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(sm100::smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// exclusive prefix sum over the block, *total: the sum; blocks of up to 1024 threads
__device__ __forceinline__ int block_scan(int v, int *red, int *total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[w] = x;
  __syncthreads();
  if (w == 0) {
    int y = lane < nw ? red[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    red[lane] = y;
  }
  __syncthreads();
  *total = red[nw - 1];
  return x - v + (w ? red[w - 1] : 0);
}

// blockIdx.y: (sequence, kv head); the CTAs of its cluster take runs of whole chunks of its tokens.
__global__ void __launch_bounds__(kThreads) evict_pick(const ork_b200_evict e, Picked *picked, int2 *before, int chunks, int hold) {
  extern __shared__ uint32_t keys[];
  __shared__ __align__(8) int hist[2][kDigits];
  __shared__ int sum[128], red[32], ends[2];
  __shared__ int s_digit, s_left;
  const int sh = blockIdx.y, tid = threadIdx.x;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int n = held_len(e, sh / e.Hkv), m = min(n, e.keep), all = (n + kChunk - 1) / kChunk;
  const int c0 = (int)((long long)all * rank / size), c1 = (int)((long long)all * (rank + 1) / size);
  const int j0 = c0 * kChunk, j1 = min(n, c1 * kChunk);
  const float *score = e.score + (size_t)sh * e.cap;
  auto key_at = [&](int j) { return hold ? keys[j - j0] : key_of(score[j], j, n, e.sinks, e.recent); };
  uint32_t prefix = 0;
  int left = m;  // of the keys that share the prefix, how many are kept
  if (n > m) {
    for (int pass = 0; pass < 3; pass++) {
      const int bits = pass < 2 ? 11 : 10, shift = max(0, 21 - 11 * pass);
      int *h = hist[pass & 1];  // the other one may still be read by a CTA that is behind
      reinterpret_cast<int2 *>(h)[tid] = make_int2(0, 0);
      __syncthreads();
      for (int b = j0; b < j1; b += 8 * kThreads) {
        uint32_t ks[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
          const int j = b + u * kThreads + tid;
          ks[u] = j < j1 ? (pass == 0 || !hold ? __float_as_uint(score[j]) : keys[j - j0]) : 0u;
        }
#pragma unroll
        for (int u = 0; u < 8; u++) {
          const int j = b + u * kThreads + tid;
          if (b + u * kThreads >= j1) break;
          if (j >= j1) continue;
          uint32_t k = ks[u];
          if (pass == 0 || !hold) k = key_of(__uint_as_float(k), j, n, e.sinks, e.recent);
          if (pass == 0 && hold) keys[j - j0] = k;
          // an addition each, equal digits or not: one for the lanes that share one, found by ballots, was slower even
          // with every score the same (253 us the whole call instead of 245)
          if (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits))) atomicAdd(&h[(k >> shift) & ((1 << bits) - 1)], 1);
        }
      }
      __syncthreads();
      if (size > 1) cluster_sync();
      const int d = kDigits - 2 - 2 * tid;  // this thread's digits: d + 1, then d
      int2 v = *reinterpret_cast<const int2 *>(&h[d]);
      for (uint32_t q = 1; q < size; q++) {
        const int2 o = remote_int2(&h[d], (rank + q) % size);
        v.x += o.x, v.y += o.y;
      }
      int all_of;
      const int above = block_scan(v.x + v.y, red, &all_of);
      if (above < left && above + v.x + v.y >= left) {
        const bool low = above + v.y < left;
        s_digit = low ? d : d + 1, s_left = left - above - (low ? v.y : 0);
      }
      __syncthreads();
      prefix |= (uint32_t)s_digit << shift;
      left = s_left;
    }
  }
  // the kept tokens before each chunk: above the threshold, and equal to it. A warp counts a chunk.
  const int lane = tid & 31;
  int2 *out = before + (size_t)sh * chunks;
  int above = 0, equal = 0;
  for (int b = c0; b < c1; b += 32) {  // 32 chunks at a time
    __syncthreads();
    const int c = b + (tid >> 5);
    int a = 0, q = 0;
    if (c < c1)
      for (int j = c * kChunk + lane; j < min(j1, (c + 1) * kChunk); j += 32) {
        const uint32_t k = n > m ? key_at(j) : 1u;
        a += k > prefix, q += n > m && k == prefix;
      }
    for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o), q += __shfl_xor_sync(0xffffffffu, q, o);
    if (lane == 0) sum[tid >> 5] = a, sum[32 + (tid >> 5)] = q;
    __syncthreads();
    if (tid < 32) {
      int x = sum[tid], y = sum[32 + tid];
      for (int o = 1; o < 32; o <<= 1) {
        const int xo = __shfl_up_sync(0xffffffffu, x, o), yo = __shfl_up_sync(0xffffffffu, y, o);
        if (tid >= o) x += xo, y += yo;
      }
      if (b + tid < c1) out[b + tid] = make_int2(above + x - sum[tid], equal + y - sum[32 + tid]);
      sum[64 + tid] = x, sum[96 + tid] = y;
    }
    __syncthreads();
    above += sum[64 + 31], equal += sum[96 + 31];
  }
  if (size > 1) {  // and those of the CTAs before this one
    if (tid == 0) ends[0] = above, ends[1] = equal;
    cluster_sync();
    int a = 0, q = 0;
    for (uint32_t i = 0; i < rank; i++) a += remote_int(&ends[0], i), q += remote_int(&ends[1], i);
    for (int c = c0 + tid; c < c1; c += kThreads) out[c].x += a, out[c].y += q;
    cluster_sync();  // nobody leaves while another may read its shared memory
  }
  if (rank == 0 && tid == 0) picked[sh] = Picked{n > m ? prefix : 0u, n > m ? left : 0, n, 0};
  sm100::dependents_launch();
}

// blockIdx.x: a chunk of the tokens of (sequence, kv head) blockIdx.y; the grid also covers the budget, whose unused
// places are filled. gridDim.z CTAs share a chunk's copies where there are few chunks (wide rows of one chat,
// 4001 tokens of 8 heads of 512 bytes: 16.5 us the call instead of 22.6).
__global__ void __launch_bounds__(kChunk, 4) evict_move(const ork_b200_evict e, const Picked *picked, const int2 *before, int chunks) {
  __shared__ int red[32], from[kChunk];
  sm100::dependency_wait();
  const int sh = blockIdx.y, tid = threadIdx.x, c = blockIdx.x;
  const int j = c * kChunk + tid;
  const float score = j < e.cap ? e.score[(size_t)sh * e.cap + j] : 0.0f;
  const Picked p = picked[sh];
  const int n = p.n, m = min(n, e.keep);
  const bool tell = blockIdx.z == 0;
  // the lengths are written here, where nothing reads them any more: len_out may be len
  if (tell && c == 0 && tid == 0 && e.len_out && sh % e.Hkv == 0) e.len_out[sh / e.Hkv] = m;
  if (tell && j < e.keep && j >= m) {
    if (e.kept) e.kept[(size_t)sh * e.keep + j] = -1;
    if (e.score_out) e.score_out[(size_t)sh * e.dcap + j] = 0.0f;
  }
  if (c * kChunk >= n) return;
  const int2 b = before[(size_t)sh * chunks + c];
  const uint32_t k = j < n ? key_of(score, j, n, e.sinks, e.recent) : 0u;
  int total;
  const bool eq = n > m && j < n && k == p.threshold;
  const int ne = block_scan(eq, red, &total);
  const bool keep = j < n && (n <= m || k > p.threshold || (eq && b.y + ne < p.equal));
  const int at = block_scan(keep, red, &total), first = b.x + min(b.y, p.equal);  // kept before the chunk
  if (keep) {
    from[at] = j;
    if (tell && e.kept) e.kept[(size_t)sh * e.keep + first + at] = j;
    if (tell && e.score_out) e.score_out[(size_t)sh * e.dcap + first + at] = score;
  }
  __syncthreads();
  if (e.nplanes == 0) return;
  // the planes side by side, the warps in turn: their rows are all on their way at once
  const int warp = tid >> 5, q = warp % e.nplanes, mates = (kChunk / 32 - q + e.nplanes - 1) / e.nplanes;
  const int i00 = (warp / e.nplanes + mates * blockIdx.z) * 32 + (tid & 31), hop = mates * 32 * gridDim.z;
  {
    const int bytes = e.row_bytes[q];
    const uint8_t *src = (const uint8_t *)e.src[q] + (size_t)sh * e.cap * bytes;
    uint8_t *dst = (uint8_t *)e.dst[q] + ((size_t)sh * e.dcap + first) * bytes;
    auto copy = [&](auto word) {
      using W = decltype(word);
      const int words = bytes / (int)sizeof(W), items = total * words;
      const bool shifts = (words & (words - 1)) == 0;
      const int by = __ffs(words) - 1;
      for (int i0 = i00; i0 < items; i0 += kMoves * hop) {
        W v[kMoves];
#pragma unroll
        for (int u = 0; u < kMoves; u++) {
          const int i = i0 + u * hop, row = shifts ? i >> by : i / words;
          if (i < items) v[u] = reinterpret_cast<const W *>(src + (size_t)from[row] * bytes)[i - row * words];
        }
#pragma unroll
        for (int u = 0; u < kMoves; u++) {
          const int i = i0 + u * hop;
          if (i < items) reinterpret_cast<W *>(dst)[i] = v[u];
        }
      }
    };
    // the rows of a chunk are written one after another
    if ((bytes | (uintptr_t)src | (uintptr_t)dst) % 16 == 0) copy(uint4());
    else if ((bytes | (uintptr_t)src | (uintptr_t)dst) % 8 == 0) copy(uint2());
    else copy(0u);
  }
}

}  // namespace

unsigned int evict_error_flag(bool reset) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_evict_error, sizeof v);
  if (reset && v) {
    const unsigned int z = 0;
    cudaMemcpyToSymbol(g_evict_error, &z, sizeof z);
  }
  return v;
}

ORKB_ERR_WORD_SETTER(evict_set_err_word)

}  // namespace orkb

using namespace orkb;

static int refuse(const char *why) {
  fprintf(stderr, "[ork] ERROR ork_b200_evict_async: %s\n", why);
  return -1;
}

extern "C" int ork_b200_evict_async(ork_npu *c, const ork_b200_evict *e) {
  if (!c || !e || !e->score || !e->len) return -1;
  if (e->nseq < 1 || e->Hkv < 1 || (long long)e->nseq * e->Hkv > 65535) return refuse("nseq, Hkv >= 1, their product at most 65535");
  if (e->cap < 1 || e->keep < 1 || e->dcap < e->keep) return refuse("cap, keep >= 1 and dcap >= keep");
  if (((uintptr_t)e->score | (uintptr_t)e->len | (uintptr_t)e->kept | (uintptr_t)e->score_out | (uintptr_t)e->len_out) % 4)
    return refuse("score, len, kept, score_out and len_out are 4-byte aligned");
  if (e->max_len < 0 || e->max_len > e->cap) return refuse("max_len is 0 .. cap");
  if (e->sinks < 0 || e->recent < 0 || (long long)e->sinks + e->recent > e->keep) return refuse("sinks + recent is 0 .. keep");
  if (e->nplanes < 0 || e->nplanes > ORK_B200_EVICT_PLANES) return refuse("too many planes");
  const size_t rows = (size_t)e->nseq * e->Hkv;
  for (int p = 0; p < e->nplanes; p++) {
    if (!e->src[p] || !e->dst[p]) return refuse("a plane is NULL");
    if (e->row_bytes[p] < 4 || e->row_bytes[p] > 65536 || e->row_bytes[p] % 4 || ((uintptr_t)e->src[p] | (uintptr_t)e->dst[p]) % 4)
      return refuse("rows are multiples of 4 bytes up to 65536, planes 4-byte aligned");
    for (int q = 0; q < e->nplanes; q++)
      if (e->src[q] && overlaps(e->dst[p], rows * e->dcap * e->row_bytes[p], e->src[q], rows * e->cap * e->row_bytes[q]))
        return refuse("a destination overlaps a source");
  }
  if (e->score_out && overlaps(e->score_out, rows * e->dcap * 4, e->score, rows * e->cap * 4))
    return refuse("score_out overlaps score");
  DeviceGuard dg(c->device);
  if (!device_ptrs_ok(c, "ork_b200_evict_async", {e->score, e->len, e->kept, e->score_out, e->len_out})) return -1;
  for (int p = 0; p < e->nplanes; p++)
    if (!device_ptrs_ok(c, "ork_b200_evict_async", {e->src[p], e->dst[p]})) return -1;
  const int chunks = (e->max_len + kChunk - 1) / kChunk, cover = (std::max(e->max_len, e->keep) + kChunk - 1) / kChunk;
  const size_t pb = (rows * sizeof(Picked) + 255) / 256 * 256;
  if (!work_block(c, "ork_b200_evict_async", &c->work, pb + rows * std::max(chunks, 1) * sizeof(int2))) return -1;
  Picked *picked = (Picked *)c->work.p;
  int2 *before = (int2 *)((uint8_t *)c->work.p + pb);
  ork_b200_evict d = *e;
  // CTAs a (sequence, head): about two waves of the SMs in all, 4096 tokens each or more
  int size = 1;
  while (size < kCluster && rows * size * 2 <= 2 * 148 && (long long)size * 4096 < e->max_len) size *= 2;
  const int part = ((chunks + size - 1) / size) * kChunk, hold = part <= kHeld;
  cudaError_t err = smem_attr((const void *)evict_pick, kHeld * 4);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at = {};
  cfg.gridDim = dim3(size, (unsigned)rows);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = hold ? (size_t)part * 4 : 0;
  cfg.stream = c->stream;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = size, at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if (err == cudaSuccess) err = cudaLaunchKernelEx(&cfg, evict_pick, d, picked, before, chunks, hold);
  if (err == cudaSuccess) {
    int share = 1;
    while (share < 8 && (long long)cover * (long long)rows * share < 148 * 2) share *= 2;
    cfg.gridDim = dim3(cover, (unsigned)rows, share);
    cfg.blockDim = dim3(kChunk);
    cfg.dynamicSmemBytes = 0;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    err = cudaLaunchKernelEx(&cfg, evict_move, d, (const Picked *)picked, (const int2 *)before, chunks);
  }
  c->launches += 2;
  if (err != cudaSuccess) {
    log_err("ork_b200_evict_async", err);
    return -1;
  }
  return 0;
}
