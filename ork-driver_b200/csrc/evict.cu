// evict.cu -- eviction from a cache by accumulated attention weight (include/ork_b200.h: ork_b200_evict_async).
//
// A token's key orders it: the first `sinks` and last `recent` tokens have the largest key, others their score's
// bits mapped to an unsigned word of the same order (a NaN's: minus infinity's). The kept ones are those above a threshold key,
// found eight bits at a time from counts of the keys that share the bits found so far, and of those equal to it
// the lowest slots.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>

#include "errword.cuh"
#include "ork_internal.h"
#include "ork_structs.h"

namespace orkb {

__device__ unsigned int g_evict_error = 0;

namespace {

constexpr int kThreads = 1024;

__device__ __forceinline__ uint32_t key_of(float score, int j, int n, int sinks, int recent) {
  if (j < sinks || j >= n - recent) return 0xffffffffu;
  const uint32_t b = __float_as_uint(isnan(score) ? -INFINITY : score + 0.0f);  // -0 counts as 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// exclusive prefix sum of v over the block; *total: its sum
__device__ __forceinline__ int block_scan(int v, int *red, int *total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
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
    int y = red[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    red[lane] = y;
  }
  __syncthreads();
  *total = red[31];
  return x - v + (w ? red[w - 1] : 0);
}

// One block per (sequence, kv head).
__global__ void __launch_bounds__(kThreads) evict_kernel(const ork_b200_evict e) {
  __shared__ int hist[256], red[32], s_digit, s_left;
  const int sh = blockIdx.x, s = sh / e.Hkv, tid = threadIdx.x;
  int n = e.len[s];
  if (n < 0 || n > e.max_len || n > e.cap) {
    if (tid == 0) {
      atomicOr(&g_evict_error, 1u);
      err_word_set();
    }
    n = 0;
  }
  const float *score = e.score + (size_t)sh * e.cap;
  const int m = min(n, e.keep);
  uint32_t prefix = 0;
  int left = m;  // of the keys that share the prefix, how many are kept
  for (int shift = 24; shift >= 0 && n > m; shift -= 8) {
    for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += kThreads) {
      const uint32_t k = key_of(score[j], j, n, e.sinks, e.recent);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, d = 255;
      for (; d > 0 && above + hist[d] < left; d--) above += hist[d];
      s_digit = d, s_left = left - above;
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    left = s_left;
    __syncthreads();
  }
  int placed = 0, equal = 0;
  for (int j0 = 0; j0 < n; j0 += kThreads) {
    const int j = j0 + tid;
    const uint32_t k = j < n ? key_of(score[j], j, n, e.sinks, e.recent) : 0u;
    int te, tk;
    const int is_eq = n > m && j < n && k == prefix;
    const int ne = equal + block_scan(is_eq, red, &te);
    const int keep = j < n && (n == m || k > prefix || (is_eq && ne < left));
    const int at = placed + block_scan(keep, red, &tk);
    if (keep) {
      if (e.kept) e.kept[(size_t)sh * e.keep + at] = j;
      if (e.score_out) e.score_out[(size_t)sh * e.dcap + at] = score[j];
      for (int p = 0; p < e.nplanes; p++) {
        const int words = e.row_bytes[p] / 4;
        const uint32_t *src = (const uint32_t *)e.src[p] + ((size_t)sh * e.cap + j) * words;
        uint32_t *dst = (uint32_t *)e.dst[p] + ((size_t)sh * e.dcap + at) * words;
        for (int w = 0; w < words; w++) dst[w] = src[w];
      }
    }
    equal += te;
    placed += tk;
  }
  for (int r = m + tid; r < e.keep; r += kThreads) {
    if (e.kept) e.kept[(size_t)sh * e.keep + r] = -1;
    if (e.score_out) e.score_out[(size_t)sh * e.dcap + r] = 0.0f;
  }
  if (e.len_out && sh % e.Hkv == 0 && tid == 0) e.len_out[s] = m;
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
  if (e->max_len < 0 || e->max_len > e->cap) return refuse("max_len is 0 .. cap");
  if (e->sinks < 0 || e->recent < 0 || (long long)e->sinks + e->recent > e->keep) return refuse("sinks + recent is 0 .. keep");
  if (e->nplanes < 0 || e->nplanes > ORK_B200_EVICT_PLANES) return refuse("too many planes");
  const size_t rows = (size_t)e->nseq * e->Hkv;
  for (int p = 0; p < e->nplanes; p++) {
    if (!e->src[p] || !e->dst[p]) return refuse("a plane is NULL");
    if (e->row_bytes[p] < 4 || e->row_bytes[p] % 4 || ((uintptr_t)e->src[p] | (uintptr_t)e->dst[p]) % 4)
      return refuse("rows are multiples of 4 bytes, planes 4-byte aligned");
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
  evict_kernel<<<(int)rows, kThreads, 0, c->stream>>>(*e);
  c->launches += 1;
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) {
    log_err("ork_b200_evict_async", err);
    return -1;
  }
  return 0;
}
