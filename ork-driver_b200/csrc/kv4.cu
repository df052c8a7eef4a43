// kv4.cu -- the 4-bit key/value cache (include/ork_b200.h): rows into it and back, and attention of the last
// tokens of each sequence over it.
//
// A value is code * step + lowest with one (step, lowest) pair of fp16 for each 64 dims of a token's head.
#include <cuda_runtime.h>

#define ORK_F16_AS_U16  // nvcc cannot compile expressions of the header's _Float16; the ABI is the same

#include <algorithm>
#include <cstdint>
#include <cstdio>

#include "elem.cuh"
#include "errword.cuh"
#include "ork_internal.h"
#include "ork_structs.h"

namespace orkb {

__device__ unsigned int g_kv4_error = 0;

namespace {

constexpr int kGroup = 64;  // dims that share a step and a lowest value

__device__ __forceinline__ void kv4_error() {
  atomicOr(&g_kv4_error, 1u);
  err_word_set();
}

// ---- rows into the cache and back ------------------------------------------------------------------------------
// A thread handles 8 consecutive dims of k or of v of one row and head: one 32-bit word of codes, so that a
// group's 8 threads find its lowest and largest value with three shuffles and a row's words are stored (loaded)
// by consecutive threads. Blocks stride over (row, head, k or v) items of a sequence (blockIdx.y).
constexpr int kRowThreads = 256;

struct Rows {
  int nseq, Hkv, dk, cap, rows;
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
__device__ __forceinline__ void load8(const E *p, bool vec, float (&x)[8]) {
  if (vec) {
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    if constexpr (sizeof(E) == 4) {
      const float4 c = *reinterpret_cast<const float4 *>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = __uint_as_float(w[i]);
      x[4] = c.x, x[5] = c.y, x[6] = c.z, x[7] = c.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 f = widen2(w[i], p);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = to_f32(p[i]);
  }
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

template <class E, bool STORE>
__global__ void __launch_bounds__(kRowThreads) kv4_rows_kernel(Rows r, E *k, E *v, uint32_t *kc, uint32_t *vc,
                                                               __half2 *kp, __half2 *vp, bool vec) {
  const int s = blockIdx.y, words = r.dk / 8, lane = threadIdx.x & 31;
  const int row0 = r.start ? r.start[s] : s * r.rows;
  const int n = r.start ? r.start[s + 1] - row0 : r.rows;
  const int slot0 = r.pos ? r.pos[s] : 0;
  const long long items = (long long)(n > 0 ? n : 0) * r.Hkv * 2 * words;  // a multiple of 8: groups stay whole
  for (long long at = (long long)blockIdx.x * kRowThreads + threadIdx.x; at < items;
       at += (long long)gridDim.x * kRowThreads) {
    const int w = (int)(at % words);
    const long long rh = at / words;
    const bool is_v = rh & 1;
    const int h = (int)((rh >> 1) % r.Hkv), t = (int)((rh >> 1) / r.Hkv);
    const long long slot = (long long)slot0 + t;
    if (slot < 0 || slot >= r.cap) {  // the same for a group's eight threads
      kv4_error();
      continue;
    }
    E *row = (is_v ? v : k) + ((long long)row0 + t) * r.ts + (long long)h * r.hs + 8 * w;
    const size_t tok = ((size_t)s * r.Hkv + h) * r.cap + (size_t)slot;
    uint32_t *code = (is_v ? vc : kc) + tok * words + w;
    __half2 *par = (is_v ? vp : kp) + tok * (r.dk / kGroup) + w / 8;
    float x[8];
    if constexpr (STORE) {
      load8<E>(row, vec, x);
      float lo = x[0], hi = x[0];
      bool fin = true;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        fin = fin && fabsf(x[i]) <= 3.402823466e38f;
      }
      const unsigned mask = 0xffu << (lane & 24);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
      }
      fin = __all_sync(mask, fin);
      // every operation rounds on its own, so that any IEEE implementation of the formulas gives these bits
      __half step = __float2half_rn(fminf(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f), 65504.0f));
      __half low = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
      if (!fin) step = low = __ushort_as_half((unsigned short)0x7fff);
      const float sf = __half2float(step), lf = __half2float(low);
      uint32_t c = 0;
      if (sf > 0.0f) {
#pragma unroll
        for (int i = 0; i < 8; i++)
          c |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[i], lf), sf)), 0.0f), 15.0f) << (4 * i);
      }
      *code = c;
      if ((w & 7) == 0) *par = __halves2half2(step, low);
    } else {
      const uint32_t c = *code;
      const float2 p = __half22float2(*par);
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = __fadd_rn(__fmul_rn((float)((c >> (4 * i)) & 15u), p.x), p.y);
      store8<E>(row, vec, x);
    }
  }
}

// ---- attention over the cache ----------------------------------------------------------------------------------

struct Attn4 {
  const uint8_t *kc, *vc;
  const __half *kp, *vp;
  int nseq, Hkv, cap, H, T, window, sinks, max_len;
  long long q_ts, q_hs;
  const int *len;
  float scale;
  float *wsum;
  float2 *stat;  // softmax maximum and sum of every row, for wsum
};

// the number of tokens of sequence s; -1 (reported) where it cannot be
__device__ __forceinline__ int seq_len(const Attn4 &a, int s) {
  const int n = a.len[s];
  if (n >= 0 && n <= a.max_len && n <= a.cap) return n;
  if (threadIdx.x == 0) kv4_error();
  return -1;
}
__device__ __forceinline__ bool visible(const Attn4 &a, int p, int j) {
  return j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
}

template <int DK>
__device__ __forceinline__ float value4(const uint8_t *codes, const __half *par, size_t tok, int d) {
  const uint8_t b = codes[tok * (DK / 2) + d / 2];
  const __half *p = par + (tok * (DK / kGroup) + d / kGroup) * 2;
  return (float)((d & 1) ? b >> 4 : b & 15) * __half2float(p[0]) + __half2float(p[1]);
}

// One warp per (sequence, token, query head); lane l holds dims l + 32 u.
template <class E, int DK>
__global__ void __launch_bounds__(32) kv4_attn_kernel(Attn4 a, const E *__restrict__ q, E *__restrict__ out) {
  constexpr int PER = DK / 32;
  const int lane = threadIdx.x, h = blockIdx.x % a.H, st = blockIdx.x / a.H, s = st / a.T, t = st % a.T;
  const int n = seq_len(a, s), p = n - a.T + t, kvh = h / (a.H / a.Hkv);
  float qv[PER], o[PER] = {}, m = -INFINITY, l = 0.0f;
  for (int u = 0; u < PER; u++) qv[u] = to_f32(q[(long long)st * a.q_ts + (long long)h * a.q_hs + lane + 32 * u]) * a.scale;
  for (int j = 0; n >= 0 && j <= p; j++) {
    if (!visible(a, p, j)) continue;
    const size_t tok = ((size_t)s * a.Hkv + kvh) * a.cap + j;
    float x = 0.0f;
    for (int u = 0; u < PER; u++) x += qv[u] * value4<DK>(a.kc, a.kp, tok, lane + 32 * u);
    for (int k = 16; k; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
    const float mn = fmaxf(m, x), c = m == mn ? 1.0f : __expf(m - mn), w = x == mn ? 1.0f : expf(x - mn);
    l = l * c + w;
    for (int u = 0; u < PER; u++) o[u] = o[u] * c + w * value4<DK>(a.vc, a.vp, tok, lane + 32 * u);
    m = mn;
  }
  for (int u = 0; u < PER; u++)
    out[((long long)st * a.H + h) * DK + lane + 32 * u] = from_f32<E>(l > 0.0f ? o[u] / l : (l == 0.0f ? 0.0f : l));
  if (a.wsum && lane == 0) a.stat[(size_t)st * a.H + h] = make_float2(m, l);
}

// wsum: one warp per (sequence, kv head, key), the rows in order.
template <class E, int DK>
__global__ void __launch_bounds__(256) kv4_wsum_kernel(Attn4 a, const E *__restrict__ q) {
  constexpr int PER = DK / 32;
  const int lane = threadIdx.x & 31, s = blockIdx.y / a.Hkv, kvh = blockIdx.y % a.Hkv, G = a.H / a.Hkv;
  const int j = blockIdx.x * 8 + (threadIdx.x >> 5), n = seq_len(a, s);
  if (j >= n) return;
  const size_t tok = ((size_t)s * a.Hkv + kvh) * a.cap + j;
  float kv[PER], sum = 0.0f;
  for (int u = 0; u < PER; u++) kv[u] = value4<DK>(a.kc, a.kp, tok, lane + 32 * u) * a.scale;
  for (int t = 0; t < a.T; t++) {
    if (!visible(a, n - a.T + t, j)) continue;
    for (int g = 0; g < G; g++) {
      const int st = s * a.T + t, h = kvh * G + g;
      float x = 0.0f;
      for (int u = 0; u < PER; u++) x += kv[u] * to_f32(q[(long long)st * a.q_ts + (long long)h * a.q_hs + lane + 32 * u]);
      for (int k = 16; k; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
      const float2 ml = a.stat[(size_t)st * a.H + h];
      sum += expf(x - ml.x) / ml.y;
    }
  }
  if (lane == 0) a.wsum[tok] += sum;
}

template <class E>
cudaError_t launch_attn(const Attn4 &a, int dk, const E *q, E *out, cudaStream_t st, uint64_t *launches) {
  const int rows = a.nseq * a.T * a.H;
  const dim3 wg((a.max_len + 7) / 8, a.nseq * a.Hkv);
  if (dk == 64) kv4_attn_kernel<E, 64><<<rows, 32, 0, st>>>(a, q, out);
  else kv4_attn_kernel<E, 128><<<rows, 32, 0, st>>>(a, q, out);
  *launches += 1;
  if (a.wsum && a.max_len) {
    if (dk == 64) kv4_wsum_kernel<E, 64><<<wg, 256, 0, st>>>(a, q);
    else kv4_wsum_kernel<E, 128><<<wg, 256, 0, st>>>(a, q);
    *launches += 1;
  }
  return cudaGetLastError();
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
  DeviceGuard dg(c->device);
  if (!device_ptrs_ok(c, name, {kv->k, kv->v, kv->kp, kv->vp, k, v, start, pos})) return -1;
  if (rows == 0) return 0;
  const bool vec = ((uintptr_t)k | (uintptr_t)v | (size_t)ts * es | (size_t)hs * es) % 16 == 0;
  const Rows r = {kv->nseq, kv->Hkv, kv->dk, kv->cap, rows, ts, hs, start, pos};
  const long long items = (long long)rows * kv->Hkv * 2 * (kv->dk / 8);
  const long long most = std::max<long long>(1, 148LL * 8 / kv->nseq);
  const dim3 grid((unsigned)std::min<long long>((items + kRowThreads - 1) / kRowThreads, most), kv->nseq);
  const cudaError_t e = with_elem(type, [&](auto *t) {
    using E = std::remove_pointer_t<decltype(t)>;
    auto kern = store ? kv4_rows_kernel<E, true> : kv4_rows_kernel<E, false>;
    kern<<<grid, kRowThreads, 0, c->stream>>>(r, (E *)k, (E *)v, (uint32_t *)kv->k, (uint32_t *)kv->v, (__half2 *)kv->kp,
                                              (__half2 *)kv->vp, vec);
    return cudaGetLastError();
  });
  c->launches += 1;
  if (e != cudaSuccess) {
    log_err(name, e);
    return -1;
  }
  return 0;
}

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
  if (a->T < 1 || (long long)kv->nseq * a->T * a->H > 0x7fffffff) return refuse(name, "bad number of rows");
  if (a->q_ts < kv->dk || a->q_hs < kv->dk) return refuse(name, "a row stride below dk");
  if (a->max_len < 0 || a->max_len > kv->cap) return refuse(name, "max_len is 0 .. cap");
  if (a->window < 0 || a->sinks < 0) return refuse(name, "window and sinks are not negative");
  if (((uintptr_t)a->q | (uintptr_t)a->out) % elem_bytes(a->type)) return refuse(name, "rows are aligned to their type");
  DeviceGuard dg(c->device);
  if (!device_ptrs_ok(c, name, {kv->k, kv->v, kv->kp, kv->vp, a->q, a->out, a->len, a->wsum})) return -1;
  Attn4 k = {kv->k, kv->v, (const __half *)kv->kp, (const __half *)kv->vp, kv->nseq, kv->Hkv, kv->cap, a->H, a->T,
             a->window, a->sinks, a->max_len, a->q_ts, a->q_hs, a->len, a->scale, a->wsum, nullptr};
  if (a->wsum && !grow(&c->dW, &c->capW, (size_t)kv->nseq * a->T * a->H * sizeof(float2)))
    return refuse(name, "out of device memory");
  k.stat = (float2 *)c->dW;
  const cudaError_t e = with_elem(a->type, [&](auto *t) {
    using E = std::remove_pointer_t<decltype(t)>;
    return launch_attn<E>(k, kv->dk, (const E *)a->q, (E *)a->out, c->stream, &c->launches);
  });
  if (e != cudaSuccess) {
    log_err(name, e);
    return -1;
  }
  return 0;
}

}  // extern "C"
