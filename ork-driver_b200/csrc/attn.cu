// attn.cu -- attention of packed rows (prompts, or chunks after a cached prefix) with a sliding window and sink
// keys (include/ork_b200.h: ork_b200_attn_async).
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>

#include "elem.cuh"
#include "errword.cuh"
#include "ork_internal.h"
#include "ork_structs.h"

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

// One warp per (row, head): lane l holds dims l + 32 u.
template <class E, int DK>
__global__ void __launch_bounds__(32) attn_kernel(const ork_b200_attn a) {
  constexpr int PER = DK / 32;
  const int lane = threadIdx.x, i = blockIdx.x, h = blockIdx.y, kvh = h / (a.H / a.Hkv);
  Seq s;
  if (!seq_of(a, blockIdx.z, &s) || i >= s.tq) return;
  const E *q = (const E *)a.q + (s.q0 + i) * a.q_ts + h * a.q_hs;
  E *out = (E *)a.out + (s.q0 + i) * a.o_ts + h * a.o_hs;
  const int p = s.tk - s.tq + i;
  float qv[PER], o[PER] = {}, m = -INFINITY, l = 0.0f;
  for (int u = 0; u < PER; u++) qv[u] = to_f32(q[lane + 32 * u]) * a.scale;
  for (int j = 0; j <= p; j++) {
    if (a.window && j <= p - a.window && j >= a.sinks) j = p - a.window + 1;
    const E *k = (const E *)a.k + (s.k0 + j) * a.k_ts + kvh * a.k_hs, *v = (const E *)a.v + (s.k0 + j) * a.v_ts + kvh * a.v_hs;
    float x = 0.0f;
    for (int u = 0; u < PER; u++) x += qv[u] * to_f32(k[lane + 32 * u]);
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    const float mn = fmaxf(m, x), c = m == mn ? 1.0f : __expf(m - mn), w = x == mn ? 1.0f : expf(x - mn);
    l = l * c + w;
    for (int u = 0; u < PER; u++) o[u] = o[u] * c + w * to_f32(v[lane + 32 * u]);
    m = mn;
  }
  for (int u = 0; u < PER; u++) out[lane + 32 * u] = from_f32<E>(l == 0.0f ? 0.0f : o[u] / l);
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
  for (long long st : {a->q_ts, a->q_hs, a->k_ts, a->k_hs, a->v_ts, a->v_hs, a->o_ts, a->o_hs})
    if (st < a->dk || st % 8) return refuse("strides are multiples of 8, dk at least");
  if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) % 16)
    return refuse("q, k, v and out are 16-byte aligned");
  DeviceGuard dg(c->device);
  if (!device_ptrs_ok(c, "ork_b200_attn_async", {a->q, a->k, a->v, a->out, a->q_start, a->k_start})) return -1;
  if (a->max_q == 0) return 0;
  const dim3 grid(a->max_q, a->H, a->nseq);
  auto kern = a->type == ORK_B200_F16 ? (a->dk == 64 ? attn_kernel<__half, 64> : attn_kernel<__half, 128>)
                                      : (a->dk == 64 ? attn_kernel<__nv_bfloat16, 64> : attn_kernel<__nv_bfloat16, 128>);
  kern<<<grid, 32, 0, c->stream>>>(*a);
  c->launches += 1;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    log_err("ork_b200_attn_async", e);
    return -1;
  }
  return 0;
}
