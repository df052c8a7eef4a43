"""A long conversation in a bounded 4-bit cache: the attention of one layer over a batch of prompts and the tokens after
them, with every long-context operator in its place.

  python examples/long_context.py [--tokens 600] [--prompt 4000] [--budget 2048]

For each sequence: the prompt attends to itself through a sliding window with sink tokens (ork_b200_attn_async, fp16),
its keys and values go into the 4-bit cache (ork_b200_kv4_store_async), and every new token is stored and attends to the
cache (ork_b200_kv4_attn_async), which adds up how much attention each cached token gets. Whenever a cache holds
`budget + slack` tokens, ork_b200_evict_async keeps the sinks, the recent tokens and the heaviest others and moves them,
with their weights, into a spare cache that takes the full one's place. Projections are random here; a model would call
its matmuls (ork_b200_*_mm_run_async) in their place, on the same stream.
"""
import argparse
import ctypes as C
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ork-driver_b200"))
import ork_b200 as B  # noqa: E402

H, HKV, DK = 16, 8, 128  # query heads, key/value heads, head size
WINDOW, SINKS, RECENT = 1024, 4, 256
F16 = B.TYPES["f16"]


class Cache:
    """A 4-bit cache in torch's memory, the attention weights its tokens have had, and what eviction needs of it."""

    def __init__(self, nseq, cap):
        dev = dict(device="cuda")
        self.planes = [torch.zeros((nseq, HKV, cap, n), dtype=t, **dev)
                       for t, n in ((torch.uint8, DK // 2), (torch.float16, DK // 32)) * 2]
        self.weight = torch.zeros((nseq, HKV, cap), **dev)
        k, kp, v, vp = (p.data_ptr() for p in self.planes)
        self.c = B.KV4(k=k, v=v, kp=kp, vp=vp, nseq=nseq, Hkv=HKV, dk=DK, cap=cap)


class Attention:
    def __init__(self, ctx, nseq, budget, slack):
        self.ctx, self.nseq, self.budget = ctx, nseq, budget
        self.cap = (budget + slack + 63) // 64 * 64
        self.cache, self.spare = Cache(nseq, self.cap), Cache(nseq, self.cap)
        self.len = torch.zeros(nseq, dtype=torch.int32, device="cuda")  # tokens held, on the device
        self.most = 0                                                   # the largest of them, on the host
        self.evictions = 0

    def _do(self, name, *args):
        if getattr(self.ctx.L, name)(self.ctx.ctx, *args):
            raise RuntimeError(name)

    def store(self, k, v, rows, start, pos):
        self._do("ork_b200_kv4_store_async", C.byref(self.cache.c), k.data_ptr(), v.data_ptr(), F16, rows, HKV * DK, DK, start, pos)

    def prompt(self, q, k, v, start, most):
        """Packed rows q [n, H, DK], k / v [n, HKV, DK] of all prompts; start [nseq + 1]."""
        out = torch.empty_like(q)
        a = B.Attn(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), type=F16, nseq=self.nseq, H=H, Hkv=HKV,
                   dk=DK, q_ts=H * DK, q_hs=DK, k_ts=HKV * DK, k_hs=DK, v_ts=HKV * DK, v_hs=DK, o_ts=H * DK, o_hs=DK,
                   q_start=start.data_ptr(), k_start=start.data_ptr(), q_rows=q.shape[0], k_rows=k.shape[0], max_q=most,
                   max_k=most, scale=DK ** -0.5, window=WINDOW, sinks=SINKS)
        self._do("ork_b200_attn_async", C.byref(a))
        self.store(k, v, most, start.data_ptr(), None)
        self.len.copy_(start[1:] - start[:-1])
        self.most = most
        return out

    def token(self, q, k, v):
        """One new token of every sequence: q [nseq, H, DK], k / v [nseq, HKV, DK]."""
        if self.most >= self.cap:
            self.evict()
        self.store(k, v, 1, None, self.len.data_ptr())
        self.len += 1
        self.most += 1
        out = torch.empty_like(q)
        a = B.KV4Attn(q=q.data_ptr(), out=out.data_ptr(), type=F16, H=H, T=1, q_ts=H * DK, q_hs=DK, len=self.len.data_ptr(),
                      max_len=self.most, scale=DK ** -0.5, window=0, sinks=0, wsum=self.cache.weight.data_ptr())
        self._do("ork_b200_kv4_attn_async", C.byref(self.cache.c), C.byref(a))
        return out

    def evict(self):
        old, new = self.cache, self.spare
        new.weight.zero_()
        e = B.Evict(score=old.weight.data_ptr(), len=self.len.data_ptr(), nseq=self.nseq, Hkv=HKV, cap=self.cap, dcap=self.cap,
                    max_len=self.most, keep=self.budget, sinks=SINKS, recent=RECENT, nplanes=4,
                    score_out=new.weight.data_ptr(), len_out=(held := torch.empty_like(self.len)).data_ptr())
        for i, (a, b) in enumerate(zip(old.planes, new.planes)):
            e.src[i], e.dst[i], e.row_bytes[i] = a.data_ptr(), b.data_ptr(), a.shape[-1] * a.element_size()
        self._do("ork_b200_evict_async", C.byref(e))
        self.cache, self.spare, self.len = new, old, held
        self.most = min(self.most, self.budget)
        self.evictions += 1


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--sequences", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=4000)
    ap.add_argument("--tokens", type=int, default=600)
    ap.add_argument("--budget", type=int, default=2048)
    n = ap.parse_args()
    g = torch.Generator(device="cuda").manual_seed(0)

    def rows(*shape):
        return torch.randn(shape, device="cuda", generator=g).half()

    with B.Context() as ctx, torch.no_grad():
        ctx.L.ork_b200_set_stream(ctx.ctx, torch.cuda.current_stream().cuda_stream or 1)  # 1: the legacy default stream
        lens = [max(1, n.prompt - 97 * i) for i in range(n.sequences)]  # prompts of different lengths
        start = torch.tensor([sum(lens[:i]) for i in range(n.sequences + 1)], dtype=torch.int32, device="cuda")
        at = Attention(ctx, n.sequences, n.budget, max(max(lens) - n.budget, 0) + 256)
        total = sum(lens)
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
        ev[0].record()
        out = at.prompt(rows(total, H, DK), rows(total, HKV, DK), rows(total, HKV, DK), start, max(lens))
        ev[1].record()
        for _ in range(n.tokens):
            out = at.token(rows(n.sequences, H, DK), rows(n.sequences, HKV, DK), rows(n.sequences, HKV, DK))
        ev[2].record()
        if ctx.L.ork_b200_sync(ctx.ctx):
            raise RuntimeError("a kernel reported an error")
        assert torch.isfinite(out).all()
        held = at.len.tolist()
        bits = sum(p.numel() * p.element_size() for p in at.cache.planes) * 8 / (2 * n.sequences * HKV * at.cap * DK)
        print(f"{total} prompt tokens in {ev[0].elapsed_time(ev[1]):.2f} ms, {n.tokens} steps of {n.sequences} tokens in "
              f"{ev[1].elapsed_time(ev[2]):.2f} ms, {at.evictions} evictions, tokens held {held}, {bits:.2f} bits a value")


if __name__ == "__main__":
    main()
