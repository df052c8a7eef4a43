"""Measured cases of the long-context operators: prompt attention with a sliding window and sink tokens, the
4-bit key/value cache (store and read back), attention of new tokens over that cache, and eviction from a cache
by accumulated attention weight.

Where `own` is false, run() computes an operator in elementary torch operations in 32 bits; where it is true it
makes the library calls of include/ork_b200.h on the same buffers. exact() is the operator's definition in 64 bits.
"""
import math

import torch

own = False

GROUP = 64  # dims that share a step and a lowest value in the 4-bit cache
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases -----------------------------------------------------------------------------------------------------

def listed():
    return [
        # Prompt attention. A short chat turn on a 16/8-head model: latency.
        dict(name="attn_turn_48", op="attn", type="f16", nseq=1, H=16, Hkv=8, dk=128, tq=48, prefix=0, ragged=False,
             window=0, sinks=0),
        # A long document in one go, all of it visible, 16/8 heads: the largest.
        dict(name="attn_full_16384", op="attn", type="bf16", nseq=1, H=16, Hkv=8, dk=128, tq=16384, prefix=0,
             ragged=False, window=0, sinks=0),
        # A long document through a window of 1024 with four sinks, 64/8 heads.
        dict(name="attn_window_8192", op="attn", type="f16", nseq=1, H=64, Hkv=8, dk=128, tq=8192, prefix=0,
             ragged=False, window=1024, sinks=4),
        # A batch of prompts of odd lengths, each continuing a cached prefix, 64-dim heads, one key head per query head.
        dict(name="attn_ragged_dk64", op="attn", type="bf16", nseq=7, H=12, Hkv=12, dk=64, tq=777, prefix=1301,
             ragged=True, window=500, sinks=5),
        # Attention over the 4-bit cache. One token of one chat: latency, fp32 activations as the decode layer's.
        dict(name="kv4_one_1000", op="kv4_attn", type="f32", nseq=1, H=16, Hkv=8, dk=128, cap=2048, len=1000, T=1,
             ragged=False, window=0, sinks=0, wsum=False),
        # One token of one long document on a 64/8-head model: the work has to be split along the document.
        dict(name="kv4_one_131071", op="kv4_attn", type="f16", nseq=1, H=64, Hkv=8, dk=128, cap=131072, len=131071, T=1,
             ragged=False, window=0, sinks=0, wsum=True),
        # A full serving batch of ragged lengths: the largest.
        dict(name="kv4_batch_64", op="kv4_attn", type="bf16", nseq=64, H=64, Hkv=8, dk=128, cap=16384, len=16384, T=1,
             ragged=True, window=0, sinks=0, wsum=False),
        # Four drafted tokens checked at once through a window with sinks, weights accumulated for eviction.
        dict(name="kv4_draft_window", op="kv4_attn", type="f16", nseq=16, H=32, Hkv=8, dk=64, cap=8192, len=8001, T=4,
             ragged=True, window=4096, sinks=4, wsum=True),
        # The rows of a decode step of a batch into the cache, and a prompt's.
        dict(name="store_step_32", op="store", type="f32", nseq=32, Hkv=8, dk=128, cap=4096, rows=1, pos=3333,
             ragged=False),
        dict(name="store_prompts", op="store", type="bf16", nseq=5, Hkv=8, dk=128, cap=16384, rows=12345, pos=7,
             ragged=True),
        # Eviction to a budget: a chat's fp32 caches, and a batch's 4-bit caches.
        dict(name="evict_chat_f32", op="evict", rows="f32", nseq=1, Hkv=8, dk=128, cap=4096, len=4001, keep=1024,
             sinks=4, recent=256, ragged=False),
        dict(name="evict_batch_kv4", op="evict", rows="kv4", nseq=16, Hkv=8, dk=128, cap=32768, len=32768, keep=8192,
             sinks=4, recent=1024, ragged=True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "kv4_attn", "kv4_attn", "store", "evict"])
    dk = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    if op == "attn":
        G = rng.choice([1, 2, 3, 4, 8])
        nseq = rng.choice([1, 1, 2, 3, 8])
        H = G * Hkv
        most = 2.0e9 / (H * nseq)  # scores of the padded batch
        tq = _log(rng, 1, min(8192, math.sqrt(most)))
        prefix = rng.choice([0, 0, _log(rng, 1, max(2, min(8192, most / tq - tq)))])
        return dict(op=op, type=rng.choice(["f16", "bf16"]), nseq=nseq, H=H, Hkv=Hkv, dk=dk, tq=tq, prefix=prefix,
                    ragged=nseq > 1, window=rng.choice([0, _log(rng, 1, 4096)]), sinks=rng.choice([0, 1, 4, 133]))
    if op == "kv4_attn":
        G = rng.choice([1, 2, 3, 4, 7, 8, 16])
        nseq = _log(rng, 1, 64)
        n = _log(rng, 1, min(131072, (1 << 23) // (nseq * Hkv)))
        cap = (n + 63) // 64 * 64 + 64 * rng.choice([0, 3])
        return dict(op=op, type=rng.choice(["f32", "f16", "bf16"]), nseq=nseq, H=G * Hkv, Hkv=Hkv, dk=dk, cap=cap, len=n,
                    T=rng.choice([1, 1, 1, 2, 5]), ragged=nseq > 1, window=rng.choice([0, 0, _log(rng, 1, 8192)]),
                    sinks=rng.choice([0, 1, 4, 133]), wsum=rng.choice([False, True]))
    if op == "store":
        nseq = _log(rng, 1, 64)
        rows = _log(rng, 1, 65536 // nseq)
        pos = rng.choice([0, _log(rng, 1, 4096)])
        return dict(op=op, type=rng.choice(["f32", "f16", "bf16"]), nseq=nseq, Hkv=Hkv, dk=dk,
                    cap=(rows + pos + 63) // 64 * 64, rows=rows, pos=pos, ragged=nseq > 1)
    nseq = _log(rng, 1, 32)
    n = _log(rng, 64, min(65536, (1 << 21) // (nseq * Hkv)))
    keep = _log(rng, max(1, n // 16), n)
    return dict(op=op, rows=rng.choice(["f32", "kv4"]), nseq=nseq, Hkv=Hkv, dk=dk, cap=(n + 63) // 64 * 64, len=n,
                keep=keep, sinks=min(keep // 2, rng.choice([0, 1, 4])), recent=keep // rng.choice([2, 4, 8]),
                ragged=nseq > 1)


def _lens(case, top):
    """Per-sequence lengths: all `top`, or ragged ones from about half of it up to it."""
    n = case["nseq"]
    return [top - (i * 7919 * (top // 97 + 1)) % (top // 2 + 1) if case["ragged"] else top for i in range(n)]


def _seen(case, lens, new):
    """(query, key) pairs that the mask leaves, and keys seen by any query, for sequences of `lens` tokens whose last
    new[i] are the queries."""
    w, s = case["window"], case["sinks"]
    pairs = keys = 0
    for n, t in zip(lens, new):
        p = torch.arange(n - t, n, dtype=torch.int64)
        p = p[p >= 0]
        lo = (p - w + 1).clamp(min=0) if w else torch.zeros_like(p)
        pairs += int((p + 1 - lo + torch.minimum(lo, torch.full_like(lo, s))).sum())
        if p.numel():
            lo0 = int(lo[0])
            keys += n - lo0 + min(lo0, s)
    return pairs, keys


def work(case):
    op = case["op"]
    es = {"f32": 4, "f16": 2, "bf16": 2}.get(case.get("type"), 0)
    dk, Hkv = case["dk"], case["Hkv"]
    row4 = 2 * (dk // 2 + dk // GROUP * 4)  # codes and parameters of a token's k and v in one head
    if op == "attn":
        tq = _lens(case, case["tq"])
        tk = [a + b for a, b in zip(tq, _lens(case, case["prefix"]))]
        pairs, keys = _seen(case, tk, tq)
        return {"bytes": es * dk * (2 * case["H"] * sum(tq) + 2 * Hkv * keys), "flops": 4 * dk * case["H"] * pairs}
    if op == "kv4_attn":
        lens, T = _lens(case, case["len"]), case["T"]
        pairs, keys = _seen(case, lens, [T] * len(lens))
        b = 2 * es * dk * case["H"] * T * len(lens) + Hkv * keys * row4
        return {"bytes": b + (8 * Hkv * keys if case["wsum"] else 0), "flops": 4 * dk * case["H"] * pairs}
    if op == "store":  # rows read, cache written; cache read, rows written
        n = sum(_lens(case, case["rows"])) * Hkv
        return {"bytes": n * (4 * es * dk + 2 * row4), "flops": n * dk * 2 * 8}
    lens = _lens(case, case["len"])
    m = sum(min(n, case["keep"]) for n in lens) * Hkv
    row = row4 if case["rows"] == "kv4" else 8 * dk
    back = (row4 + 4 * dk) if case["rows"] == "kv4" else 0  # the 4-bit rows are read back as f16 values
    return {"bytes": 4 * sum(lens) * Hkv + m * (2 * row + 8 + back), "flops": sum(lens) * Hkv * 4}


# ---- inputs ----------------------------------------------------------------------------------------------------

_lib = None


def _library():
    """The library's binding, and one context that queues on torch's stream (handle 1: the legacy default stream)."""
    global _lib
    if _lib is None:
        import os
        import sys

        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ork-driver_b200"))
        import ork_b200

        torch.cuda.current_stream()
        c = ork_b200.Context()
        c.L.ork_b200_set_stream(c.ctx, torch.cuda.current_stream().cuda_stream or 1)
        _lib = (ork_b200, c)
    return _lib


def _quantize(x):
    """[..., dk] f32 -> codes uint8 [..., dk/2] (low nibble: even dim) and parameters f16 [..., dk/GROUP, 2] (step, low)."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    low = lo.clamp(-65504, 65504).half()
    step = ((hi - lo) * (1 / 15)).clamp(max=65504).half()
    s = step.float()
    code = torch.round((g - low.float().unsqueeze(-1)) / s.unsqueeze(-1))
    code = torch.where(s.unsqueeze(-1) > 0, code, torch.zeros_like(code)).clamp(0, 15).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.stack([step, low], -1)


def _dequantize(codes, par, dtype=torch.float32):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP)).to(dtype)
    return (c * par[..., :1].to(dtype) + par[..., 1:].to(dtype)).flatten(-2)


def _starts(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def _keys(shape, bias, g):
    """Keys with per-dim offsets, as those of trained models have, in f32."""
    return torch.randn(shape, device="cuda", generator=g) * 1.1 + bias


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, nseq, Hkv, dk = case["op"], case["nseq"], case["Hkv"], case["dk"]
    dt = TYPES.get(case.get("type"))
    s = {"case": case}
    i32 = dict(dtype=torch.int32, device="cuda")
    if op == "attn":
        H, tq = case["H"], _lens(case, case["tq"])
        tk = [a + b for a, b in zip(tq, _lens(case, case["prefix"]))]
        bias = torch.randn((Hkv, dk), device="cuda", generator=g)
        s["q"] = (torch.randn((sum(tq), H, dk), device="cuda", generator=g) * 1.6).to(dt)
        s["k"] = _keys((sum(tk), Hkv, dk), bias, g).to(dt)
        s["v"] = torch.randn((sum(tk), Hkv, dk), device="cuda", generator=g).to(dt)
        s["out"] = torch.zeros_like(s["q"])
        s["q_start"], s["k_start"] = torch.tensor(_starts(tq), **i32), torch.tensor(_starts(tk), **i32)
        if own:
            B, _ = _library()
            s["call"] = B.Attn(q=s["q"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), out=s["out"].data_ptr(),
                               type=B.TYPES[case["type"]], nseq=nseq, H=H, Hkv=Hkv, dk=dk, q_ts=H * dk, q_hs=dk,
                               k_ts=Hkv * dk, k_hs=dk, v_ts=Hkv * dk, v_hs=dk, o_ts=H * dk, o_hs=dk,
                               q_start=s["q_start"].data_ptr(), k_start=s["k_start"].data_ptr(), q_rows=sum(tq),
                               k_rows=sum(tk), max_q=max(tq), max_k=max(tk), scale=dk ** -0.5, window=case["window"],
                               sinks=case["sinks"])
        return s
    cap = case["cap"]
    if op in ("kv4_attn", "store") or case["rows"] == "kv4":
        made = [(torch.zeros((nseq, Hkv, cap, dk // 2), dtype=torch.uint8, device="cuda"),
                 torch.zeros((nseq, Hkv, cap, dk // GROUP, 2), dtype=torch.float16, device="cuda")) for _ in range(2)]
        (s["kc"], s["kp"]), (s["vc"], s["vp"]) = made
        if op != "store":
            bias = torch.randn((Hkv, 1, dk), device="cuda", generator=g)
            for i in range(nseq):
                for (c, p), b in zip(made, (bias, 0.0)):
                    c[i], p[i] = _quantize(_keys((Hkv, cap, dk), b, g))
        if own:
            B, _ = _library()
            s["cache"] = B.KV4(k=s["kc"].data_ptr(), v=s["vc"].data_ptr(), kp=s["kp"].data_ptr(), vp=s["vp"].data_ptr(),
                               nseq=nseq, Hkv=Hkv, dk=dk, cap=cap)
    if op == "kv4_attn":
        H, T, n = case["H"], case["T"], _lens(case, case["len"])
        s["q"] = (torch.randn((nseq, T, H, dk), device="cuda", generator=g) * 1.6).to(dt)
        s["out"], s["len"] = torch.zeros_like(s["q"]), torch.tensor(n, **i32)
        s["wsum"] = torch.zeros((nseq, Hkv, cap), device="cuda") if case["wsum"] else None
        if own:
            s["call"] = B.KV4Attn(q=s["q"].data_ptr(), out=s["out"].data_ptr(), type=B.TYPES[case["type"]], H=H, T=T,
                                  q_ts=H * dk, q_hs=dk, len=s["len"].data_ptr(), max_len=max(n), scale=dk ** -0.5,
                                  window=case["window"], sinks=case["sinks"],
                                  wsum=s["wsum"].data_ptr() if case["wsum"] else None)
    elif op == "store":
        n = _lens(case, case["rows"])
        s["k"] = _keys((sum(n), Hkv, dk), torch.randn((Hkv, dk), device="cuda", generator=g), g).to(dt)
        s["v"] = torch.randn((sum(n), Hkv, dk), device="cuda", generator=g).to(dt)
        s["ko"], s["vo"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        s["start"] = torch.tensor(_starts(n), **i32)
        s["pos"] = torch.full((nseq,), case["pos"], **i32)
        s["most"] = max(n)
    elif op == "evict":
        n, keep = _lens(case, case["len"]), case["keep"]
        # most tokens get next to nothing, a few a lot, some never a thing
        w = torch.exp(torch.randn((nseq, Hkv, cap), device="cuda", generator=g) * 3 - 6)
        s["score"] = torch.where(torch.rand((nseq, Hkv, cap), device="cuda", generator=g) < 0.1, torch.zeros_like(w), w)
        s["len"] = torch.tensor(n, **i32)
        dcap = (keep + 63) // 64 * 64
        if case["rows"] == "kv4":
            s["src"] = [s[x].flatten(3) for x in ("kc", "kp", "vc", "vp")]
        else:
            s["src"] = [torch.randn((nseq, Hkv, cap, dk), device="cuda", generator=g) for _ in range(2)]
        s["dst"] = [torch.zeros((nseq, Hkv, dcap, x.shape[-1]), dtype=x.dtype, device="cuda") for x in s["src"]]
        s["kept"] = torch.zeros((nseq, Hkv, keep), **i32)
        s["score_out"] = torch.zeros((nseq, Hkv, dcap), device="cuda")
        s["len_out"] = torch.zeros((nseq,), **i32)
        if case["rows"] == "kv4":
            s["zero"] = torch.zeros((nseq,), **i32)
            s["back"] = [torch.zeros((nseq, dcap, Hkv, dk), dtype=torch.float16, device="cuda") for _ in range(2)]
        if own:
            B, _ = _library()
            s["call"] = B.Evict(score=s["score"].data_ptr(), len=s["len"].data_ptr(), nseq=nseq, Hkv=Hkv, cap=cap,
                                dcap=dcap, max_len=max(n), keep=keep, sinks=case["sinks"], recent=case["recent"],
                                nplanes=len(s["src"]), kept=s["kept"].data_ptr(),
                                score_out=s["score_out"].data_ptr(), len_out=s["len_out"].data_ptr())
            for i, (a, b) in enumerate(zip(s["src"], s["dst"])):
                s["call"].src[i], s["call"].dst[i] = a.data_ptr(), b.data_ptr()
                s["call"].row_bytes[i] = a.shape[-1] * a.element_size()
            if case["rows"] == "kv4":
                s["held"] = B.KV4(k=s["dst"][0].data_ptr(), kp=s["dst"][1].data_ptr(), v=s["dst"][2].data_ptr(),
                                  vp=s["dst"][3].data_ptr(), nseq=nseq, Hkv=Hkv, dk=dk, cap=dcap)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    return _own(s, op) if own else {"attn": _attn, "kv4_attn": _kv4_attn, "store": _store, "evict": _evict}[op](s)


def _own(s, op):
    B, c = _lib
    L, by = c.L, B.C.byref
    if op == "attn":
        rc = L.ork_b200_attn_async(c.ctx, by(s["call"]))
        out = s["out"]
    elif op == "kv4_attn":
        rc = L.ork_b200_kv4_attn_async(c.ctx, by(s["cache"]), by(s["call"]))
        out = s["out"] if s["wsum"] is None else (s["out"], s["wsum"])
    elif op == "store":
        t, hd = B.TYPES[s["case"]["type"]], s["k"].shape[1] * s["k"].shape[2]
        a = (t, s["most"], hd, s["k"].shape[2], s["start"].data_ptr(), s["pos"].data_ptr())
        rc = L.ork_b200_kv4_store_async(c.ctx, by(s["cache"]), s["k"].data_ptr(), s["v"].data_ptr(), *a)
        rc |= L.ork_b200_kv4_load_async(c.ctx, by(s["cache"]), s["ko"].data_ptr(), s["vo"].data_ptr(), *a)
        out = (s["ko"], s["vo"])
    else:
        rc = L.ork_b200_evict_async(c.ctx, by(s["call"]))
        out = [s["kept"], s["score_out"], s["len_out"]]
        if s["case"]["rows"] == "kv4":  # the kept rows as the values they stand for
            (nseq, dcap, Hkv, dk), (k, v) = s["back"][0].shape, s["back"]
            rc |= L.ork_b200_kv4_load_async(c.ctx, by(s["held"]), k.data_ptr(), v.data_ptr(), B.TYPES["f16"], dcap,
                                            Hkv * dk, dk, None, s["zero"].data_ptr())
            out += s["back"]
        else:
            out += s["dst"]
    if rc:
        raise RuntimeError("the library refused the call")
    return out


def _mask(p, j, case):
    """Whether key j is visible from position p."""
    ok = j <= p
    if case["window"]:
        ok = ok & ((j > p - case["window"]) | (j < case["sinks"]))
    return ok


def _weights(a, ok):
    """Softmax over the last axis of the places that `ok` leaves; rows without any give zeros. Works in a's memory."""
    a.masked_fill_(~ok, -math.inf)
    m = a.amax(-1, keepdim=True)
    a.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    t = a.sum(-1, keepdim=True)
    return a.div_(t.masked_fill(t == 0, 1.0))


def _attn(s):
    case = s["case"]
    H, Hkv, dk, nseq = case["H"], case["Hkv"], case["dk"], case["nseq"]
    G = H // Hkv
    qs, ks = s["q_start"].long(), s["k_start"].long()
    tq, tk = qs[1:] - qs[:-1], ks[1:] - ks[:-1]
    lq, lk = _lens(case, case["tq"]), [a + b for a, b in zip(_lens(case, case["tq"]), _lens(case, case["prefix"]))]
    i, j = torch.arange(max(lq), device="cuda"), torch.arange(max(lk), device="cuda")
    iq = (qs[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    ik = (ks[:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
    q = s["q"].float()[iq].view(nseq, max(lq), Hkv, G, dk).permute(0, 2, 3, 1, 4).reshape(nseq, Hkv, -1, dk)
    k = s["k"].float()[ik].permute(0, 2, 3, 1)  # [nseq, Hkv, dk, tk]
    v = s["v"].float()[ik].permute(0, 2, 1, 3)
    p = (tk - tq)[:, None, None] + i[None, :, None]
    ok = _mask(p, j[None, None, :], case) & (j[None, None, :] < tk[:, None, None])  # [nseq, tq, tk]
    a = torch.matmul(q, k).mul_(dk ** -0.5).view(nseq, H, max(lq), max(lk))
    a = _weights(a, ok[:, None])
    o = torch.matmul(a.view(nseq, Hkv, G * max(lq), max(lk)), v).view(nseq, H, max(lq), dk).transpose(1, 2)
    s["out"].copy_(o[i[None, :] < tq[:, None]].to(s["q"].dtype))
    return s["out"]


def _kv4_attn(s):
    case = s["case"]
    H, Hkv, dk, nseq, T = case["H"], case["Hkv"], case["dk"], case["nseq"], case["T"]
    G, n = H // Hkv, case["len"]
    k = _dequantize(s["kc"][:, :, :n], s["kp"][:, :, :n])
    q = s["q"].float().view(nseq, T, Hkv, G, dk).permute(0, 2, 1, 3, 4).reshape(nseq, Hkv, T * G, dk)
    a = torch.matmul(q, k.transpose(-1, -2)).mul_(dk ** -0.5).view(nseq, Hkv, T, G, n)
    del k
    j = torch.arange(n, device="cuda")
    p = s["len"].long()[:, None] - T + torch.arange(T, device="cuda")
    ok = _mask(p[:, :, None], j, case)  # [nseq, T, n]
    a = _weights(a, ok[:, None, :, None]).view(nseq, Hkv, T * G, n)
    o = torch.matmul(a, _dequantize(s["vc"][:, :, :n], s["vp"][:, :, :n])).view(nseq, Hkv, T, G, dk)
    s["out"].copy_(o.permute(0, 2, 1, 3, 4).reshape(nseq, T, H, dk).to(s["q"].dtype))
    if s["wsum"] is None:
        return s["out"]
    s["wsum"][:, :, :n] += a.sum(2)
    return s["out"], s["wsum"]


def _slots(s):
    """(sequence, slot) of every packed row."""
    st = s["start"].long()
    r = torch.arange(s["k"].shape[0], device="cuda")
    q = torch.searchsorted(st[1:], r, right=True)
    return q, s["pos"].long()[q] + r - st[q]


def _store(s):
    q, t = _slots(s)
    for x, c, p, o in (("k", "kc", "kp", "ko"), ("v", "vc", "vp", "vo")):
        codes, par = _quantize(s[x].float())
        s[c][q, :, t] = codes
        s[p][q, :, t] = par
        s[o].copy_(_dequantize(s[c][q, :, t], s[p][q, :, t]).to(s[x].dtype))
    return s["ko"], s["vo"]


def _evict(s):
    case = s["case"]
    nseq, Hkv, cap, keep = case["nseq"], case["Hkv"], case["cap"], case["keep"]
    n = s["len"].long()[:, None, None]
    j = torch.arange(cap, device="cuda").expand(nseq, Hkv, cap)
    key = torch.nan_to_num(s["score"], nan=-math.inf)
    key = torch.where((j < case["sinks"]) | (j >= n - case["recent"]), torch.full_like(key, math.inf), key)
    first = torch.sort(key, dim=-1, descending=True, stable=True)[1]
    live = torch.gather(j < n, 2, first)  # the places within the sequence come first, in the same order
    first = torch.gather(first, 2, torch.sort((~live).to(torch.uint8), dim=-1, stable=True)[1])[:, :, :keep]
    m = n.clamp(max=keep)
    r = torch.arange(keep, device="cuda")
    at = torch.sort(torch.where(r < m, first, torch.full_like(first, cap)), dim=-1)[0]
    s["kept"].copy_(torch.where(r < m, at, torch.full_like(at, -1)))
    at = at.clamp(max=cap - 1)
    s["score_out"][:, :, :keep] = torch.where(r < m, torch.gather(s["score"], 2, at), torch.zeros((), device="cuda"))
    s["len_out"].copy_(m[:, 0, 0])
    for a, b in zip(s["src"], s["dst"]):
        rows = torch.gather(a, 2, at[..., None].expand(-1, -1, -1, a.shape[-1]))
        b[:, :, :keep] = torch.where((r < m)[..., None], rows, b[:, :, :keep])
    out = [s["kept"], s["score_out"], s["len_out"]]
    if case["rows"] != "kv4":
        return out + s["dst"]
    for o, c, p in ((s["back"][0], 0, 1), (s["back"][1], 2, 3)):
        o.copy_(_dequantize(s["dst"][c], s["dst"][p].unflatten(-1, (-1, 2))).transpose(1, 2))
    return out + s["back"]


# ---- the definitions in 64 bits --------------------------------------------------------------------------------

def _one_softmax(logits, ok):
    """Rows of float64 logits under a mask: e^x / sum e^x, and zeros where a row has nothing."""
    x = torch.where(ok, logits, torch.full_like(logits, -math.inf))
    top = x.max(-1, keepdim=True).values
    e = torch.where(ok, (x - torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp(), torch.zeros_like(x))
    t = e.sum(-1, keepdim=True)
    return e / torch.where(t > 0, t, torch.ones_like(t))


def _rows4(codes, par):
    """[n, dk/2] codes and [n, dk/GROUP, 2] parameters -> [n, dk] float64."""
    c = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device="cuda")
    c[..., 0::2], c[..., 1::2] = (codes % 16).double(), (codes // 16).double()
    return c * par[..., 0].double().repeat_interleave(GROUP, -1) + par[..., 1].double().repeat_interleave(GROUP, -1)


def exact(case, seed):
    s = prepare(case, seed)
    op, nseq, Hkv, dk = case["op"], case["nseq"], case["Hkv"], case["dk"]
    if op == "attn":
        H = case["H"]
        q0, k0 = s["q_start"].tolist(), s["k_start"].tolist()
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for i in range(nseq):
            nk, nq = k0[i + 1] - k0[i], q0[i + 1] - q0[i]
            for h in range(H):
                k = s["k"][k0[i]:k0[i + 1], h * Hkv // H].double()
                v = s["v"][k0[i]:k0[i + 1], h * Hkv // H].double()
                for a in range(0, nq, 4096):
                    b = min(nq, a + 4096)
                    p = torch.arange(nk - nq + a, nk - nq + b, device="cuda")[:, None]
                    j = torch.arange(nk, device="cuda")[None]
                    ok = (j <= p) & ((j < case["sinks"]) | (p - j < (case["window"] or nk + 1)))
                    w = _one_softmax(s["q"][q0[i] + a:q0[i] + b, h].double() @ k.T / math.sqrt(dk), ok)
                    out[q0[i] + a:q0[i] + b, h] = w @ v
        return out
    if op == "kv4_attn":
        H, T, n = case["H"], case["T"], s["len"].tolist()
        G = H // Hkv
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        ws = torch.zeros((nseq, Hkv, case["cap"]), dtype=torch.float64, device="cuda")
        for i in range(nseq):
            j = torch.arange(n[i], device="cuda")
            p = torch.arange(n[i] - T, n[i], device="cuda")[:, None]
            ok = ((j <= p) & ((j < case["sinks"]) | (p - j < (case["window"] or n[i] + 1))))[:, None]
            for h in range(Hkv):
                k, v = (_rows4(s[c][i, h, :n[i]], s[x][i, h, :n[i]]) for c, x in (("kc", "kp"), ("vc", "vp")))
                q = s["q"][i, :, h * G:(h + 1) * G].double()
                w = _one_softmax(q @ k.T / math.sqrt(dk), ok.expand(T, G, n[i]))
                out[i, :, h * G:(h + 1) * G] = w @ v
                ws[i, h, :n[i]] = w.sum((0, 1))
        return out if s["wsum"] is None else (out, ws)
    if op == "store":
        back = []
        for x in ("k", "v"):
            g = s[x].double().unflatten(-1, (-1, GROUP))
            lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
            step, low = ((hi - lo) / 15).half().double(), lo.half().double()
            code = torch.round((g - low) / torch.where(step > 0, step, torch.ones_like(step))).clamp(0, 15)
            back.append((code * step + low).flatten(-2))
        return tuple(back)
    keep, n = case["keep"], s["len"].tolist()
    kept = torch.full(s["kept"].shape, -1, dtype=torch.int32)
    score = s["score"].double().cpu()
    got = torch.zeros(s["score_out"].shape, dtype=torch.float64)
    for i in range(nseq):
        for h in range(Hkv):
            w = score[i, h, :n[i]].clone()
            w[:case["sinks"]] = math.inf
            w[max(0, n[i] - case["recent"]):] = math.inf
            at = torch.sort(torch.argsort(-w, stable=True)[:keep]).values
            kept[i, h, :at.numel()] = at.int()
            got[i, h, :at.numel()] = score[i, h, at]
    out = [kept, got, torch.tensor([min(x, keep) for x in n], dtype=torch.int32)]
    for c in range(0, len(s["src"]), len(s["src"]) // 2):
        full = torch.zeros(s["dst"][c].shape[:3] + (dk,), dtype=torch.float64, device="cuda")
        for i in range(nseq):
            m, at = min(n[i], keep), kept[i].clamp(min=0).long().cuda()
            for h in range(Hkv):
                rows = s["src"][c][i, h][at[h, :m]]
                full[i, h, :m] = rows.double() if case["rows"] == "f32" else _rows4(
                    rows, s["src"][c + 1][i, h][at[h, :m]].unflatten(-1, (-1, 2)))
        out.append(full if case["rows"] == "f32" else full.transpose(1, 2))
    return out
