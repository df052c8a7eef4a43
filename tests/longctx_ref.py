"""The long-context operators in plain float64 (torch, any device), one sequence and head at a time."""
import math

import torch

GROUP = 64


def weights(logits, ok):
    """Softmax of the visible places of each row; rows without any are zero."""
    x = logits.masked_fill(~ok, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = (x - m.masked_fill(m == -math.inf, 0.0)).exp().masked_fill(~ok, 0.0)
    return e / e.sum(-1, keepdim=True).clamp(min=1e-300)


def mask(nk, nq, window, sinks, device):
    p = torch.arange(nk - nq, nk, device=device)[:, None]
    j = torch.arange(nk, device=device)[None]
    ok = j <= p
    return ok & ((p - j < window) | (j < sinks)) if window else ok


def attention(q, k, v, scale, window, sinks):
    """q [tq, H, dk], k / v [tk, Hkv, dk] -> out [tq, H, dk], per-key weights [Hkv, tk], the largest sum |q k| * scale
    of a visible pair and the largest |v| (for error bounds). Values of keys that a row cannot see are not touched."""
    tq, H, dk = q.shape
    tk, Hkv = k.shape[0], k.shape[1]
    out = torch.zeros((tq, H, dk), dtype=torch.float64, device=q.device)
    wsum = torch.zeros((Hkv, tk), dtype=torch.float64, device=q.device)
    big = top = 0.0
    if tk:
        ok = mask(tk, tq, window, sinks, q.device)
        for h in range(H):
            g = h // (H // Hkv)
            qh, kh, vh = q[:, h].double(), k[:, g].double(), v[:, g].double()
            w = weights(qh @ kh.T * scale, ok)
            if bool(torch.isfinite(vh).all()):
                out[:, h] = w @ vh
            else:  # row by row over what it sees
                for i in range(tq):
                    if ok[i].any():
                        out[i, h] = w[i, ok[i]] @ vh[ok[i]]
            wsum[g] += w.sum(0)
            seen = (qh.abs() @ kh.abs().T * scale).masked_fill(~ok, 0.0)
            big = max(big, float(seen[torch.isfinite(seen)].max()) if seen.numel() else 0.0)
            fv = vh[ok.any(0)]
            top = max(top, float(fv[torch.isfinite(fv)].abs().max()) if torch.isfinite(fv).any() else 0.0)
    return out, wsum, big, top


def quantize(x):
    """[..., dk] -> integer codes [..., dk], and steps and lowest values [..., dk / 64] (fp16), operation by operation
    in fp32 as the store defines them."""
    g = x.float().unflatten(-1, (-1, GROUP))
    fin = torch.isfinite(g).all(-1)
    g = torch.where(fin[..., None], g, torch.zeros_like(g))
    lo, hi = g.amin(-1), g.amax(-1)
    step = torch.minimum((hi - lo) * torch.tensor(1.0 / 15.0, dtype=torch.float32), torch.tensor(65504.0)).half() \
        if not g.is_cuda else ((hi - lo) * (1.0 / 15.0)).clamp(max=65504.0).half()
    low = lo.clamp(-65504.0, 65504.0).half()
    s = step.float()[..., None]
    code = torch.where(s > 0, torch.round((g - low.float()[..., None]) / s), torch.zeros_like(g)).clamp(0, 15)
    nan = torch.full_like(step, math.nan)
    return code.to(torch.uint8).flatten(-2), torch.where(fin, step, nan), torch.where(fin, low, nan)


def values(code, step, low):
    c = code.double().unflatten(-1, (-1, GROUP))
    return (c * step.double()[..., None] + low.double()[..., None]).flatten(-2)


def pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def unpack(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)
