"""The long-context operators (ork_b200_attn_async, _kv4_store_async, _kv4_load_async, _kv4_attn_async, _evict_async)
against plain float64, at the sizes and masks where they can go wrong, and their refusals.

Error bounds. A logit is a sum of dk products of operands that are exact (fp16 / bf16 inputs, 4-bit codes) or split
in two halves of 11 bits (residual 2^-22 relative), added in fp32 in at most 16 partial steps that may truncate
(2^-23 each): its error is at most d = 2^-18 * sum |q k| scale (two bits to spare), plus 2^-20 for the exponential's
own. A softmax weight is then off by 2 d relatively, numerator and denominator, the output by 4 d max |v|. Where the
weights enter the second product in 16 bits (prompt attention), each adds u / 2 of its weight, u = 2^-10 (fp16) or
2^-7 (bf16), at most u max |v|, and those under fp16's range 2^-25 each. The output's own rounding adds u / 2 of it."""
import ctypes as C
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import longctx_ref as ref  # noqa: E402
import ork_b200 as B  # noqa: E402

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}
NAN = float("nan")


@pytest.fixture
def on(ctx):
    """The session context queueing on torch's stream; errors that a test left behind fail it."""
    ctx.L.ork_b200_set_stream(ctx.ctx, 1)
    yield ctx
    assert ctx.L.ork_b200_sync(ctx.ctx) == 0
    ctx.L.ork_b200_set_stream(ctx.ctx, None)


def rnd(shape, seed, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def bound(typ, out, big, top, nk=0, second=False):
    d = 2.0 ** -18 * big + 2.0 ** -20
    b = 4 * d * top + U[typ] / 2 * out.abs() + 2.0 ** -24
    if second:
        b = b + U[typ] * top + nk * 2.0 ** -25 * top
    return b


def near(got, want, tol):
    got = got.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    bad = ((got - want).abs() > tol) & ~nan & ~(got == want)
    assert not bad.any(), (int(bad.sum()), float((got - want)[bad].abs().max()), bad.nonzero()[:4].tolist())


# ---- prompt attention --------------------------------------------------------------------------------------------

def attn_call(q, k, v, out, tq, tk, typ, window=0, sinks=0, scale=None, /, **over):
    H, Hkv, dk = q.shape[1], k.shape[1], q.shape[2]
    st = lambda n: ints([sum(n[:i]) for i in range(len(n) + 1)])  # noqa: E731
    qs, ks = st(tq), st(tk)
    a = B.Attn(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), type=B.TYPES[typ], nseq=len(tq), H=H,
               Hkv=Hkv, dk=dk, q_ts=q.stride(0), q_hs=q.stride(1), k_ts=k.stride(0), k_hs=k.stride(1), v_ts=v.stride(0),
               v_hs=v.stride(1), o_ts=out.stride(0), o_hs=out.stride(1), q_start=qs.data_ptr(), k_start=ks.data_ptr(),
               q_rows=q.shape[0], k_rows=k.shape[0], max_q=max(tq), max_k=max(tk), scale=scale or dk ** -0.5,
               window=window, sinks=sinks)
    for n, x in over.items():
        setattr(a, n, x)
    return a, (qs, ks)


def attn_check(on, q, k, v, tq, tk, typ, window=0, sinks=0, out=None, scale=None):
    out = torch.full_like(q, NAN) if out is None else out
    a, held = attn_call(q, k, v, out, tq, tk, typ, window, sinks, scale)
    assert on.L.ork_b200_attn_async(on.ctx, C.byref(a)) == 0
    assert on.L.ork_b200_sync(on.ctx) == 0
    q0 = k0 = 0
    for a_, b_ in zip(tq, tk):
        want, _, big, top = ref.attention(q[q0:q0 + a_], k[k0:k0 + b_], v[k0:k0 + b_], scale or q.shape[2] ** -0.5, window,
                                          sinks)
        near(out[q0:q0 + a_], want, bound(typ, want, big, top, b_, True))
        q0, k0 = q0 + a_, k0 + b_
    return out


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 4), (8, 2), (6, 2), (16, 1), (5, 1)])
@pytest.mark.parametrize("tq,tk", [([1], [1]), ([2], [129]), ([130], [130]), ([257, 0, 63], [300, 5, 63])])
def test_attn_heads_and_lengths(on, dk, typ, H, Hkv, tq, tk):
    q, k, v = rnd((sum(tq), H, dk), 1, 1.5, DT[typ]), rnd((sum(tk), Hkv, dk), 2, 1, DT[typ]), rnd((sum(tk), Hkv, dk), 3, 1, DT[typ])
    attn_check(on, q, k, v, tq, tk, typ)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 4), (128, 128), (129, 1), (200, 133), (5000, 4), (300, 5000)])
@pytest.mark.parametrize("tq,tk", [(600, 600), (37, 777), (256, 384), (128, 1024)])
def test_attn_windows_and_sinks(on, window, sinks, tq, tk):
    q, k, v = rnd((tq, 4, 128), 4, 1.5, DT["f16"]), rnd((tk, 2, 128), 5, 1, DT["f16"]), rnd((tk, 2, 128), 6, 1, DT["f16"])
    attn_check(on, q, k, v, [tq], [tk], "f16", window, sinks)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_attn_more_rows_than_keys_leaves_rows_empty(on, typ):
    tq, tk = [200, 3, 129], [70, 0, 128]
    q, k, v = rnd((332, 4, 64), 7, 1, DT[typ]), rnd((198, 2, 64), 8, 1, DT[typ]), rnd((198, 2, 64), 9, 1, DT[typ])
    out = attn_check(on, q, k, v, tq, tk, typ)
    assert not out[:130].any() and not out[200:204].any()


def test_attn_strides(on):
    # heads-major k and v with a capacity, q and out as slices of wider rows
    T, H, Hkv, dk = 333, 8, 4, 128
    qkv, kc, vc = rnd((T, H + 3, dk), 10, 1, DT["bf16"]), rnd((Hkv, 512, dk), 11, 1, DT["bf16"]), rnd((Hkv, 512, dk), 12, 1, DT["bf16"])
    kc[:, T:], vc[:, T:] = NAN, math.inf  # past the sequence
    wide = torch.full((T, H + 1, dk + 8), 7.0, device="cuda", dtype=DT["bf16"])
    attn_check(on, qkv[:, 2:2 + H], kc.transpose(0, 1), vc.transpose(0, 1), [T], [T], "bf16", 0, 0, wide[:, :H, :dk])
    assert (wide[:, H] == 7).all() and (wide[..., dk:] == 7).all()


def test_attn_large_logits_and_rising_maxima(on):
    # maxima that rise by hundreds from tile to tile, and rows whose weights sit on one key
    T, dk = 700, 128
    q, k, v = rnd((T, 2, dk), 13, 6, DT["f16"]), rnd((T, 2, dk), 14, 1, DT["f16"]), rnd((T, 2, dk), 15, 1, DT["f16"])
    k *= torch.linspace(0.01, 8, T, device="cuda")[:, None, None].half()
    attn_check(on, q, k, v, [T], [T], "f16")
    k = k.flip(0).contiguous()
    attn_check(on, q, k, v, [T], [T], "f16", 300, 3)


def test_attn_lowest_logits(on):
    # every logit far below zero: a maximum that starts anywhere else would lose the row
    T, dk = 300, 64
    q, k, v = torch.full((T, 1, dk), 30.0, device="cuda", dtype=DT["bf16"]), torch.full((T, 1, dk), -40.0, device="cuda", dtype=DT["bf16"]), rnd((T, 1, dk), 16, 1, DT["bf16"])
    attn_check(on, q, k, v, [T], [T], "bf16")


@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_attn_nonfinite_values_stay_where_they_are_seen(on, bad, typ):
    T, dk = 300, 128
    q, k, v = rnd((T, 2, dk), 17, 1, DT[typ]), rnd((T, 1, dk), 18, 1, DT[typ]), rnd((T, 1, dk), 19, 1, DT[typ])
    v[140, 0, 5] = bad
    out = attn_check(on, q, k, v, [T], [T], typ, 50, 2)
    assert torch.isfinite(out[:140]).all() and torch.isfinite(out[190:]).all()
    assert not torch.isfinite(out[140:190, :, 5]).any()


def test_attn_nonfinite_keys_out_of_sight(on):
    T, dk = 300, 128
    q, k, v = rnd((T, 2, dk), 20, 1, DT["f16"]), rnd((T, 1, dk), 21, 1, DT["f16"]), rnd((T, 1, dk), 22, 1, DT["f16"])
    k[130] = NAN
    out = torch.zeros_like(q)
    a, held = attn_call(q, k, v, out, [T], [T], "f16", 40, 1)
    assert on.L.ork_b200_attn_async(on.ctx, C.byref(a)) == 0 and on.L.ork_b200_sync(on.ctx) == 0
    k2 = k.clone()
    k2[130] = 0
    want, _, big, top = ref.attention(q, k2, v, dk ** -0.5, 40, 1)
    rows = torch.ones(T, dtype=torch.bool)
    rows[130:170] = False
    near(out[rows], want[rows], bound("f16", want[rows], big, top, T, True))
    assert torch.isnan(out[130:170]).all()


def test_attn_repeats_bit_for_bit(on):
    q, k, v = rnd((1000, 8, 128), 23, 1, DT["bf16"]), rnd((1000, 2, 128), 24, 1, DT["bf16"]), rnd((1000, 2, 128), 25, 1, DT["bf16"])
    outs = []
    for _ in range(3):
        out = torch.zeros_like(q)
        a, held = attn_call(q, k, v, out, [1000], [1000], "bf16", 600, 4)
        assert on.L.ork_b200_attn_async(on.ctx, C.byref(a)) == 0 and on.L.ork_b200_sync(on.ctx) == 0
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_attn_refuses(on):
    q, k, v = (torch.zeros((64, 4, 64), device="cuda", dtype=DT["f16"]) for _ in range(3))
    out = torch.full_like(q, 3.0)
    n = on.launches()
    for bad in (dict(type=0), dict(type=3), dict(dk=32), dict(dk=256), dict(H=3, Hkv=2), dict(Hkv=0), dict(nseq=0), dict(window=-1),
                dict(sinks=-1), dict(max_q=65), dict(max_k=65), dict(q_ts=63), dict(k_hs=68), dict(o_ts=100), dict(q_rows=-1),
                dict(q=q.data_ptr() + 2), dict(out=None), dict(k_start=None), dict(v=torch.zeros(4).data_ptr())):
        a, held = attn_call(q, k, v, out, [64], [64], "f16", **bad)
        assert on.L.ork_b200_attn_async(on.ctx, C.byref(a)) == -1, bad
    assert on.L.ork_b200_attn_async(on.ctx, None) == -1 and on.L.ork_b200_attn_async(None, None) == -1
    assert on.launches() == n and on.L.ork_b200_sync(on.ctx) == 0 and (out == 3).all()


def test_attn_row_ranges_outside_the_tensors_are_reported(on):
    q, k, v = (rnd((64, 2, 64), 26 + i, 1, DT["f16"]) for i in range(3))
    out = torch.full_like(q, 3.0)
    a, held = attn_call(q, k, v, out, [32, 32], [32, 32], "f16")
    held[0].copy_(ints([0, 32, 65]))
    assert on.L.ork_b200_attn_async(on.ctx, C.byref(a)) == 0
    assert on.L.ork_b200_sync(on.ctx) == -1
    assert on.L.ork_b200_sync(on.ctx) == 0
    want, _, big, top = ref.attention(q[:32], k[:32], v[:32], 64 ** -0.5, 0, 0)
    near(out[:32], want, bound("f16", want, big, top, 32, True))
    assert (out[32:] == 3).all()


# ---- the 4-bit cache ---------------------------------------------------------------------------------------------

class Cache:
    def __init__(self, nseq, Hkv, dk, cap, fill=0xff, par=NAN):
        self.k = torch.full((nseq, Hkv, cap, dk // 2), fill, dtype=torch.uint8, device="cuda")
        self.kp = torch.full((nseq, Hkv, cap, dk // 64, 2), par, dtype=torch.float16, device="cuda")
        self.v, self.vp = self.k.clone(), self.kp.clone()
        self.c = B.KV4(k=self.k.data_ptr(), v=self.v.data_ptr(), kp=self.kp.data_ptr(), vp=self.vp.data_ptr(), nseq=nseq,
                       Hkv=Hkv, dk=dk, cap=cap)

    def put(self, s, k, v):
        """k, v [n, Hkv, dk] at slots 0.. of sequence s."""
        for x, c, p in ((k, self.k, self.kp), (v, self.v, self.vp)):
            code, step, low = ref.quantize(x)
            c[s, :, :x.shape[0]] = ref.pack(code).transpose(0, 1)
            p[s, :, :x.shape[0]] = torch.stack([step, low], -1).transpose(0, 1)

    def get(self, s, n):
        """float64 values [n, Hkv, dk] of k and v."""
        return tuple(ref.values(ref.unpack(c[s, :, :n]), p[s, :, :n, :, 0], p[s, :, :n, :, 1]).transpose(0, 1)
                     for c, p in ((self.k, self.kp), (self.v, self.vp)))


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,Hkv", [(64, 1), (128, 3)])
@pytest.mark.parametrize("rows,pos", [([1], [0]), ([1, 1, 1], [5, 63, 0]), ([70, 0, 129], [0, 7, 55])])
def test_store_and_load(on, typ, dk, Hkv, rows, pos):
    cap, n = 192, sum(rows)
    c = Cache(len(rows), Hkv, dk, cap)
    was = [x.clone() for x in (c.k, c.kp, c.v, c.vp)]
    k, v = rnd((n, Hkv, dk), 30, 2, DT[typ]), rnd((n, Hkv, dk), 31, 1, DT[typ])
    k[0, 0, :64] = 1.25  # a constant group
    v[0] *= 1e-4 if typ != "f16" else 1
    start, p = ints([sum(rows[:i]) for i in range(len(rows) + 1)]), ints(pos)
    args = (B.TYPES[typ], max(rows), Hkv * dk, dk, start.data_ptr(), p.data_ptr())
    assert on.L.ork_b200_kv4_store_async(on.ctx, C.byref(c.c), k.data_ptr(), v.data_ptr(), *args) == 0
    want = Cache(len(rows), Hkv, dk, cap)
    r0 = 0
    for s, m in enumerate(rows):
        for x, cc, pp in ((k, want.k, want.kp), (v, want.v, want.vp)):
            code, step, low = ref.quantize(x[r0:r0 + m])
            cc[s, :, pos[s]:pos[s] + m] = ref.pack(code).transpose(0, 1)
            pp[s, :, pos[s]:pos[s] + m] = torch.stack([step, low], -1).transpose(0, 1)
        r0 += m
    for x, y in zip((c.k, c.kp, c.v, c.vp), (want.k, want.kp, want.v, want.vp)):
        assert torch.equal(x.view(torch.uint8 if x.dtype == torch.uint8 else torch.int16), y.view(torch.uint8 if y.dtype == torch.uint8 else torch.int16)) \
            or torch.equal(torch.nan_to_num(x.float(), nan=-7), torch.nan_to_num(y.float(), nan=-7))
    ko, vo = torch.full_like(k, NAN), torch.full_like(v, NAN)
    assert on.L.ork_b200_kv4_load_async(on.ctx, C.byref(c.c), ko.data_ptr(), vo.data_ptr(), *args) == 0
    r0 = 0
    for s, m in enumerate(rows):
        for i, got in ((0, ko), (1, vo)):
            full = c.get(s, cap)[i][pos[s]:pos[s] + m]
            assert torch.equal(got[r0:r0 + m], full.float().to(DT[typ]))  # exact in fp32 but for one rounding
        r0 += m
    # half a step from the input, and the fp16 rounding of the step and the lowest value
    err = (ko.double() - k.double()).abs().unflatten(-1, (-1, 64))
    g = k.double().unflatten(-1, (-1, 64))
    step = (g.amax(-1) - g.amin(-1)) / 15
    tol = 0.5 * step + 16 * step * 2.0 ** -11 + g.amin(-1).abs() * 2.0 ** -11 + 2.0 ** -20 + g.abs().amax(-1) * U[typ]
    assert (err <= tol[..., None]).all()


def test_store_strided_rows_and_device_layer_caches(on):
    # rows of fused projections at an odd element offset, and the decode layer's [Hkv][hstride][dk] fp32 caches
    Hkv, dk, n = 2, 64, 33
    wide = rnd((n, 3 * Hkv * dk + 5), 33)
    a, b = Cache(1, Hkv, dk, 64, 0, 0.0), Cache(1, Hkv, dk, 64, 0, 0.0)
    k, v = wide[:, 1:1 + Hkv * dk], wide[:, 3 + Hkv * dk:3 + 2 * Hkv * dk]
    assert on.L.ork_b200_kv4_store_async(on.ctx, C.byref(a.c), k.data_ptr(), v.data_ptr(), 0, n, wide.shape[1], dk, None, None) == 0
    kc, vc = (x.reshape(n, Hkv, dk).transpose(0, 1).contiguous() for x in (k, v))
    assert on.L.ork_b200_kv4_store_async(on.ctx, C.byref(b.c), kc.data_ptr(), vc.data_ptr(), 0, n, dk, n * dk, None, None) == 0
    for x, y in zip((a.k, a.kp, a.v, a.vp), (b.k, b.kp, b.v, b.vp)):
        assert torch.equal(x, y)
    code, step, low = ref.quantize(kc)
    assert torch.equal(a.k[0, :, :n], ref.pack(code)) and torch.equal(a.kp[0, :, :n], torch.stack([step, low], -1))


def test_store_extremes(on):
    x = rnd((8, 1, 64), 34)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2, 0, 3] = NAN
    x[3, 0, 60] = math.inf
    x[4, 0, 9] = -math.inf
    x[5] = -70000.0
    x[6] = 0.0
    c = Cache(1, 1, 64, 64, 0, 0.0)
    assert on.L.ork_b200_kv4_store_async(on.ctx, C.byref(c.c), x.data_ptr(), x.data_ptr(), 0, 8, 64, 64, None, None) == 0
    code, step, low = ref.quantize(x[:, 0])
    p = c.kp[0, 0, :8, 0]
    assert torch.isnan(p[2:5]).all() and not c.k[0, 0, 2:5].any()
    fin = [0, 1, 5, 6, 7]
    assert torch.equal(p[fin], torch.cat([step, low], -1)[fin]) and torch.equal(c.k[0, 0, fin], ref.pack(code)[fin])
    assert torch.equal(c.k, c.v)


def test_store_slots_outside_the_cache_are_reported(on):
    x = rnd((4, 1, 64), 35)
    c = Cache(2, 1, 64, 64, 0, 0.0)
    pos = ints([-1, 63])
    assert on.L.ork_b200_kv4_store_async(on.ctx, C.byref(c.c), x.data_ptr(), x.data_ptr(), 0, 2, 64, 64, None, pos.data_ptr()) == 0
    assert on.L.ork_b200_sync(on.ctx) == -1 and on.L.ork_b200_sync(on.ctx) == 0
    code, _, _ = ref.quantize(x)
    want = torch.zeros_like(c.k)
    want[0, 0, 0], want[1, 0, 63] = ref.pack(code)[1, 0], ref.pack(code)[2, 0]
    assert torch.equal(c.k, want) and torch.equal(c.v, want)


def test_store_refuses(on):
    x = rnd((4, 1, 64), 36)
    c = Cache(1, 1, 64, 64, 0, 0.0)
    n = on.launches()

    def call(kv=None, k=x.data_ptr(), v=x.data_ptr(), t=0, rows=4, ts=64, hs=64, start=None, pos=None):
        kv = B.KV4.from_buffer_copy(c.c) if kv is None else kv
        r = on.L.ork_b200_kv4_store_async(on.ctx, C.byref(kv), k, v, t, rows, ts, hs, start, pos)
        assert r == on.L.ork_b200_kv4_load_async(on.ctx, C.byref(kv), k, v, t, rows, ts, hs, start, pos)
        return r

    for bad in (dict(k=None), dict(v=None), dict(t=3), dict(t=-1), dict(rows=-1), dict(ts=63), dict(hs=32), dict(k=x.data_ptr() + 2),
                dict(pos=torch.zeros(4).data_ptr()), dict(v=torch.zeros(4).data_ptr())):
        assert call(**bad) == -1, bad
    for f, val in (("k", None), ("dk", 32), ("dk", 96), ("cap", 65), ("cap", 0), ("nseq", 0), ("Hkv", 0), ("vp", c.vp.data_ptr() + 4)):
        kv = B.KV4.from_buffer_copy(c.c)
        setattr(kv, f, val)
        assert call(kv=kv) == -1, f
    assert call(rows=0) == 0
    assert on.launches() == n


def attn4(on, c, q, lens, typ, /, window=0, sinks=0, wsum=None, scale=None, out=None, **over):
    nseq, T, H, dk = q.shape
    out = torch.full((nseq, T, H, dk), NAN, device="cuda", dtype=DT[typ]) if out is None else out
    ln = ints(lens)
    a = B.KV4Attn(q=q.data_ptr(), out=out.data_ptr(), type=B.TYPES[typ], H=H, T=T, q_ts=q.stride(1), q_hs=q.stride(2),
                  len=ln.data_ptr(), max_len=max(lens), scale=scale or dk ** -0.5, window=window, sinks=sinks,
                  wsum=None if wsum is None else wsum.data_ptr())
    for n, x in over.items():
        setattr(a, n, x)
    return on.L.ork_b200_kv4_attn_async(on.ctx, C.byref(c.c), C.byref(a)), out


def attn4_raw(on, c, q, over, /):
    """The return code of a call whose fields `over` replaces."""
    out, ln = torch.zeros_like(q), ints([64])
    a = B.KV4Attn(q=q.data_ptr(), out=out.data_ptr(), type=0, H=q.shape[2], T=q.shape[1], q_ts=q.stride(1), q_hs=q.stride(2),
                  len=ln.data_ptr(), max_len=64, scale=1.0, window=0, sinks=0, wsum=None)
    for n, x in over.items():
        setattr(a, n, x)
    return on.L.ork_b200_kv4_attn_async(on.ctx, C.byref(c.c), C.byref(a))


def attn4_check(on, c, q, lens, typ, window=0, sinks=0, weigh=True, scale=None):
    nseq, T, H, dk = q.shape
    Hkv, cap = c.c.Hkv, c.c.cap
    ws = torch.full((nseq, Hkv, cap), 0.5, device="cuda") if weigh else None
    rc, out = attn4(on, c, q, lens, typ, window, sinks, ws, scale)
    assert rc == 0 and on.L.ork_b200_sync(on.ctx) == 0
    for s, n in enumerate(lens):
        k, v = c.get(s, n)
        want, w, big, top = ref.attention(q[s], k, v, scale or dk ** -0.5, window, sinks)
        near(out[s], want, bound(typ, want, big, top))
        if weigh:  # 0.5 plus the weights: twice the logit error, relatively, and the rounding of the sum
            d = 2 * (2.0 ** -18 * big + 2.0 ** -20)
            near(ws[s, :, :n] - 0.5, w, w * d + 2.0 ** -22 * (1 + w))
            assert (ws[s, :, n:] == 0.5).all()
    return out


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,T", [(1, 1, 1), (4, 4, 1), (8, 1, 1), (16, 2, 1), (7, 1, 1), (9, 1, 1), (32, 2, 1), (6, 2, 3), (4, 1, 5)])
def test_kv4_attn_heads_and_types(on, dk, typ, H, Hkv, T):
    lens = [1, 64, 200, 0, 2, 333]
    c = Cache(len(lens), Hkv, dk, 384)
    for s, n in enumerate(lens):
        c.put(s, rnd((n, Hkv, dk), 40 + s), rnd((n, Hkv, dk), 50 + s))
    q = rnd((len(lens), T, H, dk), 60, 1.5, DT[typ])
    out = attn4_check(on, c, q, lens, typ)
    assert not out[3].any()


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 1023, 1025, 4097, 20000])
def test_kv4_attn_lengths(on, n):
    cap = (n + 63) // 64 * 64
    c = Cache(2, 2, 128, cap)
    for s, m in enumerate((n, max(1, n // 2))):
        c.put(s, rnd((m, 2, 128), 70 + s, 1.2) + rnd((1, 2, 128), 72), rnd((m, 2, 128), 74 + s))
    q = rnd((2, 1, 8, 128), 76, 1.5)
    attn4_check(on, c, q, [n, max(1, n // 2)], "f32")


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 64), (63, 4), (64, 0), (65, 133), (500, 4), (5000, 4), (300, 5000)])
@pytest.mark.parametrize("T", [1, 4])
def test_kv4_attn_windows_and_sinks(on, window, sinks, T):
    lens = [1000, 129, 3, 700]
    c = Cache(4, 2, 64, 1024)
    for s, n in enumerate(lens):
        c.put(s, rnd((n, 2, 64), 80 + s), rnd((n, 2, 64), 90 + s))
        # what the mask hides holds NaN
        lo = max(0, n - T - window + 1)
        if lo > sinks:
            c.kp[s, :, sinks:lo] = NAN
            c.vp[s, :, sinks:lo] = math.inf
    q = rnd((4, T, 6, 64), 100, 1.5)
    nseq, _, H, dk = q.shape
    ws = torch.zeros((4, 2, 1024), device="cuda")
    rc, out = attn4(on, c, q, lens, "f32", window, sinks, ws)
    assert rc == 0 and on.L.ork_b200_sync(on.ctx) == 0
    for s, n in enumerate(lens):
        k, v = (torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0) for x in c.get(s, n))
        want, w, big, top = ref.attention(q[s], k, v, dk ** -0.5, window, sinks)
        near(out[s], want, bound("f32", want, big, top))
        near(ws[s, :, :n], w, w * 2 * (2.0 ** -18 * big + 2.0 ** -20) + 2.0 ** -22 * (1 + w))


def test_kv4_attn_scales_of_many_sizes(on):
    # groups whose steps differ by thousands within a head and along the tokens, tiny and huge
    n, dk = 500, 128
    c = Cache(1, 1, dk, 512)
    k, v = rnd((n, 1, dk), 110), rnd((n, 1, dk), 111)
    f = torch.exp(torch.linspace(-12, 8, n, device="cuda"))[:, None, None]
    v = v * f
    v[:, :, 64:] *= 1e-3
    k[:, :, 64:] *= 40
    c.put(0, k, v)
    attn4_check(on, c, rnd((1, 1, 4, dk), 112), [n], "f32")
    c.put(0, k, v.flip(0))
    attn4_check(on, c, rnd((1, 1, 4, dk), 113), [n], "f32")
    c.put(0, k * 1e-3, v * 1e-5)
    out = attn4_check(on, c, rnd((1, 1, 4, dk), 114, 1e4), [n], "f32")
    kk, vv = c.get(0, n)
    want = ref.attention(rnd((1, 1, 4, dk), 114, 1e4)[0], kk, vv, dk ** -0.5, 0, 0)[0]
    assert float((out[0].double() - want).norm() / want.norm()) < 1e-4  # small values keep their digits


def test_kv4_attn_large_queries(on):
    n, dk = 300, 64
    c = Cache(1, 1, dk, 320)
    c.put(0, rnd((n, 1, dk), 115, 1e-3), rnd((n, 1, dk), 116))
    attn4_check(on, c, rnd((1, 1, 3, dk), 117, 1e6), [n], "f32", scale=1e-3)
    c.put(0, rnd((n, 1, dk), 118, 10.0), rnd((n, 1, dk), 119))
    attn4_check(on, c, rnd((1, 2, 3, dk), 120, 1e-6), [n], "f32", scale=1e4)


def test_kv4_attn_nan_token_is_seen_only_where_visible(on):
    c = Cache(1, 2, 64, 128)
    k, v = rnd((100, 2, 64), 121), rnd((100, 2, 64), 122)
    c.put(0, k, v)
    c.vp[0, 1, 98] = NAN
    q = rnd((1, 3, 4, 64), 123)  # positions 97, 98, 99
    rc, out = attn4(on, c, q, [100], "f32")
    assert rc == 0 and on.L.ork_b200_sync(on.ctx) == 0
    assert torch.isfinite(out[0, 0]).all() and torch.isfinite(out[0, :, :2]).all() and torch.isnan(out[0, 1:, 2:]).all()


def test_kv4_attn_strided_queries(on):
    c = Cache(2, 2, 64, 128)
    for s in range(2):
        c.put(s, rnd((100, 2, 64), 124 + s), rnd((100, 2, 64), 126 + s))
    wide = rnd((2, 3, 5, 67), 128, 1, DT["f16"])
    q = wide[:, :, :4, 1:65]
    assert q.stride(0) == 3 * q.stride(1)
    attn4_check(on, c, q, [100, 77], "f16")
    heads = rnd((4, 6, 64), 129).permute(1, 0, 2).unflatten(0, (2, 3))  # [H][rows][dk], as the prompt glue leaves it
    attn4_check(on, c, heads, [100, 77], "f32")


def test_kv4_attn_repeats_bit_for_bit_and_on_another_stream(on):
    n = 9000
    c = Cache(2, 2, 128, 9024)
    for s in range(2):
        c.put(s, rnd((n, 2, 128), 130 + s), rnd((n, 2, 128), 132 + s))
    q = rnd((2, 1, 16, 128), 134)
    got = []
    for _ in range(3):
        ws = torch.zeros((2, 2, 9024), device="cuda")
        rc, out = attn4(on, c, q, [n, n - 7], "f32", wsum=ws)
        assert rc == 0 and on.L.ork_b200_sync(on.ctx) == 0
        got.append((out, ws))
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    on.L.ork_b200_set_stream(on.ctx, st.cuda_stream)
    ws = torch.zeros((2, 2, 9024), device="cuda")
    torch.cuda.synchronize()
    rc, out = attn4(on, c, q, [n, n - 7], "f32", wsum=ws)
    assert rc == 0 and on.L.ork_b200_sync(on.ctx) == 0
    on.L.ork_b200_set_stream(on.ctx, 1)
    got.append((out, ws))
    for o, w in got[1:]:
        assert torch.equal(o, got[0][0]) and torch.equal(w, got[0][1])


def test_kv4_attn_accumulates_over_calls(on):
    c = Cache(1, 1, 64, 128)
    c.put(0, rnd((100, 1, 64), 135), rnd((100, 1, 64), 136))
    ws, want = torch.zeros((1, 1, 128), device="cuda"), torch.zeros(100, dtype=torch.float64, device="cuda")
    for i in range(4):
        q = rnd((1, 1, 2, 64), 137 + i)
        rc, out = attn4(on, c, q, [97 + i], "f32", wsum=ws)
        assert rc == 0
        k, v = c.get(0, 97 + i)
        want[:97 + i] += ref.attention(q[0], k, v, 0.125, 0, 0)[1][0]
    assert on.L.ork_b200_sync(on.ctx) == 0
    near(ws[0, 0, :100], want, want * 2.0 ** -13 + 2.0 ** -20)
    assert abs(float(ws.sum()) - 8) < 1e-4


def test_kv4_attn_in_a_graph(on):
    c = Cache(1, 2, 64, 256)
    c.put(0, rnd((200, 2, 64), 141), rnd((200, 2, 64), 142))
    q, out = rnd((1, 1, 4, 64), 143), torch.zeros((1, 1, 4, 64), device="cuda")
    ws, ln = torch.zeros((1, 2, 256), device="cuda"), ints([0])
    st = torch.cuda.Stream()
    on.L.ork_b200_set_stream(on.ctx, st.cuda_stream)
    args = dict(len=ln.data_ptr(), max_len=256)
    torch.cuda.synchronize()
    assert attn4(on, c, q, [256], "f32", wsum=ws, out=out, **args)[0] == 0
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        a = B.KV4Attn(q=q.data_ptr(), out=out.data_ptr(), type=0, H=4, T=1, q_ts=256, q_hs=64, len=ln.data_ptr(), max_len=256,
                      scale=0.125, window=0, sinks=0, wsum=ws.data_ptr())
        assert on.L.ork_b200_kv4_attn_async(on.ctx, C.byref(c.c), C.byref(a)) == 0
    for n in (1, 200, 64):
        ln.copy_(ints([n]))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        k, v = c.get(0, n)
        want, w, big, top = ref.attention(q[0], k, v, 0.125, 0, 0)
        near(out[0], want, bound("f32", want, big, top))
    on.L.ork_b200_set_stream(on.ctx, 1)


def test_kv4_attn_offsets_past_32_bits(on):
    # a cache whose arrays pass 4 GiB: the last sequence's rows lie past 2^32 bytes
    nseq, Hkv, dk, cap = 33, 2, 128, 1 << 20
    c = Cache(nseq, Hkv, dk, cap, 0, 0.0)
    assert c.k.numel() > 1 << 32
    k, v = rnd((300, Hkv, dk), 144), rnd((300, Hkv, dk), 145)
    rows, pos = torch.cat([k] * 1), ints([0] * 32 + [cap - 300])
    start = ints([0] * 33 + [300])
    assert on.L.ork_b200_kv4_store_async(on.ctx, C.byref(c.c), rows.data_ptr(), v.data_ptr(), 0, 300, Hkv * dk, dk,
                                         start.data_ptr(), pos.data_ptr()) == 0
    q = rnd((nseq, 1, 4, dk), 146)
    rc, out = attn4(on, c, q, [0] * 32 + [cap], "f32", window=300)
    assert rc == 0 and on.L.ork_b200_sync(on.ctx) == 0
    code, step, low = ref.quantize(k)
    kv = ref.values(code, step, low)
    code, step, low = ref.quantize(v)
    want, _, big, top = ref.attention(q[32], kv, ref.values(code, step, low), dk ** -0.5, 0, 0)
    near(out[32], want, bound("f32", want, big, top))
    assert not out[:32].any()


def test_kv4_attn_lengths_outside_the_cache_are_reported(on):
    c = Cache(3, 1, 64, 128)
    for s in range(3):
        c.put(s, rnd((100, 1, 64), 147), rnd((100, 1, 64), 148))
    q = rnd((3, 1, 2, 64), 149)
    ws = torch.zeros((3, 1, 128), device="cuda")
    rc, out = attn4(on, c, q, [129, 100, -1], "f32", wsum=ws, max_len=128)
    assert rc == 0 and on.L.ork_b200_sync(on.ctx) == -1 and on.L.ork_b200_sync(on.ctx) == 0
    assert not out[0].any() and not out[2].any() and not ws[0].any() and not ws[2].any()
    k, v = c.get(1, 100)
    want, _, big, top = ref.attention(q[1], k, v, 0.125, 0, 0)
    near(out[1], want, bound("f32", want, big, top))


def test_kv4_attn_refuses(on):
    c = Cache(1, 2, 64, 128, 0, 0.0)
    q = torch.zeros((1, 1, 4, 64), device="cuda")
    n = on.launches()
    for bad in (dict(type=3), dict(H=3), dict(H=0), dict(T=0), dict(q_ts=32), dict(q_hs=63), dict(max_len=129), dict(max_len=-1),
                dict(window=-1), dict(sinks=-1), dict(q=None), dict(out=None), dict(len=None), dict(q=q.data_ptr() + 2),
                dict(len=torch.zeros(4).data_ptr()), dict(wsum=torch.zeros(4).data_ptr())):
        assert attn4_raw(on, c, q, bad) == -1, bad
    assert on.L.ork_b200_kv4_attn_async(on.ctx, C.byref(c.c), None) == -1
    assert on.launches() == n


# ---- eviction ----------------------------------------------------------------------------------------------------

def evict_want(score, n, keep, sinks, recent):
    """The kept slots, by the definition: a stable sort by score, the forced ones first."""
    s = [(-math.inf if x != x else x) for x in score[:n].tolist()]
    forced = [j for j in range(n) if j < sinks or j >= n - recent]
    rest = sorted((j for j in range(n) if not (j < sinks or j >= n - recent)), key=lambda j: (-s[j], j))
    return sorted((forced + rest)[:keep])


def evict_check(on, lens, Hkv, cap, keep, sinks, recent, row_bytes, score, dcap=None, align=0):
    nseq, dcap = len(lens), dcap or keep
    g = torch.Generator(device="cuda").manual_seed(5)
    src = [torch.randint(0, 256, (nseq * Hkv * cap * b + align,), dtype=torch.uint8, device="cuda", generator=g) for b in row_bytes]
    dst = [torch.full((nseq * Hkv * dcap * b + align,), 9, dtype=torch.uint8, device="cuda") for b in row_bytes]
    kept = torch.full((nseq, Hkv, keep), 99, dtype=torch.int32, device="cuda")
    so, lo, ln = torch.full((nseq, Hkv, dcap), 5.0, device="cuda"), ints([77] * nseq), ints(lens)
    e = B.Evict(score=score.data_ptr(), len=ln.data_ptr(), nseq=nseq, Hkv=Hkv, cap=cap, dcap=dcap, max_len=max(lens), keep=keep,
                sinks=sinks, recent=recent, nplanes=len(src), kept=kept.data_ptr(), score_out=so.data_ptr(), len_out=lo.data_ptr())
    for i, b in enumerate(row_bytes):
        e.src[i], e.dst[i], e.row_bytes[i] = src[i].data_ptr() + align, dst[i].data_ptr() + align, b
    assert on.L.ork_b200_evict_async(on.ctx, C.byref(e)) == 0 and on.L.ork_b200_sync(on.ctx) == 0
    sc = score.cpu()
    S = [x[align:].view(nseq, Hkv, cap, b).cpu() for x, b in zip(src, row_bytes)]
    D = [x[align:].view(nseq, Hkv, dcap, b).cpu() for x, b in zip(dst, row_bytes)]
    kept, so = kept.cpu(), so.cpu()
    for s, n in enumerate(lens):
        m = min(n, keep)
        assert int(lo[s]) == m
        for h in range(Hkv):
            at = evict_want(sc[s, h], n, keep, sinks, recent)
            assert kept[s, h].tolist() == at + [-1] * (keep - m), (s, h)
            got, want = so[s, h, :m], sc[s, h][at]
            assert torch.equal(torch.nan_to_num(got, nan=-123), torch.nan_to_num(want, nan=-123))
            assert (so[s, h, m:keep] == 0).all() and (so[s, h, keep:] == 5).all()
            for a, b in zip(S, D):
                assert torch.equal(b[s, h, :m], a[s, h][at])
                assert (b[s, h, m:] == 9).all()


@pytest.mark.parametrize("lens,keep,sinks,recent", [([1], 1, 0, 0), ([100, 0, 7], 10, 2, 3), ([5000, 4999], 1024, 4, 256),
                                                   ([300], 300, 4, 9), ([300], 400, 4, 9), ([2050], 1, 1, 0), ([2050], 7, 0, 7),
                                                   ([9000], 8999, 4, 64), ([700, 1025], 64, 32, 32)])
def test_evict_lengths_and_budgets(on, lens, keep, sinks, recent):
    cap = max(lens) + 3
    score = torch.exp(rnd((len(lens), 2, cap), 150, 3))
    evict_check(on, lens, 2, cap, keep, sinks, recent, [64, 8, 64, 8], score)


def test_evict_ties_go_to_the_lowest_slot(on):
    score = torch.zeros((2, 2, 3000), device="cuda")
    score[0, 1] = (torch.arange(3000, device="cuda") % 7).float()
    score[1, 0] = -(torch.arange(3000, device="cuda") % 3).float()
    score[1, 0, ::5] *= 0.0  # minus zero counts as zero
    evict_check(on, [3000, 2777], 2, 3000, 1111, 3, 100, [16], score)


def test_evict_scores_of_every_kind(on):
    score = rnd((1, 3, 4000), 151, 1e3)
    score[0, 0, 5::9], score[0, 0, 7::11], score[0, 0, 8::13] = NAN, math.inf, -math.inf
    score[0, 1] *= 1e-42  # subnormal scores keep their order
    score[0, 2] = -score[0, 2].abs()
    evict_check(on, [3999], 3, 4000, 2000, 4, 10, [4, 12], score)
    score[0, 0, :] = NAN
    score[0, 0, 100] = -math.inf
    evict_check(on, [3999], 3, 4000, 50, 4, 10, [4], score)


@pytest.mark.parametrize("row_bytes,align", [([4], 0), ([8, 20], 4), ([512, 256], 0), ([512], 8), ([68, 1024], 0)])
def test_evict_rows_of_any_width(on, row_bytes, align):
    score = torch.rand((3, 2, 1500), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    evict_check(on, [1500, 800, 1499], 2, 1500, 900, 4, 100, row_bytes, score, 912, align)


def test_evict_long(on):
    score = torch.exp(rnd((1, 1, 150000), 152, 3))
    evict_check(on, [149999], 1, 150000, 40000, 4, 1000, [4], score)


def test_evict_without_planes_or_outputs(on):
    score = torch.rand((1, 1, 200), device="cuda")
    ln, kept = ints([200]), torch.zeros(20, dtype=torch.int32, device="cuda")
    e = B.Evict(score=score.data_ptr(), len=ln.data_ptr(), nseq=1, Hkv=1, cap=200, dcap=20, max_len=200, keep=20, sinks=0, recent=0,
                nplanes=0, kept=kept.data_ptr())
    assert on.L.ork_b200_evict_async(on.ctx, C.byref(e)) == 0 and on.L.ork_b200_sync(on.ctx) == 0
    assert kept.tolist() == evict_want(score[0, 0].cpu(), 200, 20, 0, 0)
    e.kept = None
    assert on.L.ork_b200_evict_async(on.ctx, C.byref(e)) == 0 and on.L.ork_b200_sync(on.ctx) == 0


def test_evict_lengths_outside_the_cache_are_reported(on):
    score = torch.rand((2, 1, 64), device="cuda")
    ln, kept, lo = ints([65, 64]), torch.zeros((2, 1, 8), dtype=torch.int32, device="cuda"), ints([5, 5])
    e = B.Evict(score=score.data_ptr(), len=ln.data_ptr(), nseq=2, Hkv=1, cap=64, dcap=8, max_len=64, keep=8, sinks=0, recent=0,
                nplanes=0, kept=kept.data_ptr(), len_out=lo.data_ptr())
    assert on.L.ork_b200_evict_async(on.ctx, C.byref(e)) == 0
    assert on.L.ork_b200_sync(on.ctx) == -1 and on.L.ork_b200_sync(on.ctx) == 0
    assert lo.tolist() == [0, 8] and (kept[0] == -1).all()
    assert kept[1, 0].tolist() == evict_want(score[1, 0].cpu(), 64, 8, 0, 0)


def test_evict_refuses(on):
    score, ln = torch.zeros((1, 1, 64), device="cuda"), ints([64])
    a, b = torch.zeros(64 * 16, dtype=torch.uint8, device="cuda"), torch.zeros(64 * 16, dtype=torch.uint8, device="cuda")
    n = on.launches()

    def call(**over):
        e = B.Evict(score=score.data_ptr(), len=ln.data_ptr(), nseq=1, Hkv=1, cap=64, dcap=32, max_len=64, keep=32, sinks=4, recent=8,
                    nplanes=1)
        e.src[0], e.dst[0], e.row_bytes[0] = a.data_ptr(), b.data_ptr(), 16
        for k, x in over.items():
            if k in ("src", "dst", "row_bytes"):
                getattr(e, k)[0] = x
            else:
                setattr(e, k, x)
        return on.L.ork_b200_evict_async(on.ctx, C.byref(e))

    for bad in (dict(score=None), dict(len=None), dict(nseq=0), dict(Hkv=0), dict(cap=0), dict(keep=0), dict(dcap=31), dict(max_len=65),
                dict(max_len=-1), dict(sinks=-1), dict(recent=-1), dict(sinks=30), dict(nplanes=9), dict(nplanes=-1), dict(nplanes=2),
                dict(src=None), dict(dst=None), dict(row_bytes=3), dict(row_bytes=0), dict(dst=a.data_ptr()), dict(dst=a.data_ptr() + 512),
                dict(src=a.data_ptr() + 2), dict(score_out=score.data_ptr()), dict(kept=torch.zeros(4).data_ptr())):
        assert call(**bad) == -1, bad
    assert on.launches() == n


# ---- together ----------------------------------------------------------------------------------------------------

def test_prompt_store_decode_evict_decode(on):
    """A prompt's attention and store, decode steps that accumulate weights, an eviction, and steps on what is left."""
    H, Hkv, dk, T, cap, keep, sinks, recent = 8, 2, 128, 300, 384, 128, 4, 32
    q, k, v = rnd((T, H, dk), 160, 1.5, DT["f16"]), rnd((T, Hkv, dk), 161, 1, DT["f16"]), rnd((T, Hkv, dk), 162, 1, DT["f16"])
    attn_check(on, q, k, v, [T], [T], "f16")
    c, d = Cache(1, Hkv, dk, cap), Cache(1, Hkv, dk, keep + 64)
    assert on.L.ork_b200_kv4_store_async(on.ctx, C.byref(c.c), k.data_ptr(), v.data_ptr(), 1, T, Hkv * dk, dk, None, None) == 0
    ws = torch.zeros((1, Hkv, cap), device="cuda")
    want = torch.zeros((Hkv, cap), dtype=torch.float64, device="cuda")

    def step(cache, n, seed, w=None):
        x = [rnd((1, h, dk), seed + i, 1.2, DT["f16"]) for i, h in enumerate((H, Hkv, Hkv))]
        pos = ints([n])
        assert on.L.ork_b200_kv4_store_async(on.ctx, C.byref(cache.c), x[1].data_ptr(), x[2].data_ptr(), 1, 1, Hkv * dk, dk, None,
                                             pos.data_ptr()) == 0
        rc, out = attn4(on, cache, x[0][None], [n + 1], "f16", wsum=w)
        assert rc == 0 and on.L.ork_b200_sync(on.ctx) == 0
        kk, vv = cache.get(0, n + 1)
        o, sums, big, top = ref.attention(x[0], kk, vv, dk ** -0.5, 0, 0)
        near(out[0], o, bound("f16", o, big, top))
        return sums

    for i in range(20):
        want[:, :T + i + 1] += step(c, T + i, 170 + 3 * i, ws)
    n = T + 20
    near(ws[0], want, want * 2.0 ** -12 + 2.0 ** -18)
    ln, kept, so, lo = ints([n]), torch.zeros((1, Hkv, keep), dtype=torch.int32, device="cuda"), torch.zeros((1, Hkv, keep + 64), device="cuda"), ints([0])
    e = B.Evict(score=ws.data_ptr(), len=ln.data_ptr(), nseq=1, Hkv=Hkv, cap=cap, dcap=keep + 64, max_len=n, keep=keep, sinks=sinks,
                recent=recent, nplanes=4, kept=kept.data_ptr(), score_out=so.data_ptr(), len_out=lo.data_ptr())
    for i, (x, y) in enumerate(((c.k, d.k), (c.kp, d.kp), (c.v, d.v), (c.vp, d.vp))):
        e.src[i], e.dst[i], e.row_bytes[i] = x.data_ptr(), y.data_ptr(), x[0, 0, 0].numel() * x.element_size()
    assert on.L.ork_b200_evict_async(on.ctx, C.byref(e)) == 0 and on.L.ork_b200_sync(on.ctx) == 0
    kk, vv = c.get(0, n)
    gk, gv = d.get(0, keep)
    for h in range(Hkv):
        at = torch.tensor(evict_want(ws[0, h].cpu(), n, keep, sinks, recent), device="cuda")
        assert torch.equal(gk[:, h], kk[at, h]) and torch.equal(gv[:, h], vv[at, h])
    for i in range(5):
        step(d, keep + i, 300 + 3 * i, so)


def test_the_example_runs_within_its_budget():
    import os
    import re
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "examples", "long_context.py"), "--prompt", "700", "--tokens", "700",
                        "--budget", "512", "--sequences", "3"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    held = [int(x) for x in re.search(r"tokens held \[(.*?)\]", r.stdout).group(1).split(",")]
    # caches of 512 + 444 rounded up to 960 tokens: full after 260 of the 700 steps, down to 512, 440 more
    assert "1 evictions" in r.stdout and held == [952] * 3 and "4.50 bits" in r.stdout
