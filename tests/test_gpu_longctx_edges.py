"""The long-context operators at their edges: arrays updated in place, values far apart, calls that come late.

Tolerances are derived beside each test. u is the spacing of the output's type at 1 (2^-10 fp16, 2^-7 bf16, 2^-23 fp32)."""
import ctypes as C
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import longctx_ref as ref  # noqa: E402
import ork_b200 as B  # noqa: E402
from test_gpu_longctx import evict_want, ints, on, rnd  # noqa: E402,F401


# ---- eviction ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("nseq,Hkv,n,keep", [(40, 8, 3000, 700), (2, 8, 9000, 2000), (1, 1, 40000, 64), (300, 1, 600, 599)])
def test_evict_updates_lengths_in_place(on, nseq, Hkv, n, keep):
    # len_out is len: every head of every sequence picks from all its tokens, whichever is done first
    cap = n + 8
    lens = [max(0, n - 131 * s) for s in range(nseq)]
    score = torch.exp(rnd((nseq, Hkv, cap), 400, 3))
    ln, kept = ints(lens), torch.zeros((nseq, Hkv, keep), dtype=torch.int32, device="cuda")
    e = B.Evict(score=score.data_ptr(), len=ln.data_ptr(), nseq=nseq, Hkv=Hkv, cap=cap, dcap=keep, max_len=max(lens), keep=keep,
                sinks=2, recent=5, nplanes=0, kept=kept.data_ptr(), len_out=ln.data_ptr())
    assert on.L.ork_b200_evict_async(on.ctx, C.byref(e)) == 0 and on.L.ork_b200_sync(on.ctx) == 0
    assert ln.tolist() == [min(x, keep) for x in lens]
    sc, kept = score.cpu(), kept.cpu()
    for s, m in enumerate(lens):
        for h in range(Hkv):
            at = evict_want(sc[s, h], m, keep, 2, 5)
            assert kept[s, h].tolist() == at + [-1] * (keep - len(at)), (s, h)


def test_evict_of_more_keys_than_a_block_holds(on):
    # so many heads that each gets one block, and so many tokens that it reads the scores anew in every pass
    nseq, Hkv, n, keep = 19, 8, 25000, 500
    score = torch.exp(rnd((nseq, Hkv, n), 404, 3))
    score[:, 0] = torch.floor(score[:, 0])  # many ties
    ln, kept = ints([n - 7 * s for s in range(nseq)]), torch.zeros((nseq, Hkv, keep), dtype=torch.int32, device="cuda")
    e = B.Evict(score=score.data_ptr(), len=ln.data_ptr(), nseq=nseq, Hkv=Hkv, cap=n, dcap=keep, max_len=n, keep=keep, sinks=4,
                recent=64, nplanes=0, kept=kept.data_ptr(), len_out=ln.data_ptr())
    assert on.L.ork_b200_evict_async(on.ctx, C.byref(e)) == 0 and on.L.ork_b200_sync(on.ctx) == 0
    assert ln.tolist() == [keep] * nseq
    sc, kept = score.cpu(), kept.cpu()
    for s in range(0, nseq, 3):
        for h in (0, 1 + s % 7):
            assert kept[s, h].tolist() == evict_want(sc[s, h], n - 7 * s, keep, 4, 64), (s, h)


# ---- CUDA graphs and the workspace --------------------------------------------------------------------------------

def cache(nseq, Hkv, dk, cap, seed):
    from test_gpu_longctx import Cache

    c = Cache(nseq, Hkv, dk, cap)
    for s in range(nseq):
        c.put(s, rnd((cap, Hkv, dk), seed + 2 * s), rnd((cap, Hkv, dk), seed + 2 * s + 1))
    return c


def kv4_args(q, out, ln, n, wsum=None, typ="f32", scale=None, window=0, sinks=0):
    return B.KV4Attn(q=q.data_ptr(), out=out.data_ptr(), type=B.TYPES[typ], H=q.shape[2], T=q.shape[1], q_ts=q.stride(1),
                     q_hs=q.stride(2), len=ln.data_ptr(), max_len=n, scale=scale or q.shape[3] ** -0.5, window=window,
                     sinks=sinks, wsum=None if wsum is None else wsum.data_ptr())


def test_a_graph_replays_after_larger_calls(on):
    # the graph's workspace and counters stay its own when a later call needs more
    with B.Context() as own:
        st = torch.cuda.Stream()
        own.L.ork_b200_set_stream(own.ctx, st.cuda_stream)
        n, big = 2000, 60000
        c, d = cache(1, 2, 64, 2048, 410), cache(1, 2, 64, 60032, 412)
        q, out, want = rnd((1, 1, 8, 64), 414), torch.zeros((1, 1, 8, 64), device="cuda"), torch.zeros((1, 1, 8, 64), device="cuda")
        q2, out2, ws2 = rnd((1, 64, 8, 64), 415), torch.zeros((1, 64, 8, 64), device="cuda"), torch.zeros((1, 2, 60032), device="cuda")
        ws, ln, ln2 = torch.zeros((1, 2, 2048), device="cuda"), ints([n]), ints([big])
        torch.cuda.synchronize()
        assert own.L.ork_b200_kv4_attn_async(own.ctx, C.byref(c.c), C.byref(kv4_args(q, want, ln, n, ws))) == 0
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            assert own.L.ork_b200_kv4_attn_async(own.ctx, C.byref(c.c), C.byref(kv4_args(q, out, ln, n, ws))) == 0
            # what would allocate is refused, and the capture goes on
            assert own.L.ork_b200_kv4_attn_async(own.ctx, C.byref(d.c), C.byref(kv4_args(q2, out2, ln2, big, ws2))) == -1
        small = own.L.ork_b200_staging_bytes(own.ctx)
        assert own.L.ork_b200_kv4_attn_async(own.ctx, C.byref(d.c), C.byref(kv4_args(q2, out2, ln2, big, ws2))) == 0
        torch.cuda.synchronize()
        large = own.L.ork_b200_staging_bytes(own.ctx)
        assert large - small >= 64 * 8 * big * 4  # the logits' block is new, the graph's is still held
        torch.cuda.empty_cache()
        other = [torch.full((1 << 18,), 7, dtype=torch.int32, device="cuda") for _ in range(64)]
        for i in range(3):
            out.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        assert all(bool((o == 7).all()) for o in other)
        assert abs(float(ws.sum()) - 4 * 8) < 1e-3  # one eager call and three replays, a weight of 1 a head
        assert own.L.ork_b200_kv4_attn_async(own.ctx, C.byref(d.c), C.byref(kv4_args(q2, out2, ln2, big, ws2))) == 0
        assert own.L.ork_b200_sync(own.ctx) == 0 and own.L.ork_b200_staging_bytes(own.ctx) == large
        del g


def test_a_growing_cache_seldom_grows_the_workspace(on):
    # a decode loop's logits grow with every unit of 16 tokens; the workspace by half at a time: 2 MB of logits at first,
    # 8 MB at last, four growths
    with B.Context() as own:
        own.L.ork_b200_set_stream(own.ctx, 1)
        c = cache(1, 8, 64, 32768, 420)
        q, ws, ln = rnd((1, 1, 64, 64), 422), torch.zeros((1, 8, 32768), device="cuda"), ints([100])
        out, sizes = torch.zeros_like(q), set()
        for n in range(8192, 32769, 256):
            assert own.L.ork_b200_kv4_attn_async(own.ctx, C.byref(c.c), C.byref(kv4_args(q, out, ln, n, ws))) == 0
            sizes.add(own.L.ork_b200_staging_bytes(own.ctx))
        assert own.L.ork_b200_sync(own.ctx) == 0
        assert len(sizes) <= 5


# ---- refusals ----------------------------------------------------------------------------------------------------

def test_misaligned_arrays_are_refused(on):
    i, f = ints([0] * 64), torch.zeros(64 * 64, device="cuda")
    h = torch.zeros(64 * 64, dtype=torch.float16, device="cuda")
    c = B.KV4(k=f.data_ptr(), v=f.data_ptr(), kp=h.data_ptr(), vp=h.data_ptr(), nseq=1, Hkv=1, dk=64, cap=64)
    n = on.launches()
    for off in (1, 2):
        ip, fp = i.data_ptr(), f.data_ptr()
        for bad in (dict(q_start=ip + off), dict(k_start=ip + off)):
            a = B.Attn(q=h.data_ptr(), k=h.data_ptr(), v=h.data_ptr(), out=h.data_ptr(), type=1, nseq=1, H=1, Hkv=1, dk=64, q_ts=64,
                       q_hs=64, k_ts=64, k_hs=64, v_ts=64, v_hs=64, o_ts=64, o_hs=64, q_start=ip, k_start=ip, q_rows=1, k_rows=1,
                       max_q=1, max_k=1, scale=1.0)
            for k, x in bad.items():
                setattr(a, k, x)
            assert on.L.ork_b200_attn_async(on.ctx, C.byref(a)) == -1, bad
        for start, pos in ((ip + off, None), (None, ip + off)):
            for call in (on.L.ork_b200_kv4_store_async, on.L.ork_b200_kv4_load_async):
                assert call(on.ctx, C.byref(c), fp, fp, 0, 1, 64, 64, start, pos) == -1
        for bad in (dict(len=ip + off), dict(wsum=fp + off)):
            a = B.KV4Attn(q=fp, out=fp, type=0, H=1, T=1, q_ts=64, q_hs=64, len=ip, max_len=64, scale=1.0)
            for k, x in bad.items():
                setattr(a, k, x)
            assert on.L.ork_b200_kv4_attn_async(on.ctx, C.byref(c), C.byref(a)) == -1, bad
        for bad in (dict(score=fp + off), dict(len=ip + off), dict(kept=ip + off), dict(score_out=fp + 256 + off), dict(len_out=ip + off)):
            e = B.Evict(score=fp, len=ip, nseq=1, Hkv=1, cap=64, dcap=8, max_len=64, keep=8, nplanes=0)
            for k, x in bad.items():
                setattr(e, k, x)
            assert on.L.ork_b200_evict_async(on.ctx, C.byref(e)) == -1, bad
    assert on.launches() == n


# ---- rows into the cache and back --------------------------------------------------------------------------------

@pytest.mark.parametrize("start", [[0, 3, 2, 4], [-2, 1, 2, 4]])
def test_store_offsets_that_decrease_or_are_negative_are_reported(on, start):
    from test_gpu_longctx import Cache

    x = rnd((4, 1, 64), 430)
    c = Cache(3, 1, 64, 64, 0, 0.0)
    st = ints(start)
    args = (0, 4, 64, 64, st.data_ptr(), None)
    assert on.L.ork_b200_kv4_store_async(on.ctx, C.byref(c.c), x.data_ptr(), x.data_ptr(), *args) == 0
    assert on.L.ork_b200_sync(on.ctx) == -1 and on.L.ork_b200_sync(on.ctx) == 0
    want = Cache(3, 1, 64, 64, 0, 0.0)
    for s in range(3):
        if 0 <= start[s] <= start[s + 1]:
            want.put(s, x[start[s]:start[s + 1]], x[start[s]:start[s + 1]])
    assert torch.equal(c.k, want.k) and torch.equal(c.kp, want.kp) and torch.equal(c.v, want.v)
    y = torch.full_like(x, 5.0)
    assert on.L.ork_b200_kv4_load_async(on.ctx, C.byref(c.c), y.data_ptr(), y.data_ptr(), *args) == 0
    assert on.L.ork_b200_sync(on.ctx) == -1 and on.L.ork_b200_sync(on.ctx) == 0


# ---- prompt attention --------------------------------------------------------------------------------------------

def prompt(on, q, k, v, tq, tk, typ, window=0, sinks=0, scale=None):
    from test_gpu_longctx import attn_call

    out = torch.full_like(q, 9.0)
    a, held = attn_call(q, k, v, out, tq, tk, typ, window, sinks, scale)
    assert on.L.ork_b200_attn_async(on.ctx, C.byref(a)) == 0 and on.L.ork_b200_sync(on.ctx) == 0
    return out


def same_but_rounding(got, want, typ, top):
    # a row's weights are within u / 2 each, its output within u / 2 of itself: u max |v| covers both; NaNs and infinities
    # lie where they belong
    u, got = {"f16": 2.0 ** -10, "bf16": 2.0 ** -7}[typ], got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin].nan_to_num(nan=5.0), want[~fin].nan_to_num(nan=5.0))
    assert float((got - want)[fin].abs().max()) <= 1.5 * u * top + 2.0 ** -14


def test_attn_an_infinite_value_that_every_row_sees(on):
    # 256 rows after a prefix of 150000 keys, one early value infinite: every row is computed again, which may take its
    # time, and the other sequence is whole
    tq, tk, dk = [256, 300], [150000, 300], 128
    q, k, v = (rnd((sum(n), 1, dk), 440 + i, 1, torch.float16) for i, n in enumerate((tq, tk, tk)))
    v[7, 0, 5] = math.inf
    out = prompt(on, q, k, v, tq, tk, "f16")
    fin = v.clone()
    fin[7, 0, 5] = 0
    for i, (q0, k0) in enumerate(((0, 0), (256, 150000))):
        want, _, _, top = ref.attention(q[q0:q0 + tq[i]], k[k0:k0 + tk[i]], fin[k0:k0 + tk[i]], dk ** -0.5, 0, 0)
        if i == 0:
            want[:, 0, 5] = math.inf
        same_but_rounding(out[q0:q0 + tq[i]], want, "f16", top)


@pytest.mark.parametrize("typ,dk,H,Hkv,window,sinks", [("f16", 64, 16, 8, 0, 0), ("bf16", 128, 12, 4, 700, 3)])
def test_attn_nonfinite_values_in_many_items(on, typ, dk, H, Hkv, window, sinks):
    # more items than CTAs, most of them with rows that are computed again
    T = 3000
    q, k, v = (rnd((T, h, dk), 444 + i, 1, {"f16": torch.float16, "bf16": torch.bfloat16}[typ]) for i, h in enumerate((H, Hkv, Hkv)))
    fin = v.clone()
    hit = {}
    for g in range(Hkv):
        hit[g] = [(1, 3, math.inf), (90 + 130 * g, dk - 1, math.nan), (2500, 17, -math.inf)]
        for j, d, x in hit[g]:
            v[j, g, d], fin[j, g, d] = x, 0
    out = prompt(on, q, k, v, [T], [T], typ, window, sinks)
    want, _, _, top = ref.attention(q, k, fin, dk ** -0.5, window, sinks)
    ok = ref.mask(T, T, window, sinks, q.device)
    for g in range(Hkv):
        for j, d, x in hit[g]:
            for h in range(g * (H // Hkv), (g + 1) * (H // Hkv)):
                want[ok[:, j], h, d] = x
    same_but_rounding(out, want, typ, top)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("first", [True, False])
def test_attn_a_long_tail_far_below_one_key(on, typ, first):
    # one key 18 nats above 16384 others, and all of the output theirs: 2^-26 of the weight each, 2^-12 together. The tail
    # is within its weights' rounding (u / 2 of each; fp16 holds them to 2^-32 of the largest), the output's, and the
    # logits' error (2^-22 of 18 nats)
    n, dk, top = 16384, 64, 60.0
    u = {"f16": 2.0 ** -10, "bf16": 2.0 ** -7}[typ]
    dt = {"f16": torch.float16, "bf16": torch.bfloat16}[typ]
    q, k, v = torch.zeros((1, 2, dk), device="cuda", dtype=dt), rnd((n + 1, 1, dk), 460, 1, dt), torch.full((n + 1, 1, dk), top, device="cuda", dtype=dt)
    q[..., 0], q[..., 1] = 1.0, 0.25
    k[..., 0] = 0.0
    at = 0 if first else n - 3
    k[at, 0, :2] = torch.tensor([18.0, 0.0], device="cuda").to(dt)
    v[at] = 0.0
    out = prompt(on, q, k, v, [1], [n + 1], typ, scale=1.0)
    want, _, _, _ = ref.attention(q, k, v, 1.0, 0, 0)
    tol = (1.5 * u + 2.0 ** -15) * float(want.max()) + (n * 2.0 ** -32 * top if typ == "f16" else 0.0)
    assert float(want.min()) > 3 * tol
    assert float((out.double() - want).abs().max()) <= tol


# ---- attention over the 4-bit cache ------------------------------------------------------------------------------

@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("power", [118, 121, 124])
def test_kv4_attn_queries_near_the_top_of_their_range(on, typ, power):
    # queries of 2^power and a scale that takes it back: the same logits as those of ordinary queries
    from test_gpu_longctx import Cache, attn4_check

    c = Cache(1, 2, 64, 320)
    c.put(0, rnd((300, 2, 64), 470), rnd((300, 2, 64), 471))
    q = rnd((1, 2, 8, 64), 472, 1.5, {"f32": torch.float32, "bf16": torch.bfloat16}[typ]) * 2.0 ** power
    assert torch.isfinite(q).all()
    attn4_check(on, c, q, [300], typ, scale=0.125 * 2.0 ** -power)


@pytest.mark.parametrize("T,window", [(1, 0), (3, 0), (3, 50)])
@pytest.mark.parametrize("token", [10, 60, 97, 98, 99])
def test_kv4_attn_nan_values_reach_their_own_group_alone(on, T, window, token):
    # wherever the token lies in what is loaded at once: its 64 dims are NaN in the rows that see it, the other dims and
    # the weights are the finite ones
    from test_gpu_longctx import Cache, attn4_check

    c = Cache(1, 2, 128, 128)
    c.put(0, rnd((100, 2, 128), 480), rnd((100, 2, 128), 481))
    c.vp[0, 1, token, 1] = math.nan
    out = attn4_check(on, c, rnd((1, T, 8, 128), 482), [100], "f32", window, 0)
    assert torch.isfinite(out[..., :4, :]).all() and torch.isfinite(out[..., :64]).all()
    seen = torch.tensor([token <= 100 - T + t and (not window or token > 100 - T + t - window) for t in range(T)])
    assert torch.equal(torch.isnan(out[0, :, 4:, 64:]).all(-1).all(-1).cpu(), seen)


def kv4_error_bound(c, q, n, typ, scale, bits=21):
    """For one sequence and token, q [H, dk]: what each output may be off by, and the output. Queries enter as integers
    below 2^bits, a power of two times them, so a logit is off by what that leaves of each dim, times |k|; then by six
    roundings of fp32 (2^-24 each) of its parts, per group step (q . codes) and lowest sum(q), and by 2^-21 of the
    exponential's. Weights are off by that of their own and the mean one, relatively. A value enters as (code - 8) step and
    low + 8 step, times its weight, rounded to u' = 2^-21 (fp32 queries), or to 2^-11 where 16-bit queries take p * step
    in one fp16; products below 2^-16 of a row's largest lose up to 2^-27 of that."""
    k, v = (x[:, 0] for x in c.get(0, n))
    G = k.shape[1] // 64
    codes = ref.unpack(c.k[0, 0, :n]).double().unflatten(-1, (G, 64))
    ks, kl = (c.kp[0, 0, :n, :, i].double() for i in (0, 1))
    step, low = (c.vp[0, 0, :n, :, i].double() for i in (0, 1))
    size = 8 * step + (low + 8 * step).abs()  # [n, G]
    qd = q.double()
    up = 2.0 ** (bits - 1 - torch.floor(torch.log2(qd.abs().amax(-1, keepdim=True))))
    left = (qd * up - torch.round(qd * up)).abs() / up
    x = qd @ k.T * scale
    w = torch.softmax(x, -1)
    qg = qd.unflatten(-1, (G, 64))
    parts = sum(ks[:, g] * (qg[:, g] @ codes[:, g].T).abs() + (kl[:, g] * qg[:, g].sum(-1, keepdim=True)).abs() for g in range(G))
    e = scale * (left @ k.abs().T + 6 * 2.0 ** -24 * parts) + 2.0 ** -21
    e = e + (w * e).sum(-1, keepdim=True)
    u1 = {"f32": 2.0 ** -21, "f16": 2.0 ** -11, "bf16": 2.0 ** -11}[typ]
    lost = 8 * n * 2.0 ** -27 * (w[:, :, None] * step).amax(1)
    tol = (w * (e + u1)) @ size + lost  # [H, G]
    want = w @ v
    u = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}[typ]
    tiny = 2.0 ** -25 if typ == "f16" else 1e-37
    return tol.repeat_interleave(64, -1) + u / 2 * want.abs() + tiny, want


def kv4_digits(on, c, q, n, typ, scale, bits=21):
    from test_gpu_longctx import attn4

    rc, out = attn4(on, c, q[None, None], [n], typ, scale=scale)
    assert rc == 0 and on.L.ork_b200_sync(on.ctx) == 0
    tol, want = kv4_error_bound(c, q, n, typ, scale, bits)
    err = (out[0, 0].double() - want).abs()
    assert (err <= tol).all(), (float((err / tol).max()), float(err.max()))
    return tol, want


DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("small", [0, 1])
@pytest.mark.parametrize("ratio", [1.0, 1e4, 1e6])
def test_kv4_attn_a_group_of_small_values_keeps_its_digits(on, typ, small, ratio):
    # queries in sixteenths are exact as integers, which leaves the values' digits
    from test_gpu_longctx import Cache

    n, dk = 3000, 128
    c = Cache(1, 1, dk, 3008)
    v = rnd((n, 1, dk), 490, 1e4)
    v[:, :, 64 * small:64 * small + 64] /= ratio
    c.put(0, rnd((n, 1, dk), 491), v)
    q = (torch.round(rnd((8, dk), 492, 16.0)) / 16).to(DT[typ])
    kv4_digits(on, c, q, n, typ, dk ** -0.5)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups", [(0, 1), (1,)])
@pytest.mark.parametrize("at", [0, 700, 2999])
def test_kv4_attn_a_large_value_without_weight_costs_no_digits(on, typ, groups, at):
    # one token's values a million times the others', and next to no weight on it
    from test_gpu_longctx import Cache

    n, dk = 3000, 128
    c = Cache(1, 1, dk, 3008)
    k, v = rnd((n, 1, dk), 493), rnd((n, 1, dk), 494, 0.01)
    q = (torch.round(rnd((dk,), 495, 16.0)) / 16).to(DT[typ]).expand(8, dk).contiguous()
    k[at, 0] = -8 * q[0].float()
    for g in groups:
        v[at, :, 64 * g:64 * g + 64] *= 1e6
    c.put(0, k, v)
    kv4_digits(on, c, q, n, typ, dk ** -0.5)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sink", [0.0, 0.01, 1.0])
@pytest.mark.parametrize("at", [0, 20000])
def test_kv4_attn_a_long_tail_far_below_one_token(on, typ, sink, at):
    # a token 17 nats above 32767 others, whose output is theirs where its values are 0
    from test_gpu_longctx import Cache

    n, dk = 32768, 64
    c = Cache(1, 1, dk, n)
    k, v = rnd((n, 1, dk), 496, 0.2), rnd((n, 1, dk), 497, 30.0)
    q = (torch.round(rnd((dk,), 498, 16.0)) / 16).to(DT[typ]).expand(5, dk).contiguous()
    k[at, 0] = q[0].float() / float(q[0].float().norm()) ** 2 * 17.0 * 8.0
    v[at] *= sink
    c.put(0, k, v)
    kv4_digits(on, c, q, n, typ, 0.125)


@pytest.mark.parametrize("dk,H", [(64, 3), (128, 8), (64, 16), (128, 11)])
@pytest.mark.parametrize("n", [8, 50])
def test_kv4_attn_fp32_queries_keep_digits_next_to_large_ones(on, dk, H, n):
    # two dims far above the others that cancel in every logit: integers of 29 bits below them leave the others theirs
    from test_gpu_longctx import Cache

    c = Cache(1, 1, dk, 64)
    k, q = rnd((n, 1, dk), 500), rnd((H, dk), 501, 1.6)
    q[:, 5], q[:, 9], k[..., 5], k[..., 9] = 1000.0, -1000.0, 0.25, 0.25
    c.put(0, k, rnd((n, 1, dk), 502))
    kv4_digits(on, c, q, n, "f32", dk ** -0.5, 29)


@pytest.mark.parametrize("T,H,Hkv,lens,window,sinks,cap", [(70, 8, 1, [500, 71, 30, 0], 0, 0, 512), (33, 12, 4, [1000, 5], 200, 7, 1024),
                                                          (300, 3, 3, [333, 299], 0, 0, 384)])
def test_kv4_attn_many_tokens(on, T, H, Hkv, lens, window, sinks, cap):
    # hundreds of rows a kv head, sequences shorter than the tokens among them
    from test_gpu_longctx import Cache, attn4_check

    c = Cache(len(lens), Hkv, 64, cap)
    for s, n in enumerate(lens):
        c.put(s, rnd((n, Hkv, 64), 510 + s), rnd((n, Hkv, 64), 515 + s))
    attn4_check(on, c, rnd((len(lens), T, H, 64), 520, 1.5), lens, "f32", window, sinks)


def test_kv4_attn_weights_of_many_tokens_in_bounded_memory(on):
    # 9.6 GB of logits: in passes, with a workspace of 4 GiB and half as much again at most; one sequence is shorter than
    # the tokens of the first pass
    from test_gpu_longctx import Cache, attn4_check

    T, lens, cap = 2500, [30000, 1200], 30016
    with B.Context() as own:
        own.L.ork_b200_set_stream(own.ctx, 1)
        c = Cache(2, 2, 64, cap)
        for s, n in enumerate(lens):
            c.put(s, rnd((n, 2, 64), 530 + s), rnd((n, 2, 64), 532 + s))
        attn4_check(own, c, rnd((2, T, 16, 64), 534, 1.5, torch.float16), lens, "f16")
        assert own.L.ork_b200_staging_bytes(own.ctx) < 6.5e9


def test_kv4_attn_fp32_sums_over_a_long_context_have_no_drift(on):
    # The logits' roundings, about 2^-20 of each weight, leave each output off by about 2^-20 A / sqrt(5000 tokens that
    # count) = 1.4e-8 A, A = sum p |v|, to either side: 6e-10 A in the mean of 512 outputs. What the products truncate would
    # all go one way; the mean may be off by 5e-9 A.
    from test_gpu_longctx import Cache, attn4

    n, H, Hkv, dk = 131000, 8, 2, 64
    c = Cache(1, Hkv, dk, 131008)
    bias = rnd((1, Hkv, dk), 540)
    c.put(0, rnd((n, Hkv, dk), 541, 1.1) + bias, rnd((n, Hkv, dk), 542))
    q = rnd((1, 1, H, dk), 543, 1.6)
    rc, out = attn4(on, c, q, [n], "f32")
    assert rc == 0 and on.L.ork_b200_sync(on.ctx) == 0
    k, v = c.get(0, n)
    want, size = ref.attention(q[0], k, v, dk ** -0.5, 0, 0)[0], ref.attention(q[0], k, v.abs(), dk ** -0.5, 0, 0)[0]
    off = float((out[0].double() - want).mean() / size.mean())
    assert abs(off) < 5e-9, off
