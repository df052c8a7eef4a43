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
