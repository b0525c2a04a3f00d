"""ops.chunk_attn where a row's weight lies in one key and very many others hold
a little each (an attention sink): what each of these adds may be small in fp16,
their sum counts.  Against the formula in fp64."""
import math
import sys

import pytest
import torch

from ragged import DEV, HND, NHD, Ragged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def sink(r, at, low, high):
    """Each sequence's key `at` scores 0 with a value of 0, the others `low` .. `high`
    (by turns) with values near 1."""
    x = r.hnd()
    for b in range(r.B):
        L, S = r.lens[b], r.S
        t = torch.linspace(low, high, 17, device=DEV)[torch.arange(r.P[b] * S, device=DEV) % 17]
        t[at] = 0.0
        v = 1.0 + 0.25 * torch.rand((r.P[b] * S, r.H, r.D), generator=r.g, device=DEV)
        v[at] = 0.0
        k = torch.zeros_like(v)
        k[..., 0] = (t * math.sqrt(r.D))[:, None]
        for which, y in ((0, k), (1, v)):
            y = y.half()
            y[L:] = float("nan")
            x[r.pages(b), which] = y.view(r.P[b], S, r.H, r.D).transpose(1, 2)
    r.q.zero_()
    r.q[..., 0] = 1.0
    return r


def check(r, rows, cap=0.0, **opts):
    """Rows `rows` of each sequence's chunk."""
    from aoakv import ops
    o, lse = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), return_lse=True, soft_cap=cap, **opts)
    for b in range(r.B):
        n, L = r.new[b], r.lens[b]
        k, v = r.cached(b, 0)[:, :, 0] / math.sqrt(r.D), r.cached(b, 1)
        k = cap * torch.tanh(k / cap) if cap else k
        for i in rows:
            i %= n
            see = slice(0, L - n + i + 1)
            e = torch.logsumexp(k[:, see], -1, keepdim=True)
            p = torch.exp(k[:, see] - e)
            x = (p[..., None] * v[:, see]).sum(1)[:, None]  # [H, 1, D], all of it positive
            # scores are one exact product each, their scale and the exponent a few
            # roundings in fp32, as the sums of L terms; a cap as in ragged.py
            off = (L + 64) * 2**-24 + cap * 2**-21
            # the result and probabilities are rounded to fp16, half a step each; the
            # smallest ones' step, 2^-24, is 2^-31 of the largest where that is held at
            # 2^7 or more
            tol = (2 * 2**-11 + off) * x + L * 2**-32 * v.abs().amax() + 2**-25
            got = o[r.q0[b] + i].view(r.H, r.G, r.D).double()
            bad = (got - x).abs() > tol
            assert not bad.any(), (b, i, got[bad][0].item(), x.expand_as(got)[bad][0].item(),
                                   tol.expand_as(got)[bad][0].item())
            got = lse[r.q0[b] + i].view(r.H, r.G).double()
            assert ((got - e).abs() <= off + 2**-21).all()


@pytest.mark.parametrize("low,high", [(-17.5, -17.5), (-17.6, -14.0), (-9.0, -8.0)])
@pytest.mark.parametrize("D,S,layout", [(64, 16, HND), (128, 16, NHD), (256, 16, HND),
                                        (128, 12, HND), (256, 5, NHD)])
def test_few_rows(D, S, layout, low, high):
    _say(f"[small] few rows D={D} S={S} {low} .. {high}")
    r = Ragged([16384, 40000, 333], [3, 1, 40], D, S, H=2, G=2, layout=layout, seed=D)
    check(sink(r, 0, low, high), (0, -1))


OPTS = [dict(), dict(cap=400.0), dict(slopes=True), dict(cap=400.0, slopes=True)]


def options(r, o):
    """(Slopes of 0, which change no score, run the kernels that have them.)"""
    return dict(o, slopes=torch.zeros(r.H * r.G, device=DEV)) if "slopes" in o else o


@pytest.mark.parametrize("opts", OPTS, ids=lambda o: "-".join(o) or "plain")
@pytest.mark.parametrize("D,S", [(64, 16), (128, 16), (256, 16), (128, 12)])
def test_listed(D, S, opts):
    """Rows for every workgroup that the GPU holds, and an item long enough to be cut."""
    _say(f"[small] listed D={D} S={S} {opts}")
    r = Ragged([40000, 1200], [100, 1200], D, S, H=32, G=2, seed=D)
    assert r.q.shape[0] * r.G // 128 * r.H >= 256 * (1 if D == 256 else 2)
    check(sink(r, 0, -17.5, -16.5), (0, 63, -1), **options(r, opts))


@pytest.mark.parametrize("opts", OPTS, ids=lambda o: "-".join(o) or "plain")
@pytest.mark.parametrize("D", [64, 128, 256])
def test_shares(D, opts):
    """Fewer rows, in equal shares of many tiles each."""
    _say(f"[small] shares D={D} {opts}")
    r = Ragged([16384, 16000], [3, 20], D, 16, H=32, G=1, seed=D)
    check(sink(r, 0, -17.5, -17.5), (0, -1), **options(r, opts))


@pytest.mark.parametrize("at", [70, 9000])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_sink_behind_the_others(D, at):
    """The running maximum starts from the small ones."""
    _say(f"[small] sink at {at} D={D}")
    r = Ragged([16384], [3], D, 16, H=64, G=1, seed=D)
    check(sink(r, at, -17.5, -17.5), (0, -1))
