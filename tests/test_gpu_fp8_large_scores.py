"""Attention over a cache held in 8 bits (decode, and of chunks, where an fp16 cache of the
same values goes through the same kernel) where scores are large (whole numbers, so exact in
fp32): a key's weight is that of its score to the roundings of probabilities, whether the
running maximum moved after it and wherever its part was joined.  An offset rounded apart
from the one that exponentials were taken with would weigh parts by up to a step of the
scaled scores, 2^-5 here."""
import math
import sys

import pytest
import torch

from codes import DEV, HND, Coded, values, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def batch(D, S, H, G, L, heads, steps, values=None):
    """Token j's keys are (2^15, 2^8, steps[j]) and zeros, the queries' first four dims
    ``heads(h)``; steps [L, 2]."""
    r = Coded([L], [1], D, S, H, G, seed=D + S + G, margin=0, sizes=False)
    x = r.hnd().double()
    empty = x[:, 0].isnan()
    x[:, 0] = 0.0
    x[:, 0, :, :, 0], x[:, 0, :, :, 1] = 2.0 ** 15, 2.0 ** 8
    page, j = r.pages(0), torch.arange(L, device=DEV)
    x[page[j // S], 0, :, j % S, 2:4] = steps.double()[:, None].expand(L, H, 2)
    if values is not None:
        x[page[j // S], 1, :, j % S, :] = values[:, None, None].expand(L, H, D)
    x[:, 0][empty] = float("nan")
    r.code(x)
    r.q.zero_()
    for h in range(H * G):
        r.q[:, h, :4] = torch.tensor(heads(h), dtype=torch.float64, device=DEV).half()
    return r


def decode(r):
    from aoakv import ops
    q = r.q[:1].contiguous()
    o = torch.zeros_like(q)
    ws = ops.decode_workspace(1, r.H * r.G, r.H, r.max_pages, DEV, head_dim=r.D)
    ops.decode_sparse_attn_fp8(q, o, *r.table(), None, 0, ws, r.max_pages, r.layout)
    return o


def chunk(r):
    from aoakv import ops
    return ops.chunk_attn_fp8(r.q, r.q_indptr, *r.table(), r.max_pages, r.layout)


def chunk_fp16(r):
    from aoakv import ops
    kv = values(r.bytes(), r.exp).half().contiguous()
    return ops.chunk_attn(r.q, r.q_indptr, kv, r.indptr, r.indices, r.last, r.max_pages, HND)


def check(r, call):
    """One token's attention against fp64.  Probabilities and the result are rounded to fp16
    (half a step, 2^-11, each), an exponent below 64 and the exponential are off by 2^-19 at
    most, sums of L terms by L 2^-24; scores are exact."""
    q, o, L = r.q[:1], call(r), r.lens[0]
    K, V = r.cached(0, 0), r.cached(0, 1)
    for h in range(r.H):
        k, v = K[h], V[h]
        a = slice(h * r.G, (h + 1) * r.G)
        t = q[0, a].double() @ k.t()
        assert bool((t == t.round()).all()) and float(t.abs().max()) < 2 ** 24
        p = torch.softmax(t / math.sqrt(r.D), -1)
        x, size = p @ v, p @ v.abs()
        tol = 2**-11 * (x.abs() + size) + (2**-19 + L * 2**-24) * size + \
            L * 2**-25 * v.abs().amax() * p.amax() + 2**-25
        within(o[0, a], x, tol)


@pytest.mark.parametrize("D,S,H,G,L", [(128, 16, 2, 4, 3000), (128, 7, 2, 8, 3000),
                                       (64, 16, 4, 1, 9000), (256, 16, 2, 2, 3000),
                                       (128, 16, 2, 4, 700)])
@pytest.mark.parametrize("call", [decode, chunk, chunk_fp16])
def test_near_equal_maxima(call, D, S, H, G, L):
    """A key in 97 scores 1024 more than the others, and up to 14 more than each other, just
    past 2^18 in scaled units, where the step of fp32 doubles."""
    _say(f"[large scores fp8] {call.__name__}, {H} x {G} x {D}, pages of {S}, {L} tokens")
    i = torch.arange(L, device=DEV)
    top = (i % 97 == 5).double()
    border = math.log(2) * math.sqrt(D) * 2 ** 18

    def heads(h):
        left = border - 1024 + 4 * (h % 3)
        first = left // 2 ** 15
        return first, math.ceil((left - first * 2 ** 15) / 2 ** 8 * 16) / 16, 4.0, 8.0

    check(batch(D, S, H, G, L, heads, torch.stack([256 * top, 0.25 * top * (i // 97 * 5 % 8)], 1)),
          call)


@pytest.mark.parametrize("D,S,L,step", [(128, 16, 4096, 4.0), (64, 16, 4096, 3.0),
                                        (256, 16, 2048, 6.0), (128, 5, 2055, 4.0)])
@pytest.mark.parametrize("call", [decode, chunk, chunk_fp16])
def test_a_maximum_that_moves(call, D, S, L, step):
    """Eight of the last keys have some 2^8 times the weight of each other one: what was summed
    before them is as much as they are."""
    _say(f"[large scores fp8] a maximum that moves, {call.__name__}, head dim {D}, {L} tokens")
    j = torch.arange(L, device=DEV)
    few = ((j >= L - 256) & (j % 32 == 11)).double()
    check(batch(D, S, 256, 1, L, lambda h: (63.0 - h % 32, 1.0 + h % 7, 16.0, 0.0),
                torch.stack([step * few, 0 * few], 1), 1 - 2 * few), call)
