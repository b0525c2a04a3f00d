"""ops.chunk_attn where the rows fill the GPU several times over: its items are
listed by length then, the longest first, and long ones are cut.  And
ops.attn_weights of sequences with many rows each, which it cuts into larger
tiles.  Against the formulas in fp64, with the bounds of the kernels' roundings
(ragged.py)."""
import sys

import pytest
import torch

from ragged import DEV, HND, NEG, NHD, Ragged, i32, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def listed(r):
    """Whether r's rows make an item of 128 for each workgroup that the GPU holds."""
    assert r.q.shape[0] * r.G // 128 * r.H >= 256 * (1 if r.D == 256 else 2)
    return r


def check(r, **opts):
    from aoakv import ops
    o = torch.full_like(r.q, 7.0)
    _, lse = ops.chunk_attn(listed(r).q, r.q_indptr, *r.tables(), o=o, return_lse=True, **opts)
    ref_o, ref_lse, o_tol, lse_tol = r.attention(**opts)
    live = slice(r.q0[0], r.q0[-1])
    within(o[live], ref_o[live], o_tol[live])
    within(lse[live], ref_lse[live], lse_tol[live])
    assert (o[:r.q0[0]] == 7.0).all() and (o[r.q0[-1]:] == 7.0).all()  # rows of no sequence
    return o, lse


# one sequence of many keys (its items are cut), a prompt, short and empty ones,
# more rows than cached tokens, borders of rows and keys
LENS = [20000, 1, 0, 900, 64, 700, 10, 129, 65]
NEW = [150, 1, 0, 900, 64, 700, 30, 128, 65]


@pytest.mark.parametrize("D,S,H,G,layout", [
    (128, 16, 16, 2, HND), (128, 16, 16, 2, NHD), (64, 32, 16, 2, HND), (256, 16, 8, 2, HND),
    (128, 12, 11, 3, HND), (64, 1, 4, 8, NHD), (256, 5, 4, 5, NHD), (128, 16, 33, 1, HND)])
def test_shapes(D, S, H, G, layout):
    _say(f"[list] D={D} S={S} H={H} G={G} layout={layout}")
    check(Ragged(LENS, NEW, D, S, H, G, layout, seed=D + S + G, margin=12))


@pytest.mark.parametrize("opts", [
    dict(causal=False), dict(window=50), dict(window=64, causal=False), dict(prefix=100, window=20),
    dict(soft_cap=5.0), dict(slopes=True), dict(soft_cap=30.0, slopes=True, window=90, prefix=3),
    dict(slopes=True, causal=False, prefix=9)], ids=lambda o: "-".join(o))
@pytest.mark.parametrize("D,H,G", [(128, 8, 4), (64, 32, 1), (256, 8, 2)])
def test_masks_and_scores(opts, D, H, G):
    _say(f"[list] {opts} D={D} G={G}")
    r = Ragged(LENS, NEW, D, 16, H, G, seed=3, scale=3.0, margin=12)
    o = dict(opts)
    if o.pop("slopes", None):
        o["slopes"] = r.slopes()
    if "prefix" in o:
        o["prefix_len"] = i32(*[o["prefix"] if b % 3 else 0 for b in range(r.B)])
        del o["prefix"]
    check(r, **o)


@pytest.mark.parametrize("B", [255, 256, 257, 700])
def test_many_sequences(B):
    """As many sequences as a workgroup has threads, and more."""
    _say(f"[list] {B} sequences")
    lens = [(37 * b) % 90 for b in range(B)]
    lens[B // 2] = 6000
    check(Ragged(lens, [min(n, 9 + b % 5) for b, n in enumerate(lens)], D=64, H=32, G=2, seed=9))


def test_few_rows_of_a_padded_batch():
    """q of many rows, few of them a sequence's: these are listed, and cut."""
    _say("[list] padded")
    check(Ragged([9000, 300], [3, 300], H=8, G=4, seed=5, margin=1000))


def test_rows_that_see_nothing():
    _say("[list] empty rows")
    r = Ragged([10, 0, 70], [600, 700, 900], H=16, G=2, seed=5)
    o, lse = check(r)
    assert (o[r.q0[0]:r.q0[0] + 590] == 0).all() and (lse[r.q0[0]:r.q0[0] + 590] == NEG).all()
    assert (o[r.q0[1]:r.q0[2]] == 0).all() and (lse[r.q0[1]:r.q0[2]] == NEG).all()


@pytest.mark.parametrize("D,H,G", [(64, 16, 2), (128, 8, 4), (256, 8, 2)])
def test_infinities(D, H, G):
    """A value of inf or NaN reaches the rows and dims that see it alone."""
    from aoakv import ops
    _say(f"[list] infinities D={D}")
    n, L = 2200, 2300
    r = listed(Ragged([L, 40], [n, 40], D, H=H, G=G, seed=16))
    x = r.hnd()
    places = ((120, 5, float("inf")), (1250, 6, NEG), (2260, 7, float("nan")),
              (30, 8, float("inf")), (40, 8, NEG))
    for j, d, value in places:
        x[int(r.pages(0)[j // 16]), 1, :, j % 16, d] = value
    o = ops.chunk_attn(r.q, r.q_indptr, *r.tables())
    ref, _, tol, _ = r.attention()
    rest = [d for d in range(D) if d not in (5, 6, 7, 8)]
    live = slice(r.q0[0], r.q0[-1])
    within(o[live][..., rest], ref[live][..., rest], tol[live][..., rest])
    o = o[r.q0[0]:r.q0[1]].float()
    pos = L - n + torch.arange(n, device=DEV)
    for d, kind in ((5, torch.isposinf), (6, torch.isneginf), (7, torch.isnan), (8, torch.isnan)):
        sees = pos >= max(j for j, dd, _ in places if dd == d)
        assert kind(o[sees][..., d]).all() and o[~sees][..., d].isfinite().all()


def test_graph_and_equal_bits():
    """Equal calls, replays after the tables changed, and a call of few rows
    between them give the eager results to the bit."""
    from aoakv import ops
    _say("[list] graph")
    r = listed(Ragged(LENS, NEW, H=16, G=2, seed=18, margin=12))
    few = Ragged([500, 40], [3, 40], H=2, G=2, seed=19)
    run = lambda x: [t[x.q0[0]:x.q0[-1]].clone() for t in
                     ops.chunk_attn(x.q, x.q_indptr, *x.tables(), return_lse=True)]
    eager, eager_few = run(r), run(few)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(r), eager))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), return_lse=True)
    live = slice(r.q0[0], r.q0[-1])
    for k in range(4):
        o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(run(few), eager_few))
        assert torch.equal(o[live], eager[0]) and torch.equal(lse[live], eager[1]), k
    # what the tables say at the replay: a token less, and rows moved to another sequence
    r.last.copy_(torch.clamp(r.last - 1, min=1))
    r.q_indptr[4] += 64
    r.q_indptr[5] = r.q_indptr[4]
    now = run(r)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(o[live], now[0]) and torch.equal(lse[live], now[1])


@pytest.mark.parametrize("opts", [
    dict(), dict(causal=False), dict(window=300), dict(window=64, causal=False),
    dict(prefix=100, window=20), dict(soft_cap=5.0), dict(slopes=True),
    dict(soft_cap=30.0, slopes=True, window=190, prefix=3),
    dict(slopes=True, causal=False, prefix=9)], ids=lambda o: "-".join(o) or "plain")
@pytest.mark.parametrize("D,H,G,S", [(64, 2, 2, 16), (128, 2, 2, 16), (256, 1, 2, 16),
                                     (128, 2, 3, 5), (256, 2, 1, 1), (64, 1, 5, 12)])
def test_weights_of_many_rows(D, H, G, S, opts):
    from aoakv import ops
    _say(f"[weights] {opts} D={D} G={G} S={S}")
    r = Ragged([1500, 333, 640, 1000], [1500, 333, 64, 230], D, S, H, G, seed=D + G, scale=2.0)
    assert r.q.shape[0] * G >= 256 * r.B
    o = dict(opts)
    if o.pop("slopes", None):
        o["slopes"] = r.slopes()
    if "prefix" in o:
        o["prefix_len"] = i32(*[o["prefix"] if b % 3 else 0 for b in range(r.B)])
        del o["prefix"]
    _, lse = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), return_lse=True, **o)
    w = r.weights.clone()
    ops.attn_weights(r.q, lse, r.q_indptr, w, *r.tables(), **o)
    ref, tol = r.sums(lse, **o)
    within(w, ref, tol)
