"""ops.chunk_attn_fp8 where the rows fill the GPU several times over: its items are listed by
length then, the longest first, and long ones are cut.  With caps, slopes and masks, odd
pages, and NaN codes, against the formulas in fp64 (codes.py, ragged.py)."""
import sys

import pytest
import torch

from codes import DEV, HND, NHD, Coded, i32, within

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


def run(r, **opts):
    from aoakv import ops
    o = torch.full_like(r.q, 7.0)
    return ops.chunk_attn_fp8(listed(r).q, r.q_indptr, *r.table(), r.max_pages, r.layout, o=o,
                              return_lse=True, **opts)


def check(r, **opts):
    o, lse = run(r, **opts)
    ref_o, ref_lse, o_tol, lse_tol = r.attention(**opts)
    live = slice(r.q0[0], r.q0[-1])
    within(o[live], ref_o[live], o_tol[live])
    within(lse[live], ref_lse[live], lse_tol[live])
    assert (o[:r.q0[0]] == 7.0).all() and (o[r.q0[-1]:] == 7.0).all()  # rows of no sequence
    return o, lse


# one sequence of many keys (its items are cut), a prompt, short and empty ones, more rows
# than cached tokens, borders of rows and keys
LENS = [9000, 1, 0, 900, 64, 700, 10, 129, 65]
NEW = [150, 1, 0, 900, 64, 700, 30, 128, 65]


@pytest.mark.parametrize("D,S,H,G,layout", [
    (128, 16, 16, 2, NHD), (64, 32, 16, 4, HND), (256, 16, 8, 2, HND), (128, 12, 11, 3, HND),
    (64, 1, 8, 8, NHD), (256, 5, 4, 5, NHD), (128, 16, 33, 1, HND)])
def test_shapes(D, S, H, G, layout):
    _say(f"[list fp8] D={D} S={S} H={H} G={G} layout={layout}")
    check(Coded(LENS, NEW, D, S, H, G, layout, seed=D + S + G, margin=12))


@pytest.mark.parametrize("opts", [
    dict(causal=False), dict(window=50), dict(prefix=100, window=20), dict(soft_cap=5.0),
    dict(slopes=True), dict(soft_cap=30.0, slopes=True, window=90, prefix=3),
    dict(slopes=True, causal=False, prefix=9)], ids=lambda o: "-".join(o))
@pytest.mark.parametrize("D,S,H,G", [(128, 16, 8, 4), (64, 16, 32, 2), (256, 16, 8, 2),
                                     (128, 7, 8, 4), (64, 12, 32, 2), (256, 5, 8, 2)])
def test_masks_and_scores(opts, D, S, H, G):
    _say(f"[list fp8] {opts} D={D} S={S} G={G}")
    r = Coded(LENS, NEW, D, S, H, G, seed=3, margin=12)
    o = dict(opts)
    if o.pop("slopes", None):
        o["slopes"] = r.slopes()
    if "prefix" in o:
        o["prefix_len"] = i32(*[o["prefix"] if b % 3 else 0 for b in range(r.B)])
        del o["prefix"]
    check(r, **o)


@pytest.mark.parametrize("score", ["plain", "cap", "slopes"])
@pytest.mark.parametrize("D,S,H,G", [(128, 16, 8, 4), (64, 16, 16, 4), (256, 16, 8, 2),
                                     (128, 6, 8, 4), (256, 1, 8, 2)])
def test_unseen_values(D, S, H, G, score):
    """A NaN code of V reaches the rows and the dim that see it and changes no other bit; of K
    the rows that see it."""
    _say(f"[list fp8] NaN codes D={D} S={S} {score}")
    n, L = 2200, 2300
    r = Coded([L, 40], [n, 40], D, S, H, G, seed=16)
    opts = dict(cap=dict(soft_cap=20.0), slopes=dict(slopes=r.slopes())).get(score, {})
    clean, lse = check(r, **opts)
    pos = L - n + torch.arange(n, device=DEV)
    rows = slice(r.q0[0], r.q0[1])
    want = clean.clone()
    for j, h, d in ((120, 0, 5), (1250, 1, D - 1), (2260, H - 1, 7)):
        r.bytes()[int(r.pages(0)[j // S]), 1, h, j % S, d] = 0xFF if d == 7 else 0x7F
        first = r.q0[0] + max(j - (L - n), 0)
        want[first:r.q0[1], h * G:(h + 1) * G, d] = float("nan")
    o, lse2 = run(r, **opts)
    a = slice(r.q0[0], r.q0[-1])
    assert torch.equal(lse[a], lse2[a])
    assert torch.equal(o[a].isnan(), want[a].isnan())
    assert torch.equal(o[a].nan_to_num(0.0), want[a].nan_to_num(0.0))
    r.bytes()[int(r.pages(0)[700 // S]), 0, 2, 700 % S, 1] = 0x7F
    o, lse3 = run(r, **opts)
    heads = slice(2 * G, 3 * G)
    sees = pos >= 700
    assert bool(o[rows][sees][:, heads].isnan().all()) and \
        bool(lse3[rows][sees][:, heads].isnan().all())
    assert torch.equal(o[rows][~sees][:, heads], clean[rows][~sees][:, heads])
    assert torch.equal(lse3[rows][~sees], lse[rows][~sees])
