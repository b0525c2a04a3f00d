"""Attention of ragged chunks over the paged cache (ops.chunk_attn) and the
weights their keys receive (ops.attn_weights) against the formulas in fp64.
The bounds are those of the kernels' roundings (ragged.py)."""
import sys

import pytest
import torch

from ragged import DEV, HND, I32, NEG, NHD, Ragged, i32, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def check(r, start=None, **opts):
    """Both operators on r with these options; returns o, lse, weights."""
    from aoakv import ops
    o = torch.full_like(r.q, 7.0)
    got, lse = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), o=o, return_lse=True, **opts)
    assert got.data_ptr() == o.data_ptr()
    ref_o, ref_lse, o_tol, lse_tol = r.attention(**opts)
    live = slice(r.q0[0], r.q0[-1])
    within(o[live], ref_o[live], o_tol[live])
    within(lse[live], ref_lse[live], lse_tol[live])
    assert (o[:r.q0[0]] == 7.0).all() and (o[r.q0[-1]:] == 7.0).all()  # rows of no sequence
    w = r.weights.clone()
    ops.attn_weights(r.q, lse, r.q_indptr, w, *r.tables(), start=start, **opts)
    ref_w, w_tol = r.sums(lse, start=start, **opts)
    within(w, ref_w, w_tol)
    return o, lse, w


# lengths of zero and one, chunks that start the sequence or end a long one,
# more rows than cached tokens, tile borders (64 keys, 128 rows) and one off them
LENS = [1, 17, 64, 65, 128, 300, 0, 777, 5, 200, 129, 33]
NEW = [1, 17, 1, 65, 127, 129, 0, 3, 0, 200, 128, 40]


@pytest.mark.parametrize("layout", [HND, NHD])
@pytest.mark.parametrize("D,S,H,G", [(128, 16, 4, 1), (128, 16, 2, 4), (64, 16, 3, 2),
                                     (256, 16, 2, 2), (128, 1, 2, 3), (64, 32, 1, 8),
                                     (128, 12, 2, 5), (256, 5, 1, 1), (128, 8, 1, 32)])
def test_shapes(D, S, H, G, layout):
    _say(f"[chunk] D={D} S={S} H={H} G={G} layout={layout}")
    check(Ragged(LENS, NEW, D, S, H, G, layout, seed=D + S + G))


@pytest.mark.parametrize("opts", [
    dict(causal=False), dict(window=1), dict(window=50), dict(window=64, causal=False),
    dict(prefix=4, window=20), dict(prefix=100), dict(prefix=1000, window=7),
    dict(soft_cap=5.0), dict(slopes=True), dict(soft_cap=30.0, slopes=True, window=90, prefix=3),
    dict(slopes=True, causal=False, prefix=9)], ids=lambda o: "-".join(o))
@pytest.mark.parametrize("D,G", [(128, 2), (64, 1), (256, 4)])
def test_masks_and_scores(opts, D, G):
    _say(f"[chunk] {opts} D={D} G={G}")
    r = Ragged(LENS, NEW, D, 16, 2, G, seed=3, scale=3.0)
    o = dict(opts)
    if o.pop("slopes", None):
        o["slopes"] = r.slopes()
    if "prefix" in o:
        o["prefix_len"] = i32(*[o["prefix"] if b % 3 else 0 for b in range(r.B)])
        del o["prefix"]
    check(r, **o)


@pytest.mark.parametrize("tokens", [1, 2, 5, 16, 31])
def test_few_tokens_after_long_contexts(tokens):
    """Few rows over many keys: the keys are split."""
    _say(f"[chunk] {tokens} after long contexts")
    r = Ragged([9001, 4096, 33, 2000, 12345], [tokens] * 5, H=2, G=4, seed=tokens)
    check(r)
    check(r, window=3000, prefix_len=i32(4, 0, 9, 5000, 4))


def test_one_long_sequence_beside_many_short_ones():
    _say("[chunk] one long, many short")
    check(Ragged([20000] + [40] * 300, [70] + [1] * 300, H=2, G=2, seed=8))


def test_many_sequences():
    """More sequences, and more tiles of rows, than a workgroup has threads."""
    _say("[chunk] many sequences")
    lens = [(37 * b) % 90 for b in range(1500)]
    check(Ragged(lens, [min(n, 1 + b % 5) for b, n in enumerate(lens)], D=64, H=1, G=2, seed=9))
    check(Ragged([300] * 3, [20, 300, 1], D=64, H=1, G=1, seed=9), slopes=None)


def test_a_long_prompt():
    _say("[chunk] 2500 tokens")
    check(Ragged([2500, 1300], [2500, 1300], H=2, G=2, seed=4))


def test_more_rows_than_cached_tokens():
    """Rows at positions below 0 see nothing (or the prefix): o 0, lse -inf."""
    _say("[chunk] more rows than tokens")
    r = Ragged([10, 0, 70], [30, 5, 200], H=2, G=2, seed=5)
    o, lse, _ = check(r)
    assert (o[r.q0[0]:r.q0[0] + 20] == 0).all() and (lse[r.q0[0]:r.q0[0] + 20] == NEG).all()
    assert (o[r.q0[1]:r.q0[2]] == 0).all() and (lse[r.q0[1]:r.q0[2]] == NEG).all()
    check(r, window=3)
    check(r, prefix_len=i32(4, 4, 4))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), NEG])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_unseen_values_change_nothing(D, value):
    """NaN and infinities in keys and values that a row does not see: behind it
    in its own chunk, before its window."""
    from aoakv import ops
    _say(f"[chunk] unseen {value} D={D}")
    r = Ragged([200, 90], [150, 3], D, H=2, G=2, seed=6)
    opts = dict(window=100)
    clean = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), return_lse=True, **opts)
    x = r.hnd()
    late = 180  # a token of sequence 0 that its rows before position 180 do not see
    page, slot = int(r.pages(0)[late // 16]), late % 16
    x[page, 1, :, slot, ::3] = value
    x[page, 0, :, slot, 1] = value
    dirty = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), return_lse=True, **opts)
    last = r.q0[0] + late - 50  # row of position 180
    for a, b in zip(clean, dirty):
        assert torch.equal(a[r.q0[0]:last], b[r.q0[0]:last])
        assert torch.equal(a[r.q0[1]:r.q0[2]], b[r.q0[1]:r.q0[2]])
        assert not b[last].isfinite().all()
    w = r.weights.clone()
    # (the sequence as it was when it ended before that token)
    ops.attn_weights(r.q[:last], dirty[1][:last], i32(r.q0[0], last), w, r.kv,
                     i32(r.ptr[0], r.ptr[0] + (late - 1) // 16 + 1), r.indices,
                     i32((late - 1) % 16 + 1), r.max_pages, r.layout, **opts)
    assert w.isfinite().all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_seen_infinities(D):
    """A value that a row does see reaches its own dims alone."""
    from aoakv import ops
    _say(f"[chunk] seen infinities D={D}")
    r = Ragged([300], [200], D, H=1, G=2, seed=16)
    x = r.hnd()
    places = ((120, 5, float("inf")), (250, 6, NEG), (260, 7, float("nan")), (30, 8, float("inf")),
              (40, 8, NEG))
    for j, d, value in places:
        x[int(r.pages(0)[j // 16]), 1, 0, j % 16, d] = value
    o = ops.chunk_attn(r.q, r.q_indptr, *r.tables())[r.q0[0]:r.q0[1]].float()
    pos = 100 + torch.arange(200, device=DEV)
    for d, kind in ((5, torch.isposinf), (6, torch.isneginf), (7, torch.isnan), (8, torch.isnan)):
        sees = pos >= max(j for j, dd, _ in places if dd == d)
        assert kind(o[sees][..., d]).all() and o[~sees][..., d].isfinite().all()
    rest = [d for d in range(D) if d not in (5, 6, 7, 8)]
    assert o[..., rest].isfinite().all()
    ref, _, tol, _ = r.attention()
    within(o[..., rest], ref[r.q0[0]:r.q0[1]][..., rest], tol[r.q0[0]:r.q0[1]][..., rest])


def test_large_scores():
    """Scores of hundreds, one key far above the others, and all equal."""
    _say("[chunk] large scores")
    r = Ragged([500, 300], [100, 300], H=2, seed=7, scale=60.0)
    check(r)
    r = Ragged([500, 300], [100, 300], H=2, seed=7, scale=0.0)
    check(r)
    check(r, slopes=r.slopes() * 50)


@pytest.mark.parametrize("start", [0, 40, 10000])
def test_weights_start(start):
    _say(f"[chunk] weights from {start}")
    r = Ragged([100, 333, 64], [10, 333, 0], H=2, G=3, seed=10)
    check(r, start=i32(start, 0, start))


def test_every_probability_is_counted_once():
    """The sums over a sequence's keys are its rows times the group's heads."""
    from aoakv import ops
    _say("[chunk] total weight")
    r = Ragged([1000, 400], [64, 400], H=3, G=4, seed=11)
    _, lse = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), return_lse=True)
    w = torch.zeros_like(r.weights)
    ops.attn_weights(r.q, lse, r.q_indptr, w, *r.tables(), start=i32(0, 0))
    for b in range(2):
        total = w[r.pages(b)].double().sum((0, 2))
        assert ((total - r.new[b] * 4).abs() <= r.new[b] * 4 * 1e-5).all()


def test_agrees_with_the_one_sequence_prefill():
    from aoakv import ops
    _say("[chunk] against prefill")
    r = Ragged([700], [130], H=2, G=4, seed=12, margin=0)
    a = ops.chunk_attn(r.q, r.q_indptr, *r.tables())
    b = ops.prefill_with_paged_kv_cache(r.q, r.kv, r.indices[3:], r.P[0], int(r.last[0]), r.layout)
    ref, _, tol, _ = r.attention()
    within(a, ref, tol)
    assert (a.double() - b.double()).abs().max() <= 2 * tol.max()


def test_equal_calls_give_equal_bits():
    from aoakv import ops
    _say("[chunk] equal bits")
    r = Ragged([9000, 700, 33], [60, 300, 33], H=4, G=2, seed=13)
    runs = []
    for _ in range(4):
        o, lse = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), o=torch.zeros_like(r.q),
                                return_lse=True)
        w = r.weights.clone()
        ops.attn_weights(r.q, lse, r.q_indptr, w, *r.tables())
        runs.append((o, lse[r.q0[0]:r.q0[-1]].clone(), w))
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)


def test_page_bound():
    """A table longer than max_pages is cut to it, and the error word says so."""
    from aoakv import ops
    _say("[chunk] page bound")
    r = Ragged([160, 40], [1, 2], H=2, seed=14)
    ws = ops.decode_workspace(1, 2, 2, 4)
    o = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), workspace=ws)
    assert ops.workspace_error(ws) == 0 and torch.isfinite(o[r.q0[0]:r.q0[-1]]).all()
    r.max_pages = 4
    got, lse = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), return_lse=True, workspace=ws)
    assert ops.workspace_error(ws) == ops.WS_ERR_TRUNCATED
    r.lens[0], r.ptr, r.P[0] = 64, [r.ptr[0], r.ptr[0] + 4, r.ptr[2]], 4
    short = Ragged.__new__(Ragged)
    short.__dict__.update(r.__dict__, B=1)
    ref, _, tol, _ = short.attention()
    rows = slice(r.q0[0], r.q0[1])
    within(got[rows], ref[rows], tol[rows])
    ops.workspace_init(ws)
    w = r.weights.clone()
    ops.attn_weights(r.q, lse, r.q_indptr, w, *r.tables(), workspace=ws)
    assert ops.workspace_error(ws) == ops.WS_ERR_TRUNCATED
    assert torch.equal(w[r.indices[3 + 4:3 + 10].long()], r.weights[r.indices[3 + 4:3 + 10].long()])


def test_no_rows():
    from aoakv import ops
    _say("[chunk] no rows")
    r = Ragged([50, 20], [0, 0], H=2, seed=15, margin=0)
    o, lse = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), return_lse=True)
    assert o.shape == (0, 2, 128) and lse.shape == (0, 2)
    w = r.weights.clone()
    ops.attn_weights(r.q, lse, r.q_indptr, w, *r.tables(), start=i32(0, 10))
    ref, tol = r.sums(lse, start=i32(0, 10))
    assert torch.equal(w.double(), ref)


def test_far_pages():
    """Pages whose elements lie past 2^32."""
    from aoakv import ops
    _say("[chunk] far pages")
    r = Ragged([100], [20], H=2, G=2, seed=17)
    per = r.kv[0].numel()
    far = (1 << 32) // per + 5
    kv = torch.zeros((far + r.total,) + r.kv.shape[1:], dtype=torch.float16, device=DEV)
    kv[far:] = r.kv
    w = torch.zeros((far + r.total,) + r.weights.shape[1:], device=DEV)
    near = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), return_lse=True)
    r.kv, r.indices = kv, r.indices + far
    got = ops.chunk_attn(r.q, r.q_indptr, *r.tables(), return_lse=True)
    live = slice(r.q0[0], r.q0[-1])
    assert torch.equal(near[0][live], got[0][live]) and torch.equal(near[1][live], got[1][live])
    ops.attn_weights(r.q, got[1], r.q_indptr, w, *r.tables(), start=i32(0))
    assert abs(float(w[far:].double().sum()) - 20 * 4) < 1e-3 and not w[:far].any()


def test_other_stream_and_graph():
    """On a stream of its own, and as two captured graphs that run in turn."""
    from aoakv import ops
    _say("[chunk] stream and graphs")
    r = Ragged([3000, 500], [33, 200], H=4, G=2, seed=18)
    s = Ragged([700, 5000], [64, 8], H=4, G=2, seed=19)

    def go(x, out):
        ops.chunk_attn(x.q, x.q_indptr, *x.tables(), o=out[0])
        o, lse = ops.chunk_attn(x.q, x.q_indptr, *x.tables(), return_lse=True)
        ops.attn_weights(x.q, lse, x.q_indptr, out[1], *x.tables(), start=i0)
    i0 = i32(0, 0)
    new = lambda x: (torch.zeros_like(x.q), x.weights.clone())
    eager = []
    for x in (r, s):
        eager.append(new(x))
        go(x, eager[-1])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        side = new(r)
        go(r, side)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(side, eager[0]))
    graphs, outs = [], []
    for x in (r, s):
        outs.append(new(x))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(x, outs[-1])
        graphs.append(g)
    for k in range(4):
        for out in outs:
            out[0].zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        extra = new(r)
        go(r, extra)
        for out, ref in zip(outs + [extra], eager + [eager[0]]):
            assert all(torch.equal(a, b) for a, b in zip(out, ref)), k
    # a replay takes what the tables say then: here a token less
    r.last.copy_(torch.clamp(r.last - 1, min=1))
    outs[0][1].copy_(r.weights)  # (slots behind the last token are not touched)
    graphs[0].replay()
    now = new(r)
    go(r, now)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], now))
