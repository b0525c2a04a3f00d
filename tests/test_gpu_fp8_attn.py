"""Attention over a paged cache held in 8 bits against 64 bits: chunks of a ragged batch
(ops.chunk_attn_fp8), and one token per sequence over every page or selected ones
(ops.decode_sparse_attn_fp8)."""
import math
import sys

import pytest
import torch

from codes import DEV, HND, I32, NEG, NHD, Coded, E4M3, i32, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


LENS = [300, 1, 0, 77, 64, 200, 16]
NEW = [5, 1, 0, 77, 1, 130, 0]


def chunk(r, **opts):
    from aoakv import ops
    o = torch.full_like(r.q, 3.0)
    return ops.chunk_attn_fp8(r.q, r.q_indptr, *r.table(), r.max_pages, r.layout, o=o,
                              return_lse=True, **opts)


def check_chunk(r, **opts):
    o, lse = chunk(r, **opts)
    ref, ref_lse, tol, lse_tol = r.attention(**opts)
    a = slice(r.q0[0], r.q0[-1])
    within(o[a], ref[a], tol[a])
    within(lse[a], ref_lse[a], lse_tol[a])
    for rest in (slice(0, r.q0[0]), slice(r.q0[-1], None)):
        assert torch.equal(o[rest], torch.full_like(o[rest], 3.0))
    return o, lse


@pytest.mark.parametrize("layout", [HND, NHD])
@pytest.mark.parametrize("D,S,H,G", [(128, 16, 2, 4), (128, 32, 3, 1), (128, 7, 2, 2),
                                     (128, 1, 1, 8), (64, 16, 2, 3), (64, 12, 2, 1),
                                     (256, 16, 2, 2), (256, 8, 1, 1)])
def test_chunks(D, S, H, G, layout):
    _say(f"[chunk fp8] {H} x {G} x {D}, pages of {S}, layout {layout}")
    check_chunk(Coded(LENS, NEW, D, S, H, G, layout, seed=D + S))


OPTIONS = [dict(causal=False), dict(window=20), dict(window=1), dict(window=64, prefix=4),
           dict(prefix=100), dict(soft_cap=5.0), dict(slopes=True),
           dict(slopes=True, soft_cap=30.0, window=50, prefix=3)]


@pytest.mark.parametrize("opts", OPTIONS, ids=str)
@pytest.mark.parametrize("D,S", [(128, 16), (64, 16), (256, 16), (128, 5), (256, 1)])
def test_options(D, S, opts):
    _say(f"[chunk fp8] head dim {D}, pages of {S}, {opts}")
    r = Coded(LENS, NEW, D, S, 2, 2, seed=3)
    o = dict(opts)
    if o.pop("slopes", None):
        o["slopes"] = r.slopes()
    if "prefix" in o:
        o["prefix_len"] = i32(*[min(n, o["prefix"]) if b % 2 else o["prefix"]
                                for b, n in enumerate(r.lens)])
        del o["prefix"]
    check_chunk(r, **o)


@pytest.mark.parametrize("D,S", [(128, 16), (64, 16), (256, 16), (128, 12), (256, 7)])
def test_listed_items(D, S):
    """Rows for more items than the GPU holds workgroups: the listed form."""
    _say(f"[chunk fp8] listed, head dim {D}, pages of {S}")
    H = 32
    n = 128 * (9 if D == 256 else 17)
    r = Coded([n, n // 2 + 3], [n, n // 2 - 70], D, S, H, 1, seed=4)
    check_chunk(r)


@pytest.mark.parametrize("D,S", [(128, 16), (256, 16), (64, 3)])
def test_long_contexts(D, S):
    """Items that several workgroups share; lengths that end inside of tiles and pages."""
    _say(f"[chunk fp8] long, head dim {D}, pages of {S}")
    check_chunk(Coded([9001, 130, 5000], [3, 130, 64], D, S, 2, 4, seed=6))


@pytest.mark.parametrize("D,S", [(128, 16), (64, 16), (256, 16), (128, 6), (256, 1)])
def test_unseen_values(D, S):
    """NaN codes where a row does not see them change nothing; where it does, they are
    what a product makes of them."""
    _say(f"[chunk fp8] NaN codes, head dim {D}, pages of {S}")
    r = Coded([150, 90], [40, 90], D, S, 2, 2, seed=7)
    clean, lse = check_chunk(r)
    for b, key in ((0, 131), (1, 50)):  # V alone: a dim of one key
        page, slot = int(r.pages(b)[key // S]), key % S
        v = r.bytes()
        v[page, 1, 1, slot, 5] = 0x7F
        v[page, 1, 0, slot, D - 1] = 0xFF
    o, lse2 = chunk(r)
    assert torch.equal(lse[r.q0[0]:r.q0[-1]], lse2[r.q0[0]:r.q0[-1]])
    want = clean.clone()
    for b, key in ((0, 131), (1, 50)):
        first = r.q0[b] + max(key - (r.lens[b] - r.new[b]), 0)
        want[first:r.q0[b + 1], 2:4, 5] = float("nan")
        want[first:r.q0[b + 1], 0:2, D - 1] = float("nan")
    a = slice(r.q0[0], r.q0[-1])
    assert torch.equal(o[a].isnan(), want[a].isnan())
    assert torch.equal(o[a].nan_to_num(0.0), want[a].nan_to_num(0.0))
    for b, key in ((0, 131), (1, 50)):  # and K: the rows that see the key
        r.bytes()[int(r.pages(b)[key // S]), 0, :, key % S, 1] = 0x7F
    o, lse = chunk(r)
    for b, key in ((0, 131), (1, 50)):
        first = r.q0[b] + max(key - (r.lens[b] - r.new[b]), 0)
        assert bool(o[first:r.q0[b + 1]].isnan().all()) and \
            bool(lse[first:r.q0[b + 1]].isnan().all())
        before = slice(r.q0[b], first)
        assert torch.equal(o[before], clean[before])


def test_equals_the_fp16_cache():
    """Over a cache of the same values in fp16 the result is the same but for the order of
    the sums."""
    from aoakv import ops
    _say("[chunk fp8] against an fp16 cache")
    r = Coded(LENS, NEW, 128, 16, 2, 4, seed=8)
    from codes import values
    kv = values(r.bytes(), r.exp).half().contiguous()
    o, lse = check_chunk(r)
    o2, lse2 = ops.chunk_attn(r.q, r.q_indptr, kv, r.indptr, r.indices, r.last, r.max_pages, HND,
                              return_lse=True)
    _, _, tol, lse_tol = r.attention()
    a = slice(r.q0[0], r.q0[-1])
    within(o[a], o2[a].double(), 2 * tol[a])
    within(lse[a], lse2[a].double(), 2 * lse_tol[a])


def test_chunk_calls():
    """Without a workspace, cut tables, a captured call, another stream: as documented."""
    from aoakv import ops
    _say("[chunk fp8] calls")
    r = Coded([700, 90], [4, 90], 128, 16, 2, 2, seed=9)
    o, lse = check_chunk(r)
    a = slice(r.q0[0], r.q0[-1])
    ws = ops.decode_workspace(2, 4, 2, 44, DEV)
    chunk(r, workspace=ws)
    assert ops.workspace_error(ws) == 0
    ops.chunk_attn_fp8(r.q, r.q_indptr, *r.table(), 10, r.layout, workspace=ws)
    assert ops.workspace_error(ws) == ops.WS_ERR_TRUNCATED
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        o2, lse2 = ops.chunk_attn_fp8(r.q, r.q_indptr, *r.table(), r.max_pages, r.layout,
                                      return_lse=True)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o2[a], o[a]) and torch.equal(lse2[a], lse[a])
        torch.randn(100, device=DEV).sum().item()


def test_chunk_without_workspace():
    """The C entry point with no workspace: items are not cut, the same values."""
    import ctypes

    from aoakv import _lib, ops
    _say("[chunk fp8] without a workspace")
    r = Coded([700, 90], [4, 90], 128, 16, 2, 2, seed=9)
    ref, ref_lse, tol, lse_tol = r.attention()
    o = torch.zeros_like(r.q)
    lse = torch.zeros(r.q.shape[:2], device=DEV)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    _lib.call("aoakv_chunk_attn_fp8", p(r.q), p(o), p(lse), p(r.q_indptr), r.q.shape[0], p(r.kv),
              p(r.exp), p(r.indptr), p(r.indices), p(r.last), None, None, 2, r.max_pages, 4, 2,
              128, 16, HND, 1, 0, 0.0, None, 0, None, ops._stream())
    a = slice(r.q0[0], r.q0[-1])
    within(o[a], ref[a], tol[a])
    within(lse[a], ref_lse[a], lse_tol[a])


# ------------------------------------------------------------------ one token
def decode(r, sel=None, budget=0, flags=0, budgets=None, max_pages=None, ws=None):
    from aoakv import ops
    q = r.q[:r.B].contiguous()
    o = torch.full_like(q, 3.0)
    if ws is None:
        ws = ops.decode_workspace(r.B, r.H * r.G, r.H, r.max_pages if sel is None else
                                  sel.shape[-1] + 1, DEV, head_dim=r.D)
    ops.decode_sparse_attn_fp8(q, o, *r.table(), sel, budget, ws, max_pages or r.max_pages,
                               r.layout, token_budgets=budgets, flags=flags)
    err = ops.workspace_error(ws)
    ops.workspace_init(ws[:256]) if err else None
    assert not ws.any(), "the workspace is left zeroed"
    return o, err


def expected(r, seen):
    """o and its bound; seen(b, h) -> the positions that count."""
    o = torch.zeros((r.B, r.H * r.G, r.D), dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(o)
    for b in range(r.B):
        if r.lens[b] == 0:
            continue
        k, v = r.cached(b, 0), r.cached(b, 1)
        for h in range(r.H):
            j = seen(b, h)
            q = r.q[b, h * r.G:(h + 1) * r.G].double()
            kk, vv = k[h, j], v[h, j]
            t = q @ kk.t() / math.sqrt(r.D)
            # products of fp16 are exact in fp32, sums of D terms round D times, the
            # exponent's factor and the exponential a few more
            off = (q.abs() @ kk.abs().t()).amax(-1, keepdim=True) / math.sqrt(r.D) * \
                (r.D + 8) * 2**-24 + 2**-21 * t.abs().amax(-1, keepdim=True)
            p = torch.softmax(t, -1)
            x, size = p @ vv, p @ vv.abs()
            a = slice(h * r.G, (h + 1) * r.G)
            o[b, a] = x
            # probabilities and the result are rounded to fp16 (half a step each, below
            # 2^-14 of the largest 2^-25 absolutely)
            tol[b, a] = 2**-11 * (x.abs() + size) + (off + len(j) * 2**-24) * size + \
                len(j) * 2**-25 * vv.abs().amax() + 2**-25
    return o, tol


def every(r):
    return lambda b, h: torch.arange(r.lens[b], device=DEV)


@pytest.mark.parametrize("layout", [HND, NHD])
@pytest.mark.parametrize("D,S,H,G", [(128, 16, 2, 1), (128, 16, 3, 8), (128, 32, 2, 4),
                                     (128, 7, 2, 2), (128, 1, 1, 4), (64, 16, 2, 4),
                                     (64, 12, 3, 1), (256, 16, 2, 2), (256, 3, 1, 8)])
def test_decode_every_page(D, S, H, G, layout):
    _say(f"[decode fp8] {H} x {G} x {D}, pages of {S}, layout {layout}")
    r = Coded([300, 1, 0, 77, 64, 2000, 16], [1] * 7, D, S, H, G, layout, seed=D + S + G)
    o, err = decode(r)
    ref, tol = expected(r, every(r))
    within(o, ref, tol)
    assert err == 0


def test_decode_many():
    """More sequences than a wave has lanes, with and without tokens."""
    _say("[decode fp8] 150 sequences")
    lens = [(37 * i) % 400 for i in range(150)]
    lens[77] = 9000
    r = Coded(lens, [1] * 150, 64, 16, 2, 2, seed=5)
    ref, tol = expected(r, every(r))
    within(decode(r)[0], ref, tol)
    none = Coded([0, 0, 0], [1] * 3, 64, 16, 2, 2, seed=5)
    assert not decode(none)[0].any()
    assert not decode(Coded([0], [1], 64, 16, 2, 2, seed=5))[0].any()


@pytest.mark.parametrize("n,L", [(65, 128), (100, 16), (200, 256), (64, 128)])
def test_decode_many_short(n, L):
    """Tables of a page or a few: the bound on their pages allows for no more chunks than
    sequences, and each has its own all the same."""
    _say(f"[decode fp8] {n} sequences of {L} tokens")
    r = Coded([L] * n, [1] * n, 64, 16, 2, 2, seed=6)
    ref, tol = expected(r, every(r))
    within(decode(r, max_pages=L // 16)[0], ref, tol)


@pytest.mark.parametrize("S,L", [(16, 70000), (1, 9000), (32, 40000)])
def test_decode_long(S, L):
    """Chunks of more pages than are staged at a time."""
    _say(f"[decode fp8] {L} tokens in pages of {S}")
    r = Coded([L, 30], [1, 1], 64, S, 64 if S == 16 else 128, 1, seed=2, sizes=False)
    o, _ = decode(r)
    for b in (0, 1):  # (a few heads: the reference is slow)
        k, v = r.cached(b, 0), r.cached(b, 1)
        for h in (0, r.H // 2, r.H - 1):
            q = r.q[b, h].double()
            t = k[h] @ q / 8.0
            p = torch.softmax(t, 0)
            off = (k[h].abs() @ q.abs()).max() / 8.0 * 72 * 2**-24 + 2**-21 * t.abs().max()
            x, size = p @ v[h], p @ v[h].abs()
            n = r.lens[b]
            within(o[b, h], x, 2**-11 * (x.abs() + size) + (off + n * 2**-24) * size +
                   n * 2**-25 * v[h].abs().max() * float(p.max()) + 2**-25)


def pick(r, budget, quest=False, seed=0):
    """A selection as the top-k leaves it: [B, H, n] physical ids in page order, and the
    positions that a head then attends."""
    g = torch.Generator().manual_seed(seed)
    rows, seen = [], {}
    n = max(3, budget // r.S) if not quest else max(1, budget // r.S - 1)
    sel = torch.full((r.B, r.H, n + 2), 0, **I32)
    for b in range(r.B):
        P, L = r.P[b], r.lens[b]
        if P == 0:
            continue
        k = min(max(1, budget // r.S), P) if quest else min(max(3, min(L, budget) // r.S), P)
        for h in range(r.H):
            if quest:
                ids = sorted(torch.randperm(P - 1, generator=g)[:k - 1].tolist())
            else:
                ids = sorted(torch.randperm(P, generator=g)[:k].tolist())
            if ids:
                sel[b, h, :len(ids)] = r.pages(b)[ids].int()
            pages = ids + ([P - 1] if quest else [])
            seen[b, h] = torch.tensor([p * r.S + s for p in pages for s in range(r.S)
                                       if p * r.S + s < L], device=DEV)
    return sel, lambda b, h: seen[b, h]


@pytest.mark.parametrize("quest", [False, True])
@pytest.mark.parametrize("D,S,H,G,budget", [(128, 16, 4, 1, 256), (128, 16, 2, 8, 512),
                                            (128, 32, 2, 2, 100), (64, 16, 3, 4, 2048),
                                            (256, 16, 2, 2, 320), (128, 5, 2, 2, 50),
                                            (128, 1, 2, 4, 200)])
def test_decode_selected(D, S, H, G, budget, quest):
    from aoakv import ops
    _say(f"[decode fp8] selected, {H} x {G} x {D}, pages of {S}, budget {budget}")
    r = Coded([3000, 1, 40, 0, 777, 65], [1] * 6, D, S, H, G, seed=D + S, layout=budget % 3 % 2)
    sel, seen = pick(r, budget, quest)
    o, err = decode(r, sel, budget, ops.FLAG_QUEST_KERNEL if quest else 0)
    ref, tol = expected(r, seen)
    within(o, ref, tol)
    assert err == 0


def test_decode_budgets():
    """A budget for each sequence."""
    _say("[decode fp8] budgets")
    r = Coded([3000, 500, 40], [1] * 3, 128, 16, 2, 2, seed=1)
    budgets = [64, 300, 1000]
    sel = torch.zeros((3, 2, 70), **I32)
    seen = {}
    for b, n in enumerate(budgets):
        s, f = pick(Coded([3000, 500, 40], [1] * 3, 128, 16, 2, 2, seed=1), n, seed=b)
        sel[b, :, :s.shape[2]] = s[b]
        for h in range(2):
            seen[b, h] = f(b, h)
    o, _ = decode(r, sel, 0, budgets=i32(*budgets))
    ref, tol = expected(r, lambda b, h: seen[b, h])
    within(o, ref, tol)


def test_decode_truncated():
    """A table longer than max_pages: its first pages, and the error bit."""
    from aoakv import ops
    _say("[decode fp8] a cut table")
    r = Coded([1000, 100], [1, 1], 128, 16, 2, 2, seed=3)
    o, err = decode(r, max_pages=20)
    assert err == ops.WS_ERR_TRUNCATED
    ref, tol = expected(r, lambda b, h: torch.arange(min(r.lens[b], 320), device=DEV))
    within(o, ref, tol)


@pytest.mark.parametrize("D,S", [(128, 16), (64, 5)])
def test_decode_nan_codes(D, S):
    """NaN codes in slots without a token change nothing (the batch has them there); in a
    token's they reach the heads that attend it."""
    _say("[decode fp8] NaN codes")
    r = Coded([75, 300], [1, 1], D, S, 2, 2, seed=3)
    clean, _ = decode(r)
    assert bool(clean.isfinite().all())
    r.bytes()[int(r.pages(1)[100 // S]), 1, 1, 100 % S, 7] = 0x7F
    o, _ = decode(r)
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[1, 2:, 7] = True
    assert torch.equal(o.isnan(), bad) and torch.equal(o[~bad], clean[~bad])


def test_decode_bounds_do_not_matter():
    """The page bound and the workspace's size do not change a bit; captured, on another
    stream, and twice at once with workspaces of their own neither."""
    from aoakv import ops
    _say("[decode fp8] calls")
    r = Coded([5000, 77, 0, 1200], [1] * 4, 128, 16, 4, 2, seed=8)
    first, _ = decode(r)
    ws = ops.decode_workspace(4, 8, 4, 4000, DEV)
    assert torch.equal(decode(r, max_pages=4000, ws=ws)[0], first)
    q = r.q[:4].contiguous()
    s = torch.cuda.Stream()
    graphs, outs, spaces = [], [], []
    for _ in range(2):
        w = ops.decode_workspace(4, 8, 4, r.max_pages, DEV)
        o = torch.zeros_like(q)
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.decode_sparse_attn_fp8(q, o, *r.table(), None, 0, w, r.max_pages, r.layout)
        graphs.append(g), outs.append(o), spaces.append(w)
    t = torch.cuda.Stream()
    for _ in range(3):
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(t):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, first) for o in outs)
        assert not any(w.any() for w in spaces)
        [o.zero_() for o in outs]


# ------------------------------------------------------------------ together
def test_a_batch_from_prompt_to_decode():
    """Rotation and append, attention of the prompts, decode steps over selected pages and
    over all: what the fp16 cache's calls give for the values that the codes hold."""
    from aoakv import ops
    _say("[fp8] a batch from prompt to decode")
    D, S, H, G, B, budget = 128, 16, 2, 4, 3, 256
    lens = [700, 33, 410]
    steps = 20
    P = [-(-(n + steps) // S) for n in lens]
    g = torch.Generator(device=DEV).manual_seed(0)
    ids = torch.randperm(sum(P), generator=g, device=DEV).int()
    own = [ids[sum(P[:b]):sum(P[:b + 1])] for b in range(B)]
    mids = torch.randperm(sum(-(-p // S) for p in P), generator=g, device=DEV).int()
    z = lambda *s: torch.zeros(s, dtype=torch.float16, device=DEV)  # noqa: E731
    kv = torch.zeros((sum(P), 2, H, S, D), dtype=torch.uint8, device=DEV).view(E4M3)
    exp = torch.zeros((sum(P), 2, H), dtype=torch.int8, device=DEV)
    meta, norm, mean = z(len(mids), 2, H, S, D), z(sum(P), H), z(sum(P), H, D)
    ws = ops.decode_workspace(B, H * G, H, max(P), DEV, max_pages=max(P))
    scores = torch.zeros((B, H, max(P)), device=DEV)
    sel = torch.zeros((B, H, max(P)), **I32)

    def table(now):
        n = [-(-x // S) for x in now]
        ip, mp = [0], [0]
        for x in n:
            ip.append(ip[-1] + x)
            mp.append(mp[-1] + -(-x // S))
        m = [sum(-(-p // S) for p in P[:b]) for b in range(B)]
        return (i32(*ip), torch.cat([own[b][:n[b]] for b in range(B)]),
                i32(*[(x - 1) % S + 1 for x in now]), i32(*mp),
                torch.cat([mids[m[b]:m[b] + -(-n[b] // S)] for b in range(B)]))

    for step in range(steps):
        new = lens if step == 0 else [1] * B
        now = [n + step for n in lens]
        T = sum(new)
        ip = [0]
        for n in new:
            ip.append(ip[-1] + n)
        q, k, v = (torch.randn((T, h, D), generator=g, device=DEV).half() for h in (H * G, H, H))
        kv_ip, kv_ix, last, m_ip, m_ix = table(now)
        t8 = (kv, exp, kv_ip, kv_ix, last)
        ops.rope_append_kv_cache_fp8(q, k, v, i32(*ip), *t8, HND, metadata_data=meta,
                                     metadata_indptr=m_ip, metadata_indices=m_ix, v_log_norm=norm,
                                     v_mean=mean)
        tn = [0]
        for n in now:
            tn.append(tn[-1] + n)
        K, V = ops.read_kv_cache_fp8(tn[-1], i32(*tn), *t8, HND)
        kv16 = z(*kv.shape)
        j = 0
        for b in range(B):  # the same values in an fp16 cache
            pos = torch.arange(now[b], device=DEV)
            kv16[own[b][pos // S].long(), 0, :, pos % S] = K[j:j + now[b]]
            kv16[own[b][pos // S].long(), 1, :, pos % S] = V[j:j + now[b]]
            j += now[b]
        t16 = (kv16, kv_ip, kv_ix, last)
        size = 2**-10 * 6 + 2**-12  # (|v| up to 6: two roundings of probabilities and results)
        a = ops.chunk_attn_fp8(q, i32(*ip), *t8, max(P), HND)
        within(a, ops.chunk_attn(q, i32(*ip), *t16, max(P), HND).double(),
               torch.full_like(a, size).double())
        if step == 0:
            continue
        o, o2, o3 = (torch.zeros_like(q) for _ in range(3))
        ops.decode_sparse_attn_fp8(q, o, *t8, None, 0, ws, max(P), HND)
        within(o, a.double(), torch.full_like(a, size).double())
        ops.estimate_topk(q, meta, m_ip, m_ix, kv_ip, kv_ix, last, norm, scores, sel, budget, ws,
                          max(P), HND)
        ops.decode_sparse_attn_fp8(q, o2, *t8, sel, budget, ws, max(P), HND)
        ops.decode_sparse_attn(q, o3, *t16, sel, budget, ws, max(P), H, HND)
        # (this call rounds scores to fp16: |t| below 8, 2^-9 twice, of a weight)
        within(o2, o3.double(), torch.full_like(a, size + 6 * 2**-7).double())
    assert ops.workspace_error(ws) == 0
