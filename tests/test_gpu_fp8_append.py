"""New tokens into a paged cache held in 8 bits (ops.append_kv_cache_fp8,
rope_append_kv_cache_fp8) and tokens back (ops.read_kv_cache_fp8): codes, exponents and
page statistics bit for bit, angles against 64 bits."""
import sys

import pytest
import torch

from codes import (DEV, E4M3, HND, I32, NHD, Coded, code_of, exponent, finite_top, held, i32,
                   values, within)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


LENS = [40, 1, 0, 100, 17, 64, 33, 300]
NEW = [40, 1, 0, 3, 1, 16, 20, 129]


def rows(r, seed=7, special=None):
    """k, v for the rows of r.q (NaN in those of no sequence), heads of different size."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    T = r.q.shape[0]
    x = torch.randn((2, T, r.H, r.D), generator=g, device=DEV).half()
    x *= torch.exp2(torch.randint(-12, 5, (2, T, r.H, 1), generator=g, device=DEV)).half()
    if special is not None:
        special(x)
    x[:, :r.q0[0]] = float("nan")
    x[:, r.q0[-1]:] = float("nan")
    return x[0].contiguous(), x[1].contiguous()


def expected(r, k, v):
    """The cache's bytes [pages, 2, H, S, D] and exponents after the append."""
    c, e = r.bytes().clone(), r.exp.to(torch.int32)
    for b in range(r.B):
        n, L = r.new[b], r.lens[b]
        for p in range((L - n) // r.S, r.P[b]) if n else []:
            page = int(r.pages(b)[p])
            e0 = max(L - n - p * r.S, 0)
            e1 = min(L - p * r.S, r.S)
            row = r.q0[b] + p * r.S + e0 - (L - n)
            for which, x in ((0, k), (1, v)):
                y = x[row:row + e1 - e0].transpose(0, 1).double()
                new = exponent(finite_top(y, (1, 2)))
                if e0:
                    old = values(c[page:page + 1], e[page:page + 1])[0, which, :, :e0]
                    new = torch.maximum(new, e[page, which])
                    y = torch.cat([old, y], 1)
                y = held(y, new[:, None, None])
                c[page, which, :, :e1] = code_of(y[None, None], new[None, None])[0, 0]
                e[page, which] = new
    return c, e.to(torch.int8)


def append(r, k, v, **stats):
    from aoakv import ops
    ops.append_kv_cache_fp8(k, v, r.q_indptr, *r.table(), r.layout, **stats)


def check(r, k, v):
    # (codes that the cache holds at first reach all patterns where no token is)
    c, e = expected(r, k, v)
    append(r, k, v)
    assert torch.equal(r.exp, e)
    got = r.bytes()
    nan = ((got & 0x7F) == 0x7F) & ((c & 0x7F) == 0x7F)  # (a NaN's sign is nobody's)
    bad = (got != c) & ~nan
    n = int(bad.sum())
    assert n == 0, (n, bad.nonzero()[:4].tolist(), got[bad][:8].tolist(), c[bad][:8].tolist())


@pytest.mark.parametrize("layout", [HND, NHD])
@pytest.mark.parametrize("D,S,H", [(128, 16, 4), (128, 16, 17), (64, 16, 3), (256, 16, 9),
                                   (128, 1, 2), (64, 7, 5), (128, 32, 3), (256, 32, 2),
                                   (128, 12, 4)])
def test_codes(D, S, H, layout):
    _say(f"[append fp8] {H} x {D}, pages of {S}, layout {layout}")
    r = Coded(LENS, NEW, D, S, H, layout=layout, seed=D + S, spare=2)
    check(r, *rows(r))


def test_many_sequences():
    """More sequences than a wave has lanes; none, one and several tokens each."""
    _say("[append fp8] 200 sequences")
    lens = [(7 * i) % 50 for i in range(200)]
    new = [min(n, (3 * i) % 5) for i, n in enumerate(lens)]
    r = Coded(lens, new, 64, 16, 2, seed=3)
    check(r, *rows(r))


def test_values_at_the_ends():
    """Zeros, the smallest and largest numbers, 448 times a power of two and its
    neighbours, infinities and NaN."""
    _say("[append fp8] values at the ends")
    table = torch.tensor([0.0, -0.0, 2.0 ** -24, -3 * 2.0 ** -24, 2.0 ** -14, 65504.0, -65504.0,
                          61440.0, 63488.0, 57344.0, 57376.0, 448.0, 448.5, 7.0, 7.004, 1.0, 464.0,
                          float("inf"), float("-inf"), float("nan")], device=DEV).half()

    def special(x):
        g = torch.Generator(device=DEV).manual_seed(5)
        for t in range(x.shape[1]):  # (the rows from a few values each)
            few = torch.randint(0, len(table), (3,), generator=g, device=DEV)
            pick = torch.randint(0, 3, x[:, t].shape, generator=g, device=DEV)
            x[:, t] = table[few[pick]]

    r = Coded([64, 33, 90], [64, 20, 70], 128, 16, 3, seed=4)
    check(r, *rows(r, special=special))
    r = Coded([64, 33], [64, 20], 64, 1, 3, seed=4)
    check(r, *rows(r, special=special))
    zero = Coded([40], [40], 128, 16, 2, seed=5)
    z = torch.zeros((zero.q.shape[0], 2, 128), dtype=torch.float16, device=DEV)
    check(zero, z, z)
    assert int(zero.exp[zero.pages(0)].max()) == -15


def test_token_by_token():
    """A page that grows a token at a time: the exponent only grows, the older codes move
    with it, and at the end they are those of the page appended at once, but for values
    that were subnormal on the way."""
    _say("[append fp8] token by token")
    D, S, H, n = 128, 16, 3, 37
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((2, n, H, D), generator=g, device=DEV)
    x *= torch.exp2(torch.linspace(-6, 6, n, device=DEV))[None, :, None, None]  # (growing)
    x = x.half()
    one = Coded([n], [n], D, S, H, seed=2, margin=0)
    step = Coded([n], [n], D, S, H, seed=2, margin=0)
    append(one, x[0].contiguous(), x[1].contiguous())
    for i in range(n):
        r = Coded([i + 1], [1], D, S, H, seed=2, margin=0)
        r.kv, r.exp, r.indices, r.indptr = step.kv, step.exp, step.indices, step.indptr.clone()
        r.indptr[1] = r.indptr[0] + i // S + 1
        r.ptr = r.indptr.tolist()
        check(r, x[0, i:i + 1].contiguous(), x[1, i:i + 1].contiguous())
    assert torch.equal(one.exp, step.exp)
    for which in (0, 1):
        a, b = one.cached(0, which), step.cached(0, which)
        normal = a.abs() >= 448 * 2.0 ** -13 * finite_top(a, (1, 2)).view(H, 1, 1)
        assert torch.equal(a[normal], b[normal])
        within(b, a, 2.0 ** -4 * a.abs() + 2.0 ** -17 * finite_top(a, (1, 2)).view(H, 1, 1))


@pytest.mark.parametrize("layout", [HND, NHD])
@pytest.mark.parametrize("D,S,H", [(128, 16, 4), (64, 16, 3), (256, 16, 9), (128, 7, 2),
                                   (64, 32, 5), (128, 1, 3)])
def test_statistics(D, S, H, layout):
    """The page statistics are those of an fp16 cache's append, bit for bit."""
    from aoakv import ops
    _say(f"[append fp8] statistics {H} x {D}, pages of {S}, layout {layout}")
    lens, new = [40, 1, 100, 17, 64, 33, 300], [40, 1, 3, 1, 16, 20, 129]
    r = Coded(lens, new, D, S, H, layout=layout, seed=9)
    k, v = rows(r)
    P, M = r.kv.shape[0], [-(-p // S) for p in r.P]
    md = torch.randperm(sum(M), generator=r.g, device=DEV).int()
    at = [0]
    for m in M:
        at.append(at[-1] + m)
    shape = (sum(M), 2, H, S, D) if layout == HND else (sum(M), 2, S, H, D)

    def state():
        g = torch.Generator(device=DEV).manual_seed(11)
        f = lambda *s: torch.randn(s, generator=g, device=DEV).half()  # noqa: E731
        return f(*shape), f(P, H), f(P, H, D)

    meta, norm, mean = state()
    append(r, k, v, metadata_data=meta, metadata_indptr=i32(*at), metadata_indices=md,
           v_log_norm=norm, v_mean=mean)
    meta2, norm2, mean2 = state()
    kv16 = torch.zeros(r.kv.shape, dtype=torch.float16, device=DEV)
    for b in range(r.B):
        a = slice(r.q0[b], r.q0[b + 1])
        ops.append_kv_cache_prefill(k[a], v[a], kv16, r.indices[r.ptr[b]:r.ptr[b + 1]], r.P[b],
                                    (lens[b] - 1) % S + 1, meta2, md[at[b]:at[b + 1]], norm2,
                                    mean2, layout)
    for x, y in ((meta, meta2), (norm, norm2), (mean, mean2)):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


def turned(x, pos, theta, scale):
    """Rows [n, H, D] turned in fp64, and how far fp32 with the sine and cosine
    instructions (1.3e-7) of an angle good to 2^-26 of a turn may be off."""
    D = x.shape[-1]
    f = theta ** (-2.0 * torch.arange(D // 2, dtype=torch.float64, device=DEV) / D) / scale
    a = pos.double()[:, None, None] * f
    u, w = x[..., :D // 2].double(), x[..., D // 2:].double()
    y = torch.cat([u * a.cos() - w * a.sin(), w * a.cos() + u * a.sin()], -1)
    size = u.abs() + w.abs()
    return y, torch.cat([size, size], -1) * 2.0 ** -21


@pytest.mark.parametrize("D,S,theta,scale", [(128, 16, 1e4, 1.0), (64, 16, 1e6, 4.0),
                                             (256, 7, 1e4, 8.0), (128, 1, 5e5, 0.5)])
def test_rotation(D, S, theta, scale):
    _say(f"[rope append fp8] head dim {D}, pages of {S}")
    from aoakv import ops
    H, G = 3, 2
    r = Coded([900, 5, 0, 333], [700, 1, 0, 40], D, S, H, G=G, seed=12)
    g = torch.Generator(device=DEV).manual_seed(3)
    k, v, q = (torch.randn((r.q.shape[0], h, D), generator=g, device=DEV).half()
               for h in (H, H, H * G))
    k0, q0 = k.clone(), q.clone()
    before = r.bytes().clone()
    ops.rope_append_kv_cache_fp8(q, k, v, r.q_indptr, *r.table(), r.layout, rope_scale=scale,
                                 rope_theta=theta)
    assert torch.equal(k, k0)
    for a in (slice(0, r.q0[0]), slice(r.q0[-1], None)):
        assert torch.equal(q[a], q0[a])
    seen = torch.zeros(r.kv.shape[0], dtype=torch.bool, device=DEV)
    for b in range(r.B):
        n, L = r.new[b], r.lens[b]
        if n == 0:
            continue
        a, pos = slice(r.q0[b], r.q0[b + 1]), torch.arange(L - n, L, device=DEV)
        y, off = turned(q0[a], pos, theta, scale)
        within(q[a], y, off + 2.0 ** -11 * y.abs() + 2.0 ** -25)
        y, off = turned(k0[a], pos, theta, scale)
        off = off + 2.0 ** -11 * y.abs() + 2.0 ** -25          # the fp16 row
        e = r.exp[r.pages(b)][:, 0].double().repeat_interleave(S, 0)[L - n:L][..., None]
        got = r.cached(b, 0)[:, L - n:].transpose(0, 1)
        within(got, y, off + torch.maximum(2.0 ** -4 * (y.abs() + off), 2.0 ** (e - 10)))
        seen[r.pages(b)[(L - n) // S:]] = True
    assert torch.equal(r.bytes()[~seen], before[~seen])


def test_far_positions():
    """Positions of 2^21 and more (a table that names a page over and over): angles as
    exact as near ones."""
    _say("[rope append fp8] far positions")
    from aoakv import ops
    D, H, n = 128, 2, 9
    for first in (0, 2 ** 21 + 12345, 2 ** 25 - 40):
        S = 1 if first == 0 else 32
        L = first + n
        P = -(-L // S)
        own = min(P, -(-n // S) + 1)
        idx = torch.zeros(P, **I32)
        idx[-own:] = torch.arange(1, own + 1, **I32)
        g = torch.Generator(device=DEV).manual_seed(1)
        k, v, q = (torch.randn((n, H, D), generator=g, device=DEV).half() for _ in range(3))
        q0 = q.clone()
        kv = torch.zeros((own + 2, 2, H, S, D), dtype=torch.uint8, device=DEV).view(E4M3)
        exp = torch.zeros((own + 2, 2, H), dtype=torch.int8, device=DEV)
        ops.rope_append_kv_cache_fp8(q, k, v, i32(0, n), kv, exp, i32(0, P), idx,
                                     i32((L - 1) % S + 1), HND)
        y, off = turned(q0, torch.arange(first, L, device=DEV), 1e4, 1.0)
        within(q, y, off + 2.0 ** -11 * y.abs() + 2.0 ** -25)


@pytest.mark.parametrize("layout", [HND, NHD])
@pytest.mark.parametrize("D,S,H", [(128, 16, 4), (64, 7, 17), (256, 32, 5), (128, 1, 2)])
def test_read(D, S, H, layout):
    """The rows hold the codes' exact values; rows of no token are not written."""
    from aoakv import ops
    _say(f"[read fp8] {H} x {D}, pages of {S}")
    r = Coded(LENS, NEW, D, S, H, layout=layout, seed=5)
    k, v = (torch.full((r.q.shape[0], H, D), 7.0, dtype=torch.float16, device=DEV)
            for _ in range(2))
    got = ops.read_kv_cache_fp8(k.shape[0], r.q_indptr, *r.table(), layout, k=k, v=v)
    assert got[0] is k and got[1] is v or torch.equal(got[0], k)
    for which, x in ((0, k), (1, v)):
        ref = torch.full_like(x, 7.0).double()
        for b in range(r.B):
            ref[r.q0[b]:r.q0[b + 1]] = r.cached(b, which)[:, r.lens[b] - r.new[b]:].transpose(0, 1)
        assert torch.equal(x.double().nan_to_num(0, 0, 0), ref.nan_to_num(0, 0, 0))
        assert torch.equal(x.isnan(), ref.isnan())
    k2, v2 = ops.read_kv_cache_fp8(k.shape[0], r.q_indptr, *r.table(), layout)
    a = slice(r.q0[0], r.q0[-1])
    assert torch.equal(k2[a].view(torch.int16), k[a].view(torch.int16))
    assert torch.equal(v2[a].view(torch.int16), v[a].view(torch.int16))


def test_more_rows_than_tokens():
    """A chunk of more rows than the sequence holds: the rows before its first token are
    dropped (and read back as they were)."""
    _say("[append fp8] more rows than tokens")
    from aoakv import ops
    D, S, H = 64, 16, 2
    r = Coded([20, 3], [20, 3], D, S, H, seed=6, margin=0)
    k, v = rows(r)
    check(r, k, v)
    want = r.bytes().clone(), r.exp.clone()
    pad = torch.full((5, H, D), float("nan"), dtype=torch.float16, device=DEV)
    wide = Coded([20, 3], [20, 3], D, S, H, seed=6, margin=0)
    ops.append_kv_cache_fp8(torch.cat([pad, k]), torch.cat([pad, v]), i32(0, 25, 28),
                            *wide.table(), HND)
    assert torch.equal(wide.bytes(), want[0]) and torch.equal(wide.exp, want[1])
    out = torch.full((28, H, D), 3.0, dtype=torch.float16, device=DEV)
    ops.read_kv_cache_fp8(28, i32(0, 25, 28), *wide.table(), HND, k=out, v=out.clone())
    assert torch.equal(out[:5], torch.full_like(out[:5], 3.0))


def test_graph_and_streams():
    """Captured and replayed, on another stream than torch's default: the same bits."""
    from aoakv import ops
    _say("[append fp8] graph")
    a, b = (Coded([300, 17], [40, 1], 128, 16, 4, G=2, seed=8) for _ in range(2))
    k, v = rows(a)
    q = a.q.clone()
    qa, qb = q.clone(), q.clone()

    def call(r, q):
        ops.rope_append_kv_cache_fp8(q, k, v, r.q_indptr, *r.table(), r.layout)
        return ops.read_kv_cache_fp8(q.shape[0], r.q_indptr, *r.table(), r.layout)

    eager = call(a, qa)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = call(b, qb)
    rowsof = slice(a.q0[0], a.q0[-1])
    for _ in range(3):
        qb.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(eager, out):
            assert torch.equal(x[rowsof].view(torch.int16), y[rowsof].view(torch.int16))
        assert torch.equal(qa, qb) and torch.equal(a.exp, b.exp)
        (torch.randn(1000, device=DEV) * 2).sum().item()


def test_large_calls():
    """A call whose rows pass the caches by gives the bits of smaller ones."""
    from aoakv import ops
    _say("[append fp8] large")
    H, G, D, S, n = 32, 1, 64, 16, [3001, 2999]
    one, two = (Coded(n, n, D, S, H, G, seed=13, margin=0) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k, v = (torch.randn((sum(n), H, D), generator=g, device=DEV).half() for _ in range(3))
    q2 = q.clone()
    assert q.numel() * 2 * 3 >= 64 << 20
    ops.rope_append_kv_cache_fp8(q, k, v, one.q_indptr, *one.table(), HND)
    for b in range(2):
        a = slice(two.q0[b], two.q0[b + 1])
        ops.rope_append_kv_cache_fp8(q2[a], k[a], v[a], i32(0, n[b]), two.kv, two.exp,
                                     two.indptr[b:b + 2].contiguous(), two.indices,
                                     two.last[b:b + 1].contiguous(), HND)
    assert torch.equal(q, q2) and torch.equal(one.exp, two.exp)
    assert torch.equal(one.bytes(), two.bytes())
