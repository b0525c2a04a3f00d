"""Which tokens a kv head keeps (ops.keep_tokens), and the cache packed down to
them (ops.compact_kv_cache): positions equal the definition's, packed caches and
their statistics equal a bulk append of the kept tokens bit for bit."""
import sys

import pytest
import torch

from ragged import DEV, HND, I32, NHD, Ragged, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def expected_kept(r, keep, sink, recent, weights):
    out = torch.full((r.B, r.H, keep + 3), -5, dtype=torch.int32)
    for b in range(r.B):
        n = r.lens[b]
        for h in range(r.H):
            w = weights[r.pages(b), h].reshape(-1)[:n].tolist()
            order = sorted(range(n), key=lambda j: (not (j < sink or j >= n - recent),
                                                    w[j] != w[j], -w[j] if w[j] == w[j] else 0, j))
            k = sorted(order[:keep])
            out[b, h, :len(k)] = torch.tensor(k, dtype=torch.int32)
    return out


def keep(r, n, sink=0, recent=0, weights=None):
    from aoakv import ops
    kept = torch.full((r.B, r.H, n + 3), -5, **I32)
    w = r.weights if weights is None else weights
    ops.keep_tokens(w, r.indptr, r.indices, r.last, n, kept, r.max_pages, sink=sink, recent=recent)
    return kept


@pytest.mark.parametrize("S", [16, 1, 7, 32])
@pytest.mark.parametrize("n,sink,recent", [(1, 0, 0), (1, 1, 0), (5, 2, 3), (64, 4, 32), (100, 0, 0),
                                           (333, 10, 1), (2000, 4, 4)])
def test_keep(S, n, sink, recent):
    _say(f"[keep] {n} of pages of {S}")
    r = Ragged([0, 1, 2, 64, 65, 100, 101, 999, 1024, 1025, 3000], [0] * 11, 64, S, H=3, seed=n)
    assert torch.equal(keep(r, n, sink, recent).cpu(), expected_kept(r, n, sink, recent, r.weights))


@pytest.mark.parametrize("kind", ["zeros", "few values", "small and large", "special", "negative"])
def test_keep_orders(kind):
    """Ties go to the earlier token; infinities, NaN, both zeros, subnormals."""
    _say(f"[keep] {kind}")
    r = Ragged([2500, 40, 700], [0] * 3, 64, 16, H=2, seed=1)
    w = r.weights
    if kind == "zeros":
        w = torch.zeros_like(w)
    elif kind == "few values":
        w = (w * 4).floor()
    elif kind == "small and large":
        w = torch.where(w < 0.5, w * 1e-42, w * 1e38)
    elif kind == "special":
        table = torch.tensor([0.0, -0.0, float("inf"), float("-inf"), float("nan"), 1.0, -1.0, 1e-45],
                             device=DEV)
        w = table[(w * 8).long().clamp(max=7)]
    else:
        w = -w
    for n in (1, 30, 300, 1250):
        assert torch.equal(keep(r, n, 1, 0, w).cpu(), expected_kept(r, n, 1, 0, w)), n


def test_keep_long():
    _say("[keep] 150000 tokens")
    r = Ragged([150001, 70000], [0, 0], 64, 16, H=1, seed=2)
    w = (r.weights * 4096).floor() / 4096  # many ties
    for n in (1, 2048, 69999, 70000):
        assert torch.equal(keep(r, n, 4, 1 if n == 1 else 0, w).cpu() if n != 1 else
                           keep(r, 8, 4, 1, w).cpu(),
                           expected_kept(r, n if n != 1 else 8, 4, 1 if n == 1 else 0, w)), n


def test_keep_equal_bits_and_page_bound():
    from aoakv import ops
    _say("[keep] bound")
    r = Ragged([500, 100], [0, 0], 64, 16, H=2, seed=3)
    ws = ops.decode_workspace(1, 2, 2, 4)
    kept = torch.full((2, 2, 40), -1, **I32)
    ops.keep_tokens(r.weights, r.indptr, r.indices, r.last, 40, kept, 7, recent=5, workspace=ws)
    assert ops.workspace_error(ws) == ops.WS_ERR_TRUNCATED
    r.lens[0], r.ptr = 112, [r.ptr[0], r.ptr[0] + 7, r.ptr[2]]
    short = Ragged.__new__(Ragged)
    short.__dict__.update(r.__dict__, B=1)
    assert torch.equal(kept[:1].cpu(), expected_kept(short, 40, 0, 5, r.weights)[..., :40])


class Packed:
    """Statistics of r's cache, and metadata pages for a packed list."""

    def __init__(self, r, n):
        self.new = [min(x, n) for x in r.lens]
        self.P = [-(-x // r.S) for x in self.new]
        md = [-(-p // r.S) for p in self.P]
        g = torch.Generator(device=DEV).manual_seed(5)
        tot = max(1, sum(md))
        f16 = dict(dtype=torch.float16, device=DEV)
        shape = (2, r.H, r.S, r.D) if r.layout == HND else (2, r.S, r.H, r.D)
        self.meta = torch.full((tot,) + shape, 3.0, **f16)
        self.md_indices = torch.randperm(tot, generator=g, device=DEV).int()
        ptr = [0]
        for m in md:
            ptr.append(ptr[-1] + m)
        self.md_ptr, self.md_indptr = ptr, i32(*ptr)
        pages = r.kv.shape[0]
        self.log_norm = torch.full((pages, r.H), 3.0, **f16)
        self.mean = torch.full((pages, r.H, r.D), 3.0, **f16)

    def stats(self):
        return self.meta, self.md_indptr, self.md_indices, self.log_norm, self.mean


def expected_packed(r, kept, n, new_pages, p, weights):
    """kv, meta, log_norm, mean, weights after the call, by ops.append_kv_cache_prefill
    of each sequence's kept tokens into its new pages."""
    from aoakv import ops
    kv, w = r.kv.clone(), weights.clone()
    meta, ln, mean = p.meta.clone(), p.log_norm.clone(), p.mean.clone()
    for b, L in enumerate(r.lens):
        c = min(L, n)
        if c == 0:
            continue
        rows = kept[b, :, :c].long()
        pick = lambda x: torch.gather(x, 1, rows[..., None].expand(-1, -1, r.D))
        k, v = (pick(r.hnd()[r.pages(b), i].transpose(0, 1).reshape(r.H, -1, r.D))
                .transpose(0, 1).contiguous() for i in (0, 1))
        ww = torch.gather(weights[r.pages(b)].transpose(0, 1).reshape(r.H, -1), 1, rows)
        ops.append_kv_cache_prefill(k, v, kv, new_pages[b].int().contiguous(), p.P[b],
                                    (c - 1) % r.S + 1, meta,
                                    p.md_indices[p.md_ptr[b]:p.md_ptr[b + 1]].contiguous(), ln,
                                    mean, r.layout)
        t = torch.arange(c, device=DEV)
        w[new_pages[b][t // r.S].long(), :, t % r.S] = ww.t()
    return kv, meta, ln, mean, w


def same(a, b):
    """Equal bits (NaN in slots that hold no token)."""
    return torch.equal(a.view(torch.int16 if a.dtype == torch.float16 else torch.int32),
                       b.view(torch.int16 if b.dtype == torch.float16 else torch.int32))


LENS = [300, 0, 1, 17, 64, 1000, 129, 90]


@pytest.mark.parametrize("layout", [HND, NHD])
@pytest.mark.parametrize("D,S,H", [(128, 16, 3), (64, 16, 2), (256, 16, 2), (128, 1, 2),
                                   (128, 32, 1), (64, 7, 3), (256, 32, 1)])
@pytest.mark.parametrize("where", ["new pages", "in place"])
def test_compact(D, S, H, layout, where):
    from aoakv import ops
    _say(f"[compact] D={D} S={S} H={H} layout={layout} {where}")
    for n in (1, 16, 90, 400):
        news = [-(-min(x, n) // S) for x in LENS]
        r = Ragged(LENS, [0] * len(LENS), D, S, H, layout=layout, seed=D + n, spare=sum(news))
        kept = keep(r, n, 0, 0)
        p = Packed(r, n)
        if where == "in place":
            ip = ix = None
            pages = [r.pages(b)[:news[b]] for b in range(r.B)]
        else:
            ids = torch.randperm(max(1, sum(news)), device=DEV).int() + r.total
            ptr = [0]
            for c in news:
                ptr.append(ptr[-1] + c)
            ip, ix = i32(*ptr), ids
            pages = [ids[ptr[b]:ptr[b + 1]].long() for b in range(r.B)]
        ref = expected_packed(r, kept, n, pages, p, r.weights)
        w = r.weights.clone()
        ops.compact_kv_cache(kept, n, r.kv, r.indptr, r.indices, r.last, ip, ix, *p.stats(),
                             r.max_pages, layout, weights=w)
        for name, a, b in zip(("kv", "meta", "log_norm", "mean", "weights"),
                              (r.kv, p.meta, p.log_norm, p.mean, w), ref):
            assert same(a, b), (name, n)


@pytest.mark.parametrize("n", [1024, 2048, 5000])
def test_compact_long_in_place(n):
    """Many steps of a head's workgroup, weights absent."""
    from aoakv import ops
    _say(f"[compact] {n} of 9000 in place")
    r = Ragged([9000, 6000], [0, 0], H=4, seed=n)
    kept, p = keep(r, n, 4, 32), Packed(r, n)
    pages = [r.pages(b)[:p.P[b]] for b in range(2)]
    ref = expected_packed(r, kept, n, pages, p, r.weights)
    ops.compact_kv_cache(kept, n, r.kv, r.indptr, r.indices, r.last, None, None, *p.stats(),
                         r.max_pages, r.layout)
    for a, b in zip((r.kv, p.meta, p.log_norm, p.mean), ref):
        assert same(a, b)


def test_compact_of_any_rows():
    """Rows that no selection wrote: positions past the end (the last token is
    read), the same token twice; no access leaves the sequence's pages."""
    from aoakv import ops
    _say("[compact] any rows")
    r = Ragged([100], [0], H=2, seed=4, spare=4)
    rows = torch.tensor([0, 5, 5, 50, 99, 100, 2**31 - 1, -1], **I32).expand(1, 2, -1).contiguous()
    p = Packed(r, 8)
    ids = i32(r.total + 1)
    real = rows.clone()
    real[..., 5:] = 99
    ref = expected_packed(r, real, 8, [ids.long()], p, r.weights)
    w = r.weights.clone()
    ops.compact_kv_cache(rows, 8, r.kv, r.indptr, r.indices, r.last, i32(0, 1), ids, *p.stats(),
                         r.max_pages, r.layout, weights=w)
    for a, b in zip((r.kv, p.meta, p.log_norm, p.mean, w), ref):
        assert same(a, b)


def test_far_pages():
    """Pages whose elements lie past 2^32, packed from near to far and back."""
    from aoakv import ops
    _say("[compact] far pages")
    r = Ragged([200], [0], H=2, seed=6)
    far = (1 << 32) // r.kv[0].numel() + 3
    kv = torch.zeros((far + 8,) + r.kv.shape[1:], dtype=torch.float16, device=DEV)
    kv[:r.total] = r.kv
    kept = keep(r, 50, 2, 2)
    near = r.kv
    r.kv = kv
    p = Packed(r, 50)
    ids = torch.arange(4, **I32) + far
    ops.compact_kv_cache(kept, 50, kv, r.indptr, r.indices, r.last, i32(0, 4), ids, *p.stats(),
                         r.max_pages, r.layout)
    rows = kept[0, :, :50].long()
    for which in (0, 1):
        x = torch.gather(near[r.pages(0), which].transpose(0, 1).reshape(2, -1, 128), 1,
                         rows[..., None].expand(-1, -1, 128))
        got = kv[far:far + 4, which].transpose(0, 1).reshape(2, -1, 128)[:, :50]
        assert torch.equal(x, got)
    assert p.log_norm[far:far + 4].isfinite().all()


def test_graph_of_a_whole_eviction():
    """Attention, its weights, the choice and the packing in one captured graph,
    in the order a program runs them, replayed beside eager work."""
    from aoakv import ops
    _say("[evict] graph")
    r = Ragged([3000, 900, 40], [32, 32, 8], H=4, G=2, seed=7, spare=60)
    n = 256
    p = Packed(r, n)
    ptr = [0, p.P[0], p.P[0] + p.P[1], sum(p.P)]
    ip, ix = i32(*ptr), torch.arange(sum(p.P), **I32) + r.total
    i0 = i32(0, 0, 0)

    def go(w, kept, stats, kv):
        t = (kv,) + r.tables()[1:]
        _, lse = ops.chunk_attn(r.q, r.q_indptr, *t, return_lse=True)
        ops.attn_weights(r.q, lse, r.q_indptr, w, *t, start=i0)
        ops.keep_tokens(w, r.indptr, r.indices, r.last, n, kept, r.max_pages, sink=4, recent=16)
        ops.compact_kv_cache(kept, n, kv, r.indptr, r.indices, r.last, ip, ix, *stats,
                             r.max_pages, r.layout, weights=w)
    bufs = lambda: (r.weights.clone(), torch.full((3, 4, n), -1, **I32),
                    (p.meta.clone(), p.md_indptr, p.md_indices, p.log_norm.clone(),
                     p.mean.clone()), r.kv.clone())
    flat = lambda x: [x[0], x[2][0], x[2][3], x[2][4], x[3]]
    eager = bufs()
    go(*eager)
    held = bufs()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        go(*held)
    for k in range(3):
        for a, b in zip(flat(held), flat(bufs())):
            a.copy_(b)
        held[1].fill_(-1)
        g.replay()
        torch.cuda.synchronize()
        again = bufs()
        go(*again)
        for x in (held, again):
            assert torch.equal(x[1], eager[1]), k
            assert all(same(a, b) for a, b in zip(flat(x), flat(eager))), k
