"""Appends to a cache held in 8 bits and reading back, beyond test_gpu_fp8_append.py: the
error that the header allows a value over a page's whole history, every row of a call with
more rows than tokens, and large calls, whose rows pass the caches by."""
import sys

import pytest
import torch

from codes import (DEV, HND, I32, NHD, Coded, exponent, finite_top, held, i32, two_to, within)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


@pytest.mark.parametrize("D,S,grow", [(128, 16, 1), (128, 32, 0.5), (64, 32, 1), (256, 12, 2)])
def test_error_of_a_growing_page(D, S, grow):
    """Token by token with exponents that grow: each value stays within 2^-4 of itself and
    2^(e - 9), e its block's exponent at the end."""
    from aoakv import ops
    _say(f"[append fp8] a growing page, head dim {D}, pages of {S}")
    H, n = 3, 3 * S - 5
    g = torch.Generator(device=DEV).manual_seed(S)
    x = torch.randn((2, n, H, D), generator=g, device=DEV)
    # (within a page from 2^-6 on; elements of any size below the token's own)
    x *= torch.exp2(-6 + grow * (torch.arange(n, device=DEV) % S).clamp(max=14 / grow))[
        None, :, None, None]
    x *= torch.exp2(torch.randint(-8, 1, x.shape, generator=g, device=DEV).float())
    x = x.half()
    r = Coded([n], [n], D, S, H, seed=2, margin=0)
    at = int(r.indptr[0])
    for i in range(n):
        ops.append_kv_cache_fp8(x[0, i:i + 1].contiguous(), x[1, i:i + 1].contiguous(), i32(0, 1),
                                r.kv, r.exp, i32(at, at + i // S + 1), r.indices,
                                i32(i % S + 1), r.layout)
    moved = 0
    for which in (0, 1):
        e = r.exp[r.pages(0), which].double().t().repeat_interleave(S, 1)[:, :n, None]
        y = x[which].transpose(0, 1).double()
        for p in range(-(-n // S)):  # the exponent is that of the page's largest
            a = slice(p * S, min(n, p * S + S))
            assert torch.equal(exponent(finite_top(y[:, a], (1, 2))), e[:, p * S, 0].int())
        tol = 2.0 ** -4 * y.abs() + two_to(e - 9)
        within(r.cached(0, which), y, tol)
        moved += int((r.cached(0, which) != held(y, e)).sum())
    assert moved  # (values that were rounded more than once are among them)


def test_more_rows_than_tokens_read_back():
    """Rows before a sequence's first token are dropped by the append and left as they were by
    the reading back; every other row holds its token, of K and of V."""
    from aoakv import ops
    _say("[append fp8] more rows than tokens, K and V")
    D, S, H = 64, 16, 2
    g = torch.Generator(device=DEV).manual_seed(3)
    k, v = (torch.randn((28, H, D), generator=g, device=DEV).half() for _ in range(2))
    r = Coded([20, 3], [20, 3], D, S, H, seed=6, margin=0)
    ip = i32(0, 25, 28)  # 25 rows for 20 tokens, 3 for 3
    ops.append_kv_cache_fp8(k, v, ip, *r.table(), HND)
    out = [torch.full((28, H, D), 3.0, dtype=torch.float16, device=DEV) for _ in range(2)]
    got = ops.read_kv_cache_fp8(28, ip, *r.table(), HND, k=out[0], v=out[1])
    for which, x in ((0, k), (1, v)):
        assert torch.equal(got[which], out[which])
        assert torch.equal(out[which][:5], torch.full_like(x[:5], 3.0))
        for b, a in ((0, slice(5, 25)), (1, slice(25, 28))):
            assert torch.equal(out[which][a].double(), r.cached(b, which).transpose(0, 1))
            e = r.exp[r.pages(b), which].double().repeat_interleave(S, 0)[:r.lens[b], :, None]
            y = x[a].double()
            within(out[which][a], y, 2.0 ** -4 * y.abs() + two_to(e - 10))


@pytest.mark.parametrize("layout", [HND, NHD])
@pytest.mark.parametrize("D,S", [(128, 16), (128, 7), (64, 32), (256, 16), (256, 32), (64, 1)])
def test_large_calls(D, S, layout):
    """Codes, exponents, rotated queries and page statistics of a call whose rows pass the
    caches by are those of smaller ones, bit for bit; new tokens that begin inside of a page
    among them."""
    from aoakv import ops
    _say(f"[append fp8] large, head dim {D}, pages of {S}, layout {layout}")
    H, G = 8, 2
    heads = 2 * H + H * G
    old, n = [5, 0, 37], [(x << 20) // (heads * D) + 11 for x in (32, 16, 16)]
    lens = [a + b for a, b in zip(old, n)]
    T = sum(n)
    assert T * heads * D * 2 >= 64 << 20 > (max(n) + 1) // 2 * heads * D * 2
    one, two = (Coded(lens, n, D, S, H, G, layout, seed=13, margin=0) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k, v = (torch.randn((T, h, D), generator=g, device=DEV).half() for h in (H * G, H, H))
    q2 = q.clone()
    P, M = one.kv.shape[0], [-(-p // S) for p in one.P]
    at = [sum(M[:b]) for b in range(4)]
    md = torch.randperm(at[-1], generator=g, device=DEV).int()
    shape = (at[-1], 2, H, S, D) if layout == HND else (at[-1], 2, S, H, D)

    def statistics():
        f = lambda *s: torch.ones(s, dtype=torch.float16, device=DEV)  # noqa: E731
        return f(*shape), f(P, H), f(P, H, D)

    a, b = statistics(), statistics()
    ops.rope_append_kv_cache_fp8(q, k, v, one.q_indptr, *one.table(), layout, metadata_data=a[0],
                                 metadata_indptr=i32(*at), metadata_indices=md, v_log_norm=a[1],
                                 v_mean=a[2])
    for s in range(3):
        x = slice(two.q0[s], two.q0[s + 1])
        # (halves: no call is large; the second goes on where the first ended)
        for part in (0, 1):
            rows = slice(x.start, x.start + n[s] // 2) if part == 0 else \
                slice(x.start + n[s] // 2, x.stop)
            now = old[s] + (n[s] // 2 if part == 0 else n[s])
            ip = i32(two.ptr[s], two.ptr[s] - (-now // S))
            ops.rope_append_kv_cache_fp8(
                q2[rows], k[rows], v[rows], i32(0, rows.stop - rows.start), two.kv, two.exp, ip,
                two.indices, i32((now - 1) % S + 1), layout, metadata_data=b[0],
                metadata_indptr=i32(at[s], at[s + 1]), metadata_indices=md, v_log_norm=b[1],
                v_mean=b[2])
    assert torch.equal(q, q2)
    # the page where a sequence was cut: its statistics are the running mean's, and codes that
    # moved were rounded twice
    cut = [int(two.pages(s)[(old[s] + n[s] // 2) // S]) for s in range(3)]
    keep = torch.ones(P, dtype=torch.bool, device=DEV)
    keep[cut] = False
    same = lambda x, y: torch.equal(x.view(torch.uint8), y.view(torch.uint8))  # noqa: E731
    assert same(one.exp, two.exp)
    assert same(one.bytes()[keep].contiguous(), two.bytes()[keep].contiguous())
    assert same(a[0], b[0]) and same(a[1][keep], b[1][keep]) and same(a[2][keep], b[2][keep])
    for s, page in enumerate(cut):
        i = (old[s] + n[s] // 2) // S * S
        m = min(S, lens[s] - i)
        for which in (0, 1):
            x, y = (r.cached(s, which)[:, i:i + m] for r in (one, two))
            e = one.exp[page, which].double()[:, None, None]
            within(x, y, two_to(e - 9) + 2.0**-60)
