"""The scratch memory of ops.chunk_attn: no more than the call's workgroups need,
and without it the call runs uncut."""
import random
import sys

import pytest
import torch

from ragged import DEV, HND, NHD, Ragged, i32, within


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def size(T, B, max_pages, Hq, H, D, S):
    from aoakv import _lib
    return _lib.load().aoakv_chunk_attn_call_workspace_size(T, B, max_pages, Hq, H, D, S)


def test_sizes():
    """Within the size for any context, growing with the context; a token of a short
    context takes little."""
    from aoakv import _lib
    rng = random.Random(5)
    for _ in range(300):
        D, S, H = rng.choice((64, 128, 256)), rng.choice((1, 5, 16, 32)), rng.choice((1, 3, 8, 32))
        Hq, T, B = H * rng.choice((1, 2, 5)), rng.choice((0, 1, 40, 3000, 70000)), rng.randint(1, 300)
        pages = sorted(rng.randint(1, 1 << rng.randint(1, 22)) for _ in range(2))
        a, b = (size(T, B, p, Hq, H, D, S) for p in pages)
        assert 0 < a <= b <= _lib.load().aoakv_chunk_attn_workspace_size(T, B, Hq, H, D)
    assert size(1, 1, 64, 8, 8, 128, 16) < 20 << 20
    for bad in (dict(D=96), dict(H=0), dict(Hq=512), dict(Hq=9)):
        assert size(**{**dict(T=1, B=1, max_pages=4, Hq=8, H=8, D=128, S=16), **bad}) == 0


def call(r, given, causal=1, window=0, soft_cap=0.0, slopes=None, prefix_len=None):
    """The C entry point with `given` bytes of workspace (None: no pointer)."""
    from aoakv import _lib
    o, lse = torch.full_like(r.q, 7.0), torch.full(r.q.shape[:2], 7.0, device=DEV)
    ws = None if given is None else torch.full((given + 64,), 0x55, dtype=torch.uint8, device=DEV)
    p = lambda t: None if t is None else t.data_ptr()
    _lib.call("aoakv_chunk_attn", p(r.q), p(o), p(lse), p(r.q_indptr), r.q.shape[0], p(r.kv),
              p(r.indptr), p(r.indices), p(r.last), p(prefix_len), p(slopes), r.B, r.max_pages,
              r.H * r.G, r.H, r.D, r.S, r.layout, causal, window, soft_cap, p(ws), given or 0,
              None, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return o, lse, ws


def check(r, **opts):
    """Without a workspace, with a byte too few, and with all of it."""
    need = size(r.q.shape[0], r.B, r.max_pages, r.H * r.G, r.H, r.D, r.S)
    ref_o, ref_lse, o_tol, lse_tol = r.attention(**opts)
    live = slice(r.q0[0], r.q0[-1])
    results = []
    for given in (None, need - 1, need):
        o, lse, ws = call(r, given, **opts)
        within(o[live], ref_o[live], o_tol[live])
        within(lse[live], ref_lse[live], lse_tol[live])
        assert (o[:r.q0[0]] == 7.0).all() and (o[r.q0[-1]:] == 7.0).all()
        assert ws is None or (ws[given:] == 0x55).all()
        results.append(o)
    assert torch.equal(results[0], results[1])


LENS = [1, 17, 64, 65, 128, 300, 0, 777, 5, 200, 129, 4000]
NEW = [1, 17, 1, 65, 127, 129, 0, 3, 0, 200, 128, 40]


@pytest.mark.gpu
@pytest.mark.parametrize("D,S,H,G,layout", [(128, 16, 2, 4, HND), (64, 16, 3, 2, NHD),
                                            (256, 16, 2, 2, HND), (256, 5, 1, 1, NHD),
                                            (128, 12, 2, 5, HND)])
def test_without_a_workspace(D, S, H, G, layout):
    _say(f"[room] D={D} S={S} H={H} G={G} layout={layout}")
    r = Ragged(LENS, NEW, D, S, H, G, layout, seed=D + S)
    check(r)
    check(r, soft_cap=30.0, slopes=r.slopes(), window=90, prefix_len=i32(*[3] * r.B))


@pytest.mark.gpu
def test_calls_of_many_items_without_a_workspace():
    _say("[room] many items")
    check(Ragged([9000, 900, 0, 64], [150, 900, 0, 64], 128, 16, 32, 2, seed=2, margin=12))
    check(Ragged([9000, 900, 0, 64], [150, 900, 0, 64], 256, 16, 16, 2, seed=2, margin=12))
    lens = [(37 * b) % 90 for b in range(700)]
    check(Ragged(lens, [min(n, 1 + b % 5) for b, n in enumerate(lens)], D=64, H=1, G=2, seed=9))


@pytest.mark.gpu
def test_torchs_pool_has_no_room():
    """The call runs without its scratch memory, with the bits of the call that is
    given none."""
    from aoakv import ops
    _say("[room] none in the pool")
    r = Ragged([16000, 3000], [60, 1], 128, 16, H=8, G=4, seed=3)
    need = size(r.q.shape[0], r.B, r.max_pages, 32, 8, 128, 16)
    assert need > 16 << 20
    whole, _, _ = call(r, None)
    o = torch.full_like(r.q, 7.0)

    def peak():
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        o.fill_(7.0)
        ops.chunk_attn(r.q, r.q_indptr, *r.tables(), o=o)
        return torch.cuda.max_memory_allocated() - before
    assert need <= peak() <= need + (2 << 20)
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(DEV).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (4 << 20)) / total)
    filler = []  # what the pool still has in pieces of this size
    try:
        with pytest.raises(torch.cuda.OutOfMemoryError):
            while True:
                filler.append(torch.empty(need, dtype=torch.uint8, device=DEV))
        assert peak() < need
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert torch.equal(o, whole)
