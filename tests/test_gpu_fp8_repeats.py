"""Equal calls over a cache held in 8 bits give equal bits, whichever workgroup arrives last
at a join: attention of chunks in shares and listed, decode of few and many sequences."""
import sys

import pytest
import torch

from codes import DEV, Coded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def same_bits(call, times=12):
    first = [x.clone() for x in call()]
    other = torch.zeros(1 << 26, device=DEV)
    for i in range(times):
        if i % 3 == 1:
            other.add_(1.0)  # (work beside it, caches emptied)
        if i % 3 == 2:
            torch.cuda.synchronize()
        for x, y in zip(first, call()):
            n = torch.int16 if x.dtype == torch.float16 else torch.int32
            assert torch.equal(x.view(n), y.view(n)), f"call {i}"


@pytest.mark.parametrize("lens,new,H,G", [([2000], [1], 8, 4), ([16000, 5000, 9000], [5] * 3, 8, 4),
                                          ([6000, 900, 2500], [300, 900, 1], 4, 4),
                                          ([5000, 2100], [2100, 2100], 8, 4)])
def test_chunks(lens, new, H, G):
    from aoakv import ops
    _say(f"[fp8 repeats] chunks {new} of {lens}")
    r = Coded(lens, new, 128, 16, H, G, seed=1, margin=0)
    same_bits(lambda: ops.chunk_attn_fp8(r.q, r.q_indptr, *r.table(), r.max_pages, r.layout,
                                         return_lse=True))


@pytest.mark.parametrize("B,L,H,G,D", [(1, 1000, 8, 4, 128), (1, 30000, 4, 8, 128),
                                       (17, 3000, 8, 4, 128), (70, 900, 2, 2, 64),
                                       (3, 9000, 2, 2, 256)])
def test_decode(B, L, H, G, D):
    from aoakv import ops
    _say(f"[fp8 repeats] decode, {B} sequences of {L}")
    r = Coded([L - 37 * (b % 5) for b in range(B)], [1] * B, D, 16, H, G, seed=2, margin=0)
    ws = ops.decode_workspace(B, H * G, H, r.max_pages, DEV, head_dim=D)

    def call():
        o = torch.zeros_like(r.q)
        ops.decode_sparse_attn_fp8(r.q, o, *r.table(), None, 0, ws, r.max_pages, r.layout)
        return (o,)

    same_bits(call)
