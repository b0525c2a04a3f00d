"""A sequence that is cut down to the tokens its attention goes to, as a program
drives it: InferenceController.track_weights, utils.chunk_forward and observe,
InferenceController.evict, and the calls that go on over the shorter cache; and
the same inside the Llama shim."""
import math
import sys

import pytest
import torch

from ragged import DEV, HND, NHD

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def controller(layers=2, H=8, hkv=2, D=128, S=16, max_len=1200, layout=HND, budget=16):
    from aoakv.utils import InferenceController
    c = InferenceController(layers, H, D, S, budget, max_len, torch.float16, DEV, layout=layout,
                            num_kv_heads=hkv, shuffle_seed=3)
    c.track_weights()
    return c


def tokens(c, n, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda h: torch.randn((n, h, c.head_dim), generator=g, device=DEV, dtype=torch.float16)
    return r(c.num_heads), r(c.num_kv_heads), r(c.num_kv_heads)


def cached(c, layer):
    """K and V of the sequence, [2, Hkv, L, D]."""
    x = c.kv_cache.buf_layer(layer)[torch.tensor(c.kv_cache.indicies, device=DEV)]
    x = x if c.layout == HND else x.transpose(2, 3)
    return x.permute(1, 2, 0, 3, 4).reshape(2, c.num_kv_heads, -1, c.head_dim)[
        :, :, :c.kv_cache.seqlen]


def attend(q, kv):
    """One query [H, D] over all of kv [2, Hkv, L, D] in fp64."""
    G = q.shape[0] // kv.shape[1]
    k, v = kv.double().repeat_interleave(G, 1)
    s = (q.double()[:, None] * k).sum(-1) / math.sqrt(q.shape[-1])
    return (torch.softmax(s, -1)[:, :, None] * v).sum(1)


@pytest.mark.parametrize("layout", [HND, NHD])
@pytest.mark.parametrize("D,S", [(128, 16), (64, 16), (128, 8)])
def test_a_sequence_through_an_eviction(D, S, layout):
    from aoakv import ops
    from aoakv.utils import (append_kv, chunk_forward, decode_estimate, decode_sparse_attn,
                             decode_topk, observe, prefill_forward, rope_append_kv)
    _say(f"[evict path] D={D} S={S} layout={layout}")
    N, keep, sink, recent = 700, 300, 4, 32
    c = controller(D=D, S=S, layout=layout)
    c.prepare_metadata(N)
    c.begin_forward(N)
    before, rows = [], []
    for layer in range(2):
        q, k, v = tokens(c, N, layer)
        rope_append_kv(q, k, v, c, layer)
        o, lse = chunk_forward(q, c, layer, return_lse=True)
        assert (o.float() - prefill_forward(q, c, layer).float()).abs().max() <= 4e-3
        observe(q, lse, c, layer, last=32)
        before.append(cached(c, layer).clone())
        rows.append((q, lse))
    pages = list(c.kv_cache.indicies)
    sums = [c.attn_weights_layer(i)[torch.tensor(pages, device=DEV)].transpose(0, 1)
            .reshape(c.num_kv_heads, -1)[:, :N] for i in range(2)]
    sums = [s.clone() for s in sums]
    for s in sums:  # 32 queries x 4 heads of a group
        assert ((s.double().sum(1) - 128).abs() < 1e-2).all()
    assert c.evict(keep, sink, recent) == N - keep and c.evicted == N - keep
    assert c.kv_cache.seqlen == keep and c.kv_cache.indicies == pages[:-(-keep // S)]
    assert len(c.metadata_cache.indicies) == -(-len(c.kv_cache.indicies) // S)
    assert c.evict(keep, sink, recent) == 0
    for layer in range(2):
        for h in range(c.num_kv_heads):
            w = sums[layer][h].clone()
            w[:sink] = w[N - recent:] = float("inf")
            best = torch.sort(w, descending=True, stable=True)[1][:keep].sort()[0]
            assert torch.equal(cached(c, layer)[:, h], before[layer][:, h, best])
    # decode goes on: positions count on, the cache holds one token more
    for step in range(20):
        c.prepare_metadata(1)
        c.begin_forward(1)
        for layer in range(2):
            q, k, v = tokens(c, 1, 100 + 2 * step + layer)
            q2, k2 = q.clone(), k.clone()
            ops.apply_rope_in_place(q2, k2, N + step)
            rope_append_kv(q, k, v, c, layer)
            assert torch.equal(q, q2) and torch.equal(k, k2)
            kv = cached(c, layer)
            assert kv.shape[2] == keep + step + 1
            assert torch.equal(kv[:, :, -1], torch.stack([k[0], v[0]]))
            ref = attend(q[0], kv)
            dense = decode_sparse_attn(q, c, layer, None)
            chunk, lse = chunk_forward(q, c, layer, return_lse=True)
            assert (dense[0].double() - ref).abs().max() <= 2e-3
            assert (chunk[0].double() - ref).abs().max() <= 2e-3
            observe(q, lse, c, layer)
            # page selection reads the packed pages' statistics
            scores = decode_estimate(q, c, layer)
            decode_topk(scores, c)
            o = decode_sparse_attn(q, c, layer, c.topk_dindices_buffer)
            assert scores.shape[1] == len(c.kv_cache.indicies) and o.isfinite().all()
    assert c.evict(keep, sink, recent) == 20 and c.evicted == N + 20 - keep
    c.check_errors()
    c.clean_states()
    assert c.evicted == 0 and c.kv_cache.pool.num_free_blocks == c.kv_cache.pool.capacity


def test_statistics_after_an_eviction():
    """Page scores over the packed cache are those of a cache that was filled with
    the kept tokens."""
    from aoakv.utils import append_kv, chunk_forward, decode_estimate, observe
    _say("[evict path] statistics")
    N, keep = 500, 200
    c, d = controller(layers=1), controller(layers=1)
    q, k, v = tokens(c, N, 5)
    c.prepare_metadata(N)
    c.begin_forward(N)
    append_kv(k, v, c, 0)
    _, lse = chunk_forward(q, c, 0, return_lse=True)
    observe(q, lse, c, 0)
    c.evict(keep)
    d.prepare_metadata(keep)
    d.begin_forward(keep)
    kk, vv = cached(c, 0).transpose(1, 2).contiguous()
    append_kv(kk, vv, d, 0)
    q1 = tokens(c, 1, 6)[0]
    c.begin_forward(1)
    d.begin_forward(1)
    assert torch.equal(decode_estimate(q1, c, 0), decode_estimate(q1, d, 0))


def test_refusals():
    c = controller(layers=1)
    for bad in ((0,), (10, 6, 5), (10, -1), (10, 0, -1)):
        with pytest.raises(ValueError, match="sink"):
            c.evict(*bad)
    c2 = type(c)(1, 4, 64, 16, 4, 64, torch.float16, DEV)
    with pytest.raises(RuntimeError, match="track_weights"):
        c2.evict(10)


def _model(cfg, **opts):
    from aoakv.shim import QuestLlamaModel
    torch.set_default_dtype(torch.float16)
    try:
        with torch.device(DEV):
            m = QuestLlamaModel(cfg).random_init(3, std=0.05)
    finally:
        torch.set_default_dtype(torch.float32)
    m.quest_init(page_size=16, max_seq_len=512, token_budget=128, device=DEV, **opts)
    return m


def test_the_model_evicts_after_its_prompt():
    from aoakv.shim import LlamaShape
    _say("[evict path] model")
    cfg = LlamaShape(hidden_size=512, num_attention_heads=4, num_key_value_heads=2,
                     num_hidden_layers=3, intermediate_size=1024)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((1, 300, 512), generator=g, device=DEV, dtype=torch.float16)
    steps = [torch.randn((1, 1, 512), generator=g, device=DEV, dtype=torch.float16)
             for _ in range(4)]
    plain, whole, cut = _model(cfg), _model(cfg, evict_keep=400), _model(cfg, evict_keep=150)
    h = [m(x) for m in (plain, whole, cut)]
    # the prompt itself is attended whole (by another kernel: fp16 noise of 3 layers)
    for other in h[1:]:
        assert (other.float() - h[0].float()).abs().max() <= 0.05
    assert whole.iController.evicted == 0 and cut.iController.evicted == 150
    assert cut.iController.kv_cache.seqlen == 150
    for i, s in enumerate(steps):
        a, b = plain(s), whole(s)
        assert (a.float() - b.float()).abs().max() <= 0.05
        out = cut.decode_graphed(s) if i else cut(s)
        assert out.isfinite().all() and cut.iController.kv_cache.seqlen == 151 + i
    cut.iController.check_errors()
    cut.quest_clear()
    assert cut.iController.evicted == 0
    with pytest.raises(ValueError, match="evict_keep"):
        _model(cfg, evict_keep=20)


def test_two_evictions_and_a_chunk_without_a_step_between():
    """Each goes by the tokens that the one before left, and a chunk after them
    by the pages it was given, in whatever order they come back."""
    from aoakv.utils import chunk_forward, observe, rope_append_kv
    _say("[evict path] twice")
    c = controller(layers=1)
    c.prepare_metadata(500)
    c.begin_forward(500)
    q, k, v = tokens(c, 500, 1)
    rope_append_kv(q, k, v, c, 0)
    _, lse = chunk_forward(q, c, 0, return_lse=True)
    observe(q, lse, c, 0)
    first, second = 300, 100
    sums = lambda: c.attn_weights_layer(0)[torch.tensor(c.kv_cache.indicies, device=DEV)].transpose(
        0, 1).reshape(c.num_kv_heads, -1)[:, :c.kv_cache.seqlen].clone()
    assert c.evict(first) == 200
    kv, w = cached(c, 0).clone(), sums()
    assert c.evict(second, 2, 8) == 200 and c.evicted == 400
    for h in range(c.num_kv_heads):
        x = w[h].clone()
        x[:2] = x[first - 8:] = float("inf")
        best = torch.sort(x, descending=True, stable=True)[1][:second].sort()[0]
        assert torch.equal(cached(c, 0)[:, h], kv[:, h, best])
    c.kv_cache._pool._free.reverse()  # (as another sequence's pages may leave the pool)
    kept = cached(c, 0).clone()
    c.prepare_metadata(450)
    c.begin_forward(450)
    q, k, v = tokens(c, 450, 2)
    rope_append_kv(q, k, v, c, 0)
    o = chunk_forward(q, c, 0)
    assert torch.equal(cached(c, 0)[:, :, :second], kept)
    assert torch.equal(cached(c, 0)[:, :, second:], torch.stack([k, v]).transpose(1, 2))
    for i in (0, 200, 449):
        ref = attend(q[i], cached(c, 0)[:, :, :second + i + 1])
        assert (o[i].double() - ref).abs().max() <= 2e-3
