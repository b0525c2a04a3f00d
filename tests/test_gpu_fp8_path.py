"""A cache held in 8 bits through the controller (aoakv.utils), the Llama shim and the
latency driver: what the calls give is the attention of the values that read_kv gives back,
and the pages they select are those of an fp16 cache."""
import math
import sys

import pytest
import torch

from codes import DEV, E4M3, HND, NHD, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def controller(fp8, H=4, Hkv=2, D=128, S=16, budget=8, n=700, layout=HND, **k):
    from aoakv.utils import InferenceController
    return InferenceController(2, H, D, S, budget, n, torch.float16, DEV, layout=layout,
                               num_kv_heads=Hkv, shuffle_seed=3,
                               kv_dtype=E4M3 if fp8 else None, **k)


def attention(q, K, V, seen=None):
    """Causal attention of q [n, H, D], the last rows of K, V [L, Hkv, D], in fp64, and how
    far the kernels' roundings may have it off (tests/ragged.py's bound)."""
    n, H, D = q.shape
    L, Hkv, _ = K.shape
    k = K.double().transpose(0, 1).repeat_interleave(H // Hkv, 0)
    v = V.double().transpose(0, 1).repeat_interleave(H // Hkv, 0)
    x = q.double().transpose(0, 1)
    t = x @ k.transpose(1, 2) / math.sqrt(D)
    off = (x.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) / math.sqrt(D) * \
        (D + 8) * 2**-24 + 2**-21 * t.abs().amax(-1, keepdim=True)
    hide = torch.arange(L, device=DEV) > torch.arange(L - n, L, device=DEV)[:, None]
    t = t.masked_fill(hide, float("-inf"))
    if seen is not None:
        t = t.masked_fill(~seen[:, None], float("-inf"))
    p = torch.softmax(t, -1)
    o, size = p @ v, p @ v.abs()
    tol = 2**-11 * (o.abs() + size) + (off + L * 2**-24) * size + \
        L * 2**-25 * v.abs().amax() + 2**-25
    return o.transpose(0, 1), tol.transpose(0, 1)


@pytest.mark.parametrize("semantics", ["sim", "quest_kernel"])
@pytest.mark.parametrize("D,S,layout", [(128, 16, HND), (128, 16, NHD), (64, 16, HND),
                                        (256, 8, NHD), (128, 1, HND)])
def test_a_sequence(D, S, layout, semantics):
    """A prompt, a second chunk, decode steps over all pages and over selected ones."""
    from aoakv import utils as u
    _say(f"[fp8 path] head dim {D}, pages of {S}, layout {layout}, {semantics}")
    H, Hkv, layer = 4, 2, 1
    budget = 96 // S
    c8, c16 = (controller(f, H, Hkv, D, S, budget, layout=layout, semantics=semantics)
               for f in (True, False))
    g = torch.Generator(device=DEV).manual_seed(5)
    for n in (300, 37, 1, 1, 1, 1, 1):
        q, k, v = (torch.randn((n, h, D), generator=g, device=DEV).half() for h in (H, Hkv, Hkv))
        q16, k16, k0 = q.clone(), k.clone(), k.clone()
        for c in (c8, c16):
            c.prepare_metadata(n)
            c.begin_forward(n)
        u.rope_append_kv(q, k, v, c8, layer)
        u.rope_append_kv(q16, k16, v, c16, layer)
        assert torch.equal(k, k0)
        K, V = u.read_kv(c8, layer)
        assert K.shape == (c8.kv_cache.seqlen, Hkv, D)
        tail = u.read_kv(c8, layer, last=n)
        assert torch.equal(tail[0], K[-n:]) and torch.equal(tail[1], V[-n:])
        if n > 1:
            o = u.prefill_forward(q, c8, layer)
            ref, tol = attention(q, K, V)
            within(o, ref, tol)
            o2, lse = u.chunk_forward(q, c8, layer, window=50, return_lse=True)
            assert o2.shape == o.shape and lse.shape == (n, H)
            continue
        o = u.decode_sparse_attn(q, c8, layer, c8.kv_indices_without_last)
        ref, tol = attention(q, K, V)
        within(o, ref, tol)
        assert c8.need_estimate()
        # selected pages: those of the fp16 cache (its statistics, with its own rotation)
        s8, s16 = u.decode_estimate(q, c8, layer).clone(), u.decode_estimate(q16, c16, layer)
        # (keys turned by angles of 1e-5 apart at most, rounded to fp16 alike but for a step of
        # 2^-10 here and there: sums of D such products, and the larger of two)
        within(s8, s16.double(), torch.full_like(s8, 2**-6).double() * (1 + s16.abs().max()))
        u.decode_topk(s8, c8)
        sel = c8.topk_dindices_buffer[0].clone()
        o3 = u.decode_sparse_attn(q, c8, layer, c8.topk_dindices_buffer)
        o1 = u.decode_layer(q, c8, layer)
        assert torch.equal(o1, o3) and torch.equal(c8.topk_dindices_buffer[0], sel)
        where = {p: i for i, p in enumerate(c8.kv_cache.indicies)}
        seen = torch.zeros((Hkv, K.shape[0]), dtype=torch.bool, device=DEV)
        for h in range(Hkv):
            pages = [where[p] for p in sel[h].tolist()]
            if semantics == "quest_kernel":
                pages.append(len(where) - 1)
            for p in pages:
                seen[h, p * S:(p + 1) * S] = True
        ref, tol = attention(q, K, V, seen.repeat_interleave(H // Hkv, 0))
        within(o3, ref, tol)
    c8.check_errors()


def test_without_rotation_and_refusals():
    from aoakv import utils as u
    _say("[fp8 path] append, refusals")
    c = controller(True)
    c.prepare_metadata(40)
    c.begin_forward(40)
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn((40, 2, 128), generator=g, device=DEV).half() for _ in range(2))
    u.append_kv(k, v, c, 0)
    K, V = u.read_kv(c, 0)
    assert bool(((K.float() - k.float()).abs() <= k.float().abs() * 2**-4 + 2**-13).all())
    assert bool(((V.float() - v.float()).abs() <= v.float().abs() * 2**-4 + 2**-13).all())
    with pytest.raises(RuntimeError, match="fp16"):
        c.track_weights()
    c16 = controller(False)
    with pytest.raises(RuntimeError, match="8 bits"):
        u.read_kv(c16, 0)
    # a second conversation begins anew
    c.clean_states()
    c.prepare_metadata(3)
    c.begin_forward(3)
    u.append_kv(k[:3].contiguous(), v[:3].contiguous(), c, 0)
    K2, _ = u.read_kv(c, 0)
    assert K2.shape[0] == 3
    assert bool(((K2.float() - k[:3].float()).abs() <= k[:3].float().abs() * 2**-4 + 2**-13).all())


def model(kv_dtype, single_launch=True, budget=96):
    from aoakv.shim import LlamaShape, QuestLlamaModel
    cfg = LlamaShape(hidden_size=512, num_attention_heads=4, num_key_value_heads=2,
                     num_hidden_layers=4, intermediate_size=512)
    torch.set_default_dtype(torch.float16)
    try:
        with torch.device(DEV):
            m = QuestLlamaModel(cfg, single_launch=single_launch).random_init(3, std=0.05)
    finally:
        torch.set_default_dtype(torch.float32)
    m.quest_init(page_size=16, max_seq_len=700, token_budget=budget, device=DEV,
                 kv_dtype=kv_dtype)
    return m


def test_the_model():
    """Prompt and steps: eager, with the three calls, and replayed from a graph, the same
    bits; near an fp16 cache's, where the budget covers the sequence."""
    _say("[fp8 path] the model")
    a, b, c = model(E4M3), model(E4M3, single_launch=False), model(E4M3)
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn((1, 250, 512), generator=g, device=DEV).half()
    with torch.inference_mode():
        first = a(x)
        assert torch.equal(first, b(x)) and torch.equal(first, c(x))
        for _ in range(24):
            x = torch.randn((1, 1, 512), generator=g, device=DEV).half()
            h = a(x)
            assert torch.equal(h, b(x)) and torch.equal(h, c.decode_graphed(x))
            assert bool(h.isfinite().all())
    for m in (a, b, c):
        m.iController.check_errors()
    big, half = model(E4M3, budget=4096), model(None, budget=4096)
    g = torch.Generator(device=DEV).manual_seed(2)
    with torch.inference_mode():
        for n in (250, 1, 1):
            x = torch.randn((1, n, 512), generator=g, device=DEV).half()
            d = (big(x).double() - half(x).double()).norm() / half_norm(x)
            # 2^-4 at most of keys and values on each of 4 layers, whose outputs add to a
            # stream that begins with norm 1 an element
            assert float(d) < 4 * 2**-4, float(d)


def half_norm(x):
    """The final norm's rows have unit mean square."""
    return math.sqrt(x.numel())


def test_latency_driver(tmp_path):
    from aoakv import latency
    _say("[fp8 path] latency driver")
    out = tmp_path / "x.csv"
    row = latency.main(["--kv_dtype", "fp8", "--layers", "3", "--context_len", "600",
                        "--decode_len", "4", "--token_budget", "256", "--iteration", "1",
                        "--warmup", "1", "--graph", "--out", str(out)])
    assert row["method"] == "AOA_KV_fp8_graph" and out.exists()
