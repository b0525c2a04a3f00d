"""A cache held in 8 bits beside an fp16 one that was given the same rows: page statistics,
scores and selected pages are equal, bit for bit.  And in the Llama shim every layer's
attention is that of the values that its cache gives back."""
import sys

import pytest
import torch

from codes import DEV, E4M3, HND, NHD, two_to, within
from test_gpu_fp8_append import turned
from test_gpu_fp8_path import attention, controller, model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


@pytest.mark.parametrize("semantics", ["sim", "quest_kernel"])
@pytest.mark.parametrize("D,S,H,layout,n", [(128, 16, 8, HND, 9000), (128, 16, 4, NHD, 1500),
                                            (64, 16, 4, HND, 1500), (256, 8, 2, NHD, 700)])
def test_scores_and_selected_pages(D, S, H, layout, n, semantics):
    """append_kv of the same rows to both, the same queries: a prompt, a chunk that begins
    inside of a page, single tokens."""
    from aoakv import utils as u
    _say(f"[fp8 same rows] head dim {D}, pages of {S}, {n} tokens, {semantics}")
    layer, budget = 1, 256 // S
    c8, c16 = (controller(f, H, H, D, S, budget, n + 100, layout, semantics=semantics)
               for f in (True, False))
    g = torch.Generator(device=DEV).manual_seed(6)
    for m in (n, 37, 1, 1, 1, 1, 1):
        q, k, v = (torch.randn((m, H, D), generator=g, device=DEV).half() for _ in range(3))
        for c in (c8, c16):
            c.prepare_metadata(m)
            c.begin_forward(m)
            u.append_kv(k, v, c, layer)
        if m > 1:
            continue
        s8, s16 = u.decode_estimate(q, c8, layer), u.decode_estimate(q, c16, layer)
        assert torch.equal(s8.view(torch.int32), s16.view(torch.int32))
        p8, p16 = u.decode_topk(s8, c8).clone(), u.decode_topk(s16, c16).clone()
        assert p8.numel() and torch.equal(p8, p16)
        # and as a decode layer selects them
        u.decode_layer(q, c8, layer)
        u.decode_layer(q, c16, layer)
        assert torch.equal(c8.topk_dindices_buffer[0], p8)
        assert torch.equal(c16.topk_dindices_buffer[0], p8)
    pages = torch.tensor(c8.kv_cache.indicies, device=DEV)
    assert c8.kv_cache.indicies == c16.kv_cache.indicies
    for a, b in ((c8.v_log_norm_layer(layer), c16.v_log_norm_layer(layer)),
                 (c8.v_mean_layer(layer), c16.v_mean_layer(layer))):
        assert torch.equal(a[pages].view(torch.int16), b[pages].view(torch.int16))
    c8.check_errors()
    c16.check_errors()


@pytest.mark.parametrize("budget", [96, 4096])
def test_every_layer_of_the_model(budget, monkeypatch):
    """What each layer's cache holds are the rows that the layer appended, turned, within one
    rounding to fp16 and those to codes; what its attention gives is the attention of the
    values held, within the roundings to fp16."""
    from aoakv import utils as u
    _say(f"[fp8 same rows] the model's layers, budget {budget}")
    m = model(E4M3, budget=budget)
    c, cfg = m.iController, m.cfg
    D, S = cfg.hidden_size // cfg.num_attention_heads, c.page_size
    G = cfg.num_attention_heads // cfg.num_key_value_heads
    rows = {i: [[], []] for i in range(cfg.num_hidden_layers)}
    seen = {"prefill_forward": 0, "decode_sparse_attn": 0, "decode_layer": 0}
    append = u.rope_append_kv

    def rope_append(q, k, v, c, layer, **kw):
        q0 = q.clone()
        append(q, k, v, c, layer, **kw)
        n, L = k.shape[0], c.kv_cache.seqlen
        pos = torch.arange(L - n, L, device=DEV)
        y, off = turned(q0, pos, cfg.rope_theta, cfg.rope_scale)
        within(q, y, off + 2.0 ** -11 * y.abs() + 2.0 ** -25)
        y, off = turned(k, pos, cfg.rope_theta, cfg.rope_scale)
        rows[layer][0].append((y, off + 2.0 ** -11 * y.abs() + 2.0 ** -25))
        rows[layer][1].append((v.double(), torch.zeros_like(off)))
        pages = torch.tensor(c.kv_cache.indicies, device=DEV)
        for which, got in enumerate(u.read_kv(c, layer)):
            y, off = (torch.cat([r[i] for r in rows[layer][which]]) for i in (0, 1))
            e = c.kv_exp[layer][pages, which].double().repeat_interleave(S, 0)[:L, :, None]
            within(got, y, off + 2.0 ** -4 * (y.abs() + off) + two_to(e - 9))

    def checked(name):
        call = getattr(u, name)

        def f(q, c, layer, *a, **kw):
            o = call(q, c, layer, *a, **kw)
            K, V = u.read_kv(c, layer)
            mask = None
            if name == "decode_layer":
                where = {p: i for i, p in enumerate(c.kv_cache.indicies)}
                sel = c.topk_dindices_buffer[0].tolist()
                mask = torch.zeros((len(sel), K.shape[0]), dtype=torch.bool, device=DEV)
                for h, pages in enumerate(sel):
                    for p in pages:
                        mask[h, where[p] * S:(where[p] + 1) * S] = True
                mask = mask.repeat_interleave(G, 0)
            q3 = q.view(-1, cfg.num_attention_heads, D)
            ref, tol = attention(q3, K, V, mask)
            within(o.view_as(q3), ref, tol)
            seen[name] += 1
            return o
        return f

    monkeypatch.setattr(u, "rope_append_kv", rope_append)
    for name in seen:
        monkeypatch.setattr(u, name, checked(name))
    g = torch.Generator(device=DEV).manual_seed(2)
    with torch.inference_mode():
        for n in (250, 1, 1, 1, 30, 1, 1):
            m(torch.randn((1, n, cfg.hidden_size), generator=g, device=DEV).half())
    layers = cfg.num_hidden_layers
    dense = layers if budget > 300 else 2
    assert seen == {"prefill_forward": 2 * layers, "decode_sparse_attn": 5 * dense,
                    "decode_layer": 5 * (layers - dense)}
    c.check_errors()
