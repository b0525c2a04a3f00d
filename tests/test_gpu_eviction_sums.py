"""The sums that evictions go by, over a sequence's whole life: tokens that were
appended without an observation (decode steps) have none, whatever an earlier
owner of their slots left there."""
import math
import sys

import pytest
import torch

from ragged import DEV
from test_gpu_eviction_path import _model, cached, controller, tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _aoakv():
    import aoakv  # noqa: F401
    yield


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


class Expected:
    """Each layer's sums [Hkv, L] from their definition in fp64, with the error
    that the kernels' roundings allow."""

    def __init__(self, c):
        self.c = c
        self.clear()

    def clear(self):
        z = lambda: torch.zeros((self.c.num_kv_heads, 0), dtype=torch.float64, device=DEV)
        self.w = [z() for _ in range(self.c.num_layers)]
        self.tol = [z() for _ in range(self.c.num_layers)]

    def cut(self, L):
        self.w = [x[:, :L] for x in self.w]
        self.tol = [x[:, :L] for x in self.tol]

    def observe(self, layer, q, last):
        """The last `last` rows of q, whose tokens are the newest of the cache."""
        c = self.c
        L, D, G = c.kv_cache.seqlen, c.head_dim, c.num_heads // c.num_kv_heads
        had = self.w[layer].shape[1]
        pad = torch.zeros((c.num_kv_heads, L - had), dtype=torch.float64, device=DEV)
        w, tol = (torch.cat([x[layer], pad], 1) for x in (self.w, self.tol))
        q = q.view(-1, c.num_heads, D)[-last:].double().view(-1, c.num_kv_heads, G, D)
        n = q.shape[0]
        q = q.permute(1, 2, 0, 3)  # [Hkv, G, n, D]
        k = cached(c, layer)[0].double()[:, None].transpose(2, 3).contiguous()
        t = q @ k / math.sqrt(D)
        # as in ragged.py: D roundings of a sum of D terms and a few more, then the
        # exponent's; the kernel's own lse has the scores' error once more
        off = (q.abs() @ k.abs()).amax(-1, keepdim=True) / math.sqrt(D) * (D + 8) * 2**-24
        off = off + 2**-21 * t.abs().amax(-1, keepdim=True)
        pos = L - n + torch.arange(n, device=DEV)[:, None]
        t = t.masked_fill(torch.arange(L, device=DEV) > pos, float("-inf"))
        e = torch.logsumexp(t, -1, keepdim=True)
        p = torch.exp(t - e)
        d = 2 * off + 2**-20 * (1 + e.abs()) + (n * G + L) * 2**-24
        self.w[layer] = w + p.sum((1, 2))
        self.tol[layer] = tol + (p * d).sum((1, 2)) + 2**-23 * self.w[layer]

    def sums(self, i):
        """The controller's sums of the tokens that were observed."""
        c = self.c
        pages = torch.tensor(c.kv_cache.indicies, device=DEV)
        got = c.attn_weights_layer(i)[pages].transpose(0, 1).reshape(c.num_kv_heads, -1)
        return got[:, :self.w[i].shape[1]]

    def check(self, layers=None):
        for i in range(self.c.num_layers) if layers is None else layers:
            got = self.sums(i).double()
            bad = (got - self.w[i]).abs() > self.tol[i]
            assert not bad.any(), (i, bad.nonzero()[0].tolist(), got[bad][0], self.w[i][bad][0])

    def evict(self, evict, keep, sink, recent):
        """Calls `evict` and checks the kept tokens and their sums.  (The choice goes
        by the sums in fp32, which `check` holds to the definition.)"""
        c = self.c
        self.check()
        L = c.kv_cache.seqlen
        before = [cached(c, i).clone() for i in range(c.num_layers)]
        sums = [self.sums(i).clone() for i in range(c.num_layers)]
        evict(keep, sink, recent)
        for i in range(c.num_layers):
            # appended and not observed: nothing
            full = lambda z: torch.cat([z, z.new_zeros((z.shape[0], L - z.shape[1]))], 1)
            best = []
            for h in range(c.num_kv_heads):
                x = full(sums[i])[h]
                x[:sink] = x[L - recent:] = float("inf")
                best.append(torch.sort(x, descending=True, stable=True)[1][:keep].sort()[0])
                assert torch.equal(cached(c, i)[:, h], before[i][:, h, best[-1]]), (i, h)
            best = torch.stack(best)
            self.w[i], self.tol[i] = (full(z[i]).gather(1, best) for z in (self.w, self.tol))
            assert torch.equal(self.sums(i), full(sums[i]).gather(1, best))


def prompt(c, x, n, seed, last=32, observed=None):
    """A prompt of n tokens, observed in the layers `observed` (None: all)."""
    from aoakv.utils import append_kv, chunk_forward, observe
    c.prepare_metadata(n)
    c.begin_forward(n)
    for i in range(c.num_layers):
        q, k, v = tokens(c, n, seed + i)
        append_kv(k, v, c, i)
        _, lse = chunk_forward(q, c, i, return_lse=True)
        if observed is None or i in observed:
            observe(q, lse, c, i, last=last)
            x.observe(i, q, last)


def steps(c, n, seed):
    """Decode steps, whose queries are not observed."""
    from aoakv.utils import append_kv
    for s in range(n):
        c.prepare_metadata(1)
        c.begin_forward(1)
        for i in range(c.num_layers):
            _, k, v = tokens(c, 1, seed + 7 * s + i)
            append_kv(k, v, c, i)


@pytest.mark.parametrize("S", [16, 8])
def test_decoded_tokens_start_from_nothing(S):
    """Prompt, eviction, steps, a second prompt and its eviction; and the same in
    the pages that the sequence before gave back, steps first."""
    _say(f"[sums] two prompts, pages of {S}")
    c = controller(S=S)
    x = Expected(c)
    for turn in range(2):
        if turn:
            steps(c, 37, 500)
        prompt(c, x, 300, 1 + 10 * turn)
        x.check()
        x.evict(c.evict, 150, 4, 32)
        steps(c, 40, 1000 + turn)
        prompt(c, x, 120, 3000 + turn)
        x.check()
        x.evict(c.evict, 150, 4, 32)
        c.clean_states()
        x.clear()


@pytest.mark.parametrize("keep,recent", [(120, 8), (155, 40), (151, 0)])
def test_an_eviction_right_after_steps(keep, recent):
    """Tokens without a sum are dropped first, the later ones before the others."""
    _say(f"[sums] {keep} after steps")
    c = controller()
    x = Expected(c)
    prompt(c, x, 300, 21)
    x.evict(c.evict, 150, 4, 32)
    steps(c, 40, 2000)
    x.evict(c.evict, keep, 4, recent)
    prompt(c, x, 64, 31)
    x.check()


def test_layers_observe_by_themselves():
    _say("[sums] layers by themselves")
    c = controller()
    x = Expected(c)
    prompt(c, x, 250, 41, observed=[0])
    x.evict(c.evict, 200, 2, 16)
    steps(c, 20, 2500)
    prompt(c, x, 90, 51, observed=[1])
    x.check([1])
    x.evict(c.evict, 180, 2, 16)


def test_tokens_taken_back():
    """Drafted tokens that were observed and dropped: their slots' next tokens
    start from nothing."""
    _say("[sums] taken back")
    c = controller()
    x = Expected(c)
    prompt(c, x, 200, 61)
    prompt(c, x, 30, 71, last=30)
    c.kv_cache.truncate(205)
    c.metadata_cache.truncate(len(c.kv_cache.indicies))
    x.cut(205)
    steps(c, 20, 2600)
    prompt(c, x, 50, 81)
    x.check()
    x.evict(c.evict, 100, 4, 8)


def test_the_model_goes_by_its_prompts(monkeypatch):
    """The shim's decode steps are not observed."""
    from aoakv import utils
    from aoakv.shim import LlamaShape
    _say("[sums] model")
    cfg = LlamaShape(hidden_size=512, num_attention_heads=4, num_key_value_heads=2,
                     num_hidden_layers=3, intermediate_size=1024)
    m = _model(cfg, evict_keep=150)
    c = m.iController
    x = Expected(c)
    seen, observe, evict = [], utils.observe, c.evict

    def watched(q, lse, c, layer, last=None, **opts):
        observe(q, lse, c, layer, last=last, **opts)
        x.observe(layer, q, last)
        seen.append(layer)

    def watched_evict(*a):
        x.check()
        x.evict(evict, *a)
    monkeypatch.setattr(utils, "observe", watched)
    monkeypatch.setattr(c, "evict", watched_evict)
    g = torch.Generator(device=DEV).manual_seed(2)
    new = lambda n: torch.randn((1, n, 512), generator=g, device=DEV, dtype=torch.float16)
    for turn in range(2):
        if turn:
            for _ in range(20):
                m(new(1))
        m(new(300))
        for i in range(40):
            m.decode_graphed(new(1)) if i else m(new(1))
        m(new(200))
        assert c.kv_cache.seqlen == 150 and len(seen) == 6 * (turn + 1)
        c.check_errors()
        m.quest_clear()
        x.clear()
