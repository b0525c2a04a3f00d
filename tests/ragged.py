"""A ragged batch of chunks over a paged cache, and in 64 bits what
ops.chunk_attn, attn_weights, keep_tokens and compact_kv_cache make of it, with
the error that the kernels' roundings allow."""
import math

import torch

from helpers import HND, NHD

DEV = "cuda:0"
I32 = dict(dtype=torch.int32, device=DEV)
NEG = float("-inf")


def i32(*v):
    return torch.tensor(v, **I32)


class Ragged:
    """``lens`` cached tokens per sequence, ``new`` of them the chunk's.  Pages
    shuffled, tables that start a few entries in, NaN in every slot that holds no
    token, rows before the first and behind the last sequence."""

    def __init__(self, lens, new, D=128, S=16, H=4, G=1, layout=HND, seed=0, scale=1.0, spare=0,
                 margin=2):
        self.lens, self.new, self.D, self.S, self.H, self.G = lens, new, D, S, H, G
        self.layout, self.B = layout, len(lens)
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.g = g
        P = [-(-n // S) for n in lens]
        self.P, total = P, max(1, sum(P))
        self.total = total
        f16 = dict(dtype=torch.float16, device=DEV)
        kv = torch.randn((total + spare, 2, H, S, D), generator=g, **f16)
        kv[:, 0] *= scale
        self.indices = torch.cat([i32(0, 0, 0), torch.randperm(total, generator=g,
                                                               device=DEV).int()])
        ptr = [3]
        for p in P:
            ptr.append(ptr[-1] + p)
        self.ptr, self.indptr = ptr, i32(*ptr)
        self.last = i32(*[(n - 1) % S + 1 if n else 0 for n in lens])
        for b, n in enumerate(lens):
            if n % S:
                kv[self.indices[ptr[b + 1] - 1].long(), :, :, n % S:] = float("nan")
        kv[total:] = float("nan")
        self.kv = kv if layout == HND else kv.transpose(2, 3).contiguous()
        self.margin = margin
        q0 = [margin]
        for n in new:
            q0.append(q0[-1] + n)
        self.q0, self.q_indptr = q0, i32(*q0)
        self.q = torch.randn((q0[-1] + margin, H * G, D), generator=g, **f16)
        self.max_pages = max(1, max(P))
        self.weights = torch.rand((total + spare, H, S), generator=g, device=DEV)

    def hnd(self):
        """The cache as [pages, 2, H, S, D] (a view)."""
        return self.kv if self.layout == HND else self.kv.transpose(2, 3)

    def pages(self, b):
        return self.indices[self.ptr[b]:self.ptr[b + 1]].long()

    def cached(self, b, which):
        """K (0) or V (1) of sequence b, [H, L, D] in fp64."""
        x = self.hnd()[self.pages(b), which].transpose(0, 1)
        return x.reshape(self.H, -1, self.D)[:, :self.lens[b]].double()

    def tables(self):
        return self.kv, self.indptr, self.indices, self.last, self.max_pages, self.layout

    def slopes(self):
        return 2.0 ** (-8.0 * torch.arange(1, self.H * self.G + 1, device=DEV) / (self.H * self.G))

    def scores(self, b, causal=True, window=0, soft_cap=0.0, slopes=None, prefix_len=None):
        """Scores [H, G, n, L] (-inf where unseen) and how far fp32 may have them off."""
        n, L = self.new[b], self.lens[b]
        q = self.q[self.q0[b]:self.q0[b + 1]].double().view(n, self.H, self.G, self.D)
        q = q.permute(1, 2, 0, 3)
        k = self.cached(b, 0)[:, None].transpose(2, 3)
        t = q @ k / math.sqrt(self.D)
        # products of fp16 are exact in fp32, sums of D terms round D times, the
        # factor, the cap, the distance and the exponent's factor a few more
        off = (q.abs() @ k.abs()).amax(-1, keepdim=True) / math.sqrt(self.D) * (self.D + 8) * 2**-24
        if soft_cap:
            t = soft_cap * torch.tanh(t / soft_cap)
            off = off + soft_cap * 2**-21
        pos = (L - n + torch.arange(n, device=DEV))[:, None]
        j = torch.arange(L, device=DEV)
        if slopes is not None:
            t = t - slopes.double().view(self.H, self.G, 1, 1) * (pos - j).abs()
        see = torch.ones_like(pos - j, dtype=torch.bool)
        if causal:
            see &= j <= pos
        if window:
            see &= pos - j < window
        if prefix_len is not None:
            see |= j < int(prefix_len[b])
        # (an exponent's own error; keys of infinitely small weight need no bound)
        near = torch.where(see & (t > t.masked_fill(~see, NEG).amax(-1, keepdim=True) - 30),
                           t.abs(), torch.zeros_like(t))
        off = off + 2**-21 * near.amax(-1, keepdim=True) if L else off.new_zeros(1)
        return t.masked_fill(~see, NEG), off

    def attention(self, **opts):
        """o, lse as the padded-free rows of q in fp64, and their error bounds."""
        o = torch.zeros(self.q.shape, dtype=torch.float64, device=DEV)
        lse = torch.zeros(self.q.shape[:2], dtype=torch.float64, device=DEV)
        o_tol, lse_tol = torch.zeros_like(o), torch.zeros_like(lse)
        for b in range(self.B):
            n, L = self.new[b], self.lens[b]
            if n == 0:
                continue
            rows = slice(self.q0[b], self.q0[b + 1])
            if L == 0:
                lse[rows] = NEG
                continue
            t, off = self.scores(b, **opts)
            e = torch.logsumexp(t, -1, keepdim=True)
            p = torch.where(t == NEG, torch.zeros_like(t), torch.exp(t - e))
            v = self.cached(b, 1)[:, None]
            v = torch.where(v.isfinite(), v, torch.zeros_like(v))
            x, size = p @ v, p @ v.abs()
            # probabilities and the result are rounded to fp16 (half a step each,
            # below 2^-14 of the largest 2^-25 absolutely), scores as above
            tol = 2**-11 * (x.abs() + size) + (off + L * 2**-24) * size + \
                L * 2**-25 * v.abs().amax()
            turn = lambda z: z.permute(2, 0, 1, 3).reshape(n, self.H * self.G, -1)
            o[rows], o_tol[rows] = turn(x), turn(tol)
            lse[rows] = turn(e).squeeze(-1)
            lse_tol[rows] = turn(off + L * 2**-24 + 2**-22 * (1 + e.abs().nan_to_num(0, 0, 0))
                                 ).squeeze(-1)
        return o, lse, o_tol, lse_tol

    def sums(self, lse, start=None, **opts):
        """The weights after attn_weights with these lse, in fp64, and their bounds."""
        w, tol = self.weights.double(), torch.zeros_like(self.weights, dtype=torch.float64)
        for b in range(self.B):
            n, L = self.new[b], self.lens[b]
            if L == 0:
                continue
            add = torch.zeros((self.H, L), dtype=torch.float64, device=DEV)
            off = torch.zeros((self.H, L), dtype=torch.float64, device=DEV)
            if n:
                t, d = self.scores(b, **opts)
                e = lse[self.q0[b]:self.q0[b + 1]].double().view(n, self.H, self.G)
                e = e.permute(1, 2, 0)[..., None]
                p = torch.where((t == NEG) | (e == NEG), torch.zeros_like(t), torch.exp(t - e))
                add = p.sum((1, 2))
                d = d + 2**-21 * (1 + e.abs().nan_to_num(0, 0, 0)) + n * self.G * 2**-24
                off = (p * d).sum((1, 2)) + n * self.G * 2**-120  # exponentials below the normal range
            first = L - n if start is None else int(start[b])
            pg, S = self.pages(b), self.S
            old = w[pg].transpose(0, 1).reshape(self.H, -1)
            o_tol = tol[pg].transpose(0, 1).reshape(self.H, -1)
            j = torch.arange(L, device=DEV)
            o_tol[:, :L] = off + 2**-23 * (old[:, :L].abs() + add)
            old[:, :L] = torch.where(j < first, old[:, :L], torch.zeros_like(add)) + add
            w[pg] = old.view(self.H, -1, S).transpose(0, 1)
            tol[pg] = o_tol.view(self.H, -1, S).transpose(0, 1)
        return w, tol


def within(x, ref, tol):
    """Asserts |x - ref| <= tol everywhere, infinities alike."""
    x = x.double()
    same = x == ref
    bad = ~(same | ((x - ref).abs() <= tol))
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off, first at "
                           f"{bad.nonzero()[0].tolist()}: {x[bad][0].item()} for "
                           f"{ref[bad][0].item()} (allowed {tol[bad][0].item()})")


__all__ = ["Ragged", "within", "i32", "DEV", "I32", "NEG", "HND", "NHD"]
