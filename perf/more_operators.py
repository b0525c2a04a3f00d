"""What is timed of a paged cache held in 8 bits (e4m3 codes, and for K and V of each
page and kv head the exponent of a scale: a value is code * 2^exp):
``ops.rope_append_kv_cache_fp8`` / ``append_kv_cache_fp8`` (new tokens of a ragged batch),
``ops.chunk_attn_fp8`` (their attention), ``ops.decode_sparse_attn_fp8`` (one token per
sequence over all pages or selected ones) and ``ops.read_kv_cache_fp8`` (tokens back as
fp16 rows).

A case is a dict of sizes and options.  ``kind`` names the operator; ``batch`` sequences
hold up to ``context`` cached tokens, ``tokens`` of them new, ``heads`` / ``kv_heads`` x
``dim``, ``page`` tokens per page, page tables shuffled as after some serving.
``ragged``: lengths spread down to an eighth of the case's, else all are equal.
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "aoa-kv_amd"))

own = False  # True: the framework's operators; False: elementary torch operations

DEV = "cuda:0"
NEG = float("-inf")
ELEMENTS = 1 << 31  # scores of one call at most (padded batch)
E4M3 = torch.float8_e4m3fn
LOW, HIGH = -15, 8  # exponents of a scale
MOST = 61440.0      # the largest value that is held


def _case(name, kind, context, batch=1, heads=32, kv_heads=32, dim=128, page=16, layout=1,
          tokens=1, ragged=False, rope=True, stats=False, theta=1e4, causal=True, window=0,
          cap=0.0, alibi=False, prefix=0, budget=0):
    c = dict(kind=kind, context=context, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim,
             page=page, layout=layout, tokens=tokens, ragged=ragged)
    if kind == "append":
        c.update(rope=rope, stats=stats, theta=theta)
    if kind == "attn":
        c.update(causal=causal, window=window, cap=cap, alibi=alibi, prefix=prefix)
    if kind == "decode":
        c.update(budget=budget)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # a decode step of a batch: one token each, rotated and appended
        _case("append_step_b16", "append", 16000, batch=16, kv_heads=8, ragged=True),
        # a serving step that mixes chunks of prompts with short tails, statistics kept
        _case("append_mixed_nhd", "append", 6000, batch=16, kv_heads=8, tokens=400, ragged=True,
              layout=0, stats=True),
        # a long prompt, statistics kept
        _case("append_prompt_8k", "append", 8192, tokens=8192, stats=True),
        # one new token of one conversation
        _case("attn_token_2k", "attn", 2000, kv_heads=8),
        # a batch checks a few drafted tokens each, after contexts of up to 16k
        _case("attn_draft_16k", "attn", 16384, batch=8, kv_heads=8, tokens=5, ragged=True),
        # a serving step that mixes chunks of prompts with short tails, old tokens through a window
        _case("attn_mixed_window", "attn", 12000, batch=16, heads=16, kv_heads=4, tokens=300,
              ragged=True, window=4096, prefix=4, page=32, layout=0),
        # a long prompt over itself: the largest call
        _case("attn_prompt_8k", "attn", 8192, tokens=8192),
        # a decode step of one short conversation: the smallest call, where latency counts
        _case("decode_1k", "decode", 1000, kv_heads=8),
        # a long context, the pages that a budget of 2048 tokens selects
        _case("decode_selected_32k", "decode", 32768, budget=2048),
        # a batch of conversations, every page
        _case("decode_batch16", "decode", 16000, batch=16, kv_heads=8, ragged=True),
        # the last page of each conversation handed on
        _case("read_tail_b16", "read", 4000, batch=16, kv_heads=8, tokens=16, ragged=True),
        # whole conversations handed on
        _case("read_batch4_8k", "read", 8192, batch=4, tokens=8192, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attn", "attn", "attn", "decode", "decode", "read"])
    dim, heads, kv = rng.choice([(128, 32, 32), (128, 32, 8), (128, 32, 8), (128, 16, 4),
                                 (128, 8, 8), (128, 16, 2), (64, 32, 32), (64, 32, 8),
                                 (256, 16, 16), (256, 16, 8)])
    more = dict(heads=heads, kv_heads=kv, dim=dim, page=rng.choice([16, 16, 16, 16, 8, 32, 1, 12]),
                layout=rng.choice([1, 1, 0]), ragged=rng.random() < 0.7)
    context = _log(rng, 40, 24000)
    batch = _log(rng, 1, 24)
    while batch > 1 and batch * context * kv * dim > 16 * 12000 * 8 * 128:
        batch //= 2
    while batch * context * kv * dim > 16 * 12000 * 8 * 128:
        context //= 2
    if kind == "decode":
        budget = rng.choice([0, 0, _log(rng, 64, 4096)])
        return _case(None, kind, context, batch=batch, budget=budget, **more)
    tokens = min(context, rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 64, 4096), context]))
    if kind == "append":
        while tokens * batch * heads * dim > 8192 * 32 * 128:
            tokens //= 2
        rope = rng.random() < 0.8
        return _case(None, kind, context, batch=batch, tokens=tokens, rope=rope,
                     stats=rng.random() < 0.5, theta=rng.choice([1e4, 1e6]), **more)
    if kind == "read":
        while tokens * batch * kv * dim > 4 * 8192 * 32 * 128:
            tokens //= 2
        return _case(None, kind, context, batch=batch, tokens=tokens, **more)
    while heads * tokens * context * batch > ELEMENTS // 2:
        if batch > 1:
            batch //= 2
        elif tokens > 64:
            tokens //= 2
        else:
            context //= 2
            tokens = min(tokens, context)
    mask = rng.choice([{}, {}, dict(causal=False), dict(window=_log(rng, 16, 8192)),
                       dict(window=_log(rng, 16, 2048), prefix=rng.choice([4, 64])),
                       dict(prefix=_log(rng, 1, 600))])
    score = rng.choice([{}, {}, dict(cap=30.0), dict(alibi=True)])
    return _case(None, kind, context, batch=batch, tokens=tokens, **mask, **score, **more)


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """(cached tokens, new tokens among them) of each sequence."""
    r = random.Random(case["context"] * 31 + case["batch"] * 7 + case["tokens"])
    out = []
    for _ in range(case["batch"]):
        n = r.randint(max(1, case["context"] // 8), case["context"]) if case["ragged"] \
            else case["context"]
        t = n if case["tokens"] == case["context"] else min(n, case["tokens"])
        if case["ragged"] and 1 < t < n:
            t = r.randint(1, t)
        out.append((n, t))
    if case["ragged"]:  # one sequence has the case's own length
        out[0] = (case["context"], max(1, min(case["context"], case["tokens"])))
    if case.get("stats"):  # (statistics of whole pages: new tokens begin with one)
        out = [(n, n - (n - t) // case["page"] * case["page"]) for n, t in out]
    return out


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _tokens(g, n, H, D, keys):
    """Rows of n tokens: heads of different size, keys with a few large channels."""
    x = torch.randn((n, H, D), generator=g, device=DEV, dtype=torch.float16)
    x *= torch.exp2(torch.randint(-3, 3, (H, 1), generator=g, device=DEV)).half()
    if keys:
        x[..., torch.randperm(D, generator=g, device=DEV)[:4]] *= 3
    return x


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, S, H, D = case["batch"], case["page"], case["kv_heads"], case["dim"]
    lens = _lengths(case)
    pages = [-(-n // S) for n, _ in lens]
    total = sum(pages)

    def table(counts):
        ip = [0]
        for c in counts:
            ip.append(ip[-1] + c)
        return _i32(ip), torch.randperm(ip[-1], generator=g, device=DEV).to(torch.int32)

    indptr, indices = table(pages)
    ip = [0]
    for _, t in lens:
        ip.append(ip[-1] + t)
    s = dict(case=case, lens=_i32([n for n, _ in lens]), max_len=max(n for n, _ in lens),
             max_new=max(t for _, t in lens), max_pages=max(pages), indptr=indptr,
             indices=indices, last=_i32([(n - 1) % S + 1 for n, _ in lens]), tok_indptr=_i32(ip),
             rows=ip[-1])
    # the cache as appends left it: codes with the exponents of their blocks
    hnd = case["layout"] == 1
    kv = torch.empty((total, 2, H, S, D) if hnd else (total, 2, S, H, D), dtype=torch.uint8,
                     device=DEV).view(E4M3)
    exp = torch.empty((total, 2, H), dtype=torch.int8, device=DEV)
    for which in (0, 1):
        x = _tokens(g, total * S, H, D, which == 0).view(total, S, H, D)
        e = _exponent(x.abs().amax((1, 3)).float())
        exp[:, which] = e
        codes = _codes(x, e.view(total, 1, H, 1))
        kv[:, which] = codes.transpose(1, 2) if hnd else codes
    s.update(kv=kv, exp=exp)
    if case["kind"] == "append":
        s.update(k=_tokens(g, ip[-1], H, D, True), v=_tokens(g, ip[-1], H, D, False), q=None)
        if case["rope"]:
            s["q"] = torch.randn((ip[-1], case["heads"], D), generator=g, device=DEV,
                                 dtype=torch.float16)
        # the pages that get new tokens: page, first row, first slot, rows
        plan = []
        at = 0
        for b, (n, t) in enumerate(lens):
            for p in range((n - t) // S, pages[b]):
                e0 = max(n - t - p * S, 0)
                m = min(n - p * S, S) - e0
                plan.append((sum(pages[:b]) + p, at, e0, m))
                at += m
        s["plan"] = _i32(plan).long()
        # the tokens of those pages, which a pass returns
        back = [0]
        for n, t in lens:
            back.append(back[-1] + n - (n - t) // S * S)
        s.update(back_indptr=_i32(back), back_rows=back[-1])
        s["md_indptr"], s["md_indices"] = table([-(-n // S) for n in pages])
        if case["stats"]:
            z = lambda *d: torch.zeros(d, dtype=torch.float16, device=DEV)  # noqa: E731
            m = s["md_indices"].numel()
            s["meta"] = z(m, 2, H, S, D) if hnd else z(m, 2, S, H, D)
            s["log_norm"], s["mean"] = z(total, H), z(total, H, D)
    if case["kind"] == "attn":
        s.update(q=torch.randn((ip[-1], case["heads"], D), generator=g, device=DEV,
                               dtype=torch.float16),
                 slopes=2.0 ** (-8.0 * torch.arange(1, case["heads"] + 1, device=DEV) /
                                case["heads"]) if case["alibi"] else None,
                 prefix=_i32([case["prefix"]] * B) if case["prefix"] else None)
    if case["kind"] == "decode":
        s["q"] = torch.randn((B, case["heads"], D), generator=g, device=DEV, dtype=torch.float16)
        s["o"] = torch.empty_like(s["q"])
        s["sel"], s["picked"] = None, None
        if case["budget"]:  # the pages that a selection left: the first, the last, some between
            counts = [min(max(3, min(n, case["budget"]) // S), p) for (n, _), p in zip(lens, pages)]
            wide = max(counts)
            pick = torch.full((B, H, wide), -1, dtype=torch.int64, device=DEV)
            for b, (p, k) in enumerate(zip(pages, counts)):
                r = torch.rand((H, p), generator=g, device=DEV)
                r[:, 0] = r[:, -1] = 2.0
                pick[b, :, :k] = r.topk(k, -1)[1].sort(-1)[0]
            s["picked"] = pick
            at = (indptr[:-1].view(B, 1, 1) + pick.clamp(min=0)).long()
            s["sel"] = torch.where(pick >= 0, indices[at], torch.zeros_like(indices[at]))
    return s


# ------------------------------------------------------------------ plain forms
def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e, held to LOW .. HIGH."""
    m, x = torch.frexp(amax.clamp(min=2.0 ** -24) / 448.0)  # = m * 2^x, 0.5 <= m < 1
    return (x - (m == 0.5).to(x.dtype)).clamp(LOW, HIGH).to(torch.int8)


def _pow2(e):
    """2^e as bits (exp2 and pow may be off in the last place, which moves ties)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _codes(x, e):
    return (x.float().clamp(-MOST, MOST) * _pow2(-e)).to(E4M3)


def _slots(s, positions):
    """Physical page and slot of positions [B, ...] of every sequence."""
    S = s["case"]["page"]
    at = s["indptr"][:-1].view(-1, *[1] * (positions.dim() - 1)) + positions // S
    return s["indices"][at.clamp(max=s["indices"].numel() - 1).long()].long(), \
        (positions % S).long()


def _sequence(s, indptr, rows):
    """The sequence of each row, and its position."""
    t = torch.arange(rows, device=DEV)
    b = torch.searchsorted(indptr[1:].contiguous(), t, right=True)
    return b, s["lens"][b] - indptr[b + 1] + t


def _values(s, page, which, h, slot):
    """What the codes stand for, in fp32."""
    kv = s["kv"].view(torch.uint8)
    x = kv[page, which, h, slot] if s["case"]["layout"] == 1 else kv[page, which, slot, h]
    return x.view(E4M3).float() * _pow2(s["exp"][page, which, h])[..., None]


def _heads(s, dims):
    return torch.arange(s["case"]["kv_heads"], device=DEV).view(-1, *[1] * dims)


def _read(s, indptr, rows):
    b, pos = _sequence(s, indptr, rows)
    S = s["case"]["page"]
    page = s["indices"][(s["indptr"][b] + pos // S).long()].long()[:, None]
    slot = (pos % S).long()[:, None]
    h = torch.arange(s["case"]["kv_heads"], device=DEV)[None]
    return _values(s, page, 0, h, slot).half(), _values(s, page, 1, h, slot).half()


def _rotate(x, pos, theta):
    D = x.shape[-1]
    i = torch.arange(D // 2, device=DEV, dtype=torch.float64)
    a = pos.double()[:, None] * torch.pow(torch.tensor(theta, dtype=torch.float64, device=DEV),
                                          -2.0 * i / D)
    c, n = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    u, w = x[..., :D // 2].float(), x[..., D // 2:].float()
    return torch.cat([u * c - w * n, w * c + u * n], -1).half()


def _append(s):
    c = s["case"]
    S, hnd = c["page"], c["layout"] == 1
    k, v = s["k"], s["v"]
    if c["rope"]:
        _, pos = _sequence(s, s["tok_indptr"], s["rows"])
        k = _rotate(k, pos, c["theta"])
        s["q"].copy_(_rotate(s["q"], pos, c["theta"]))
    at, row, e0, m = s["plan"].unbind(1)
    page = s["indices"][at].long()
    i = torch.arange(S, device=DEV)
    live = i < m[:, None]
    kv = s["kv"].view(torch.uint8)
    kv = kv if hnd else kv.transpose(2, 3)
    rows = (row[:, None] + i).clamp(max=s["rows"] - 1)
    for which, x in ((0, k[rows]), (1, v[rows])):
        top = torch.where(live[:, :, None, None], x, torch.zeros_like(x)).abs().amax((1, 3))
        e = _exponent(top.float())
        old = s["exp"][page, which]
        e = torch.where(e0[:, None] > 0, torch.maximum(e, old), e)
        s["exp"][page, which] = e
        # older codes of the page, at the block's new exponent
        codes = kv[page, which]                                            # [n, H, S, D]
        moved = (codes.view(E4M3).float() *
                 _pow2(old.int() - e.int())[..., None, None]).to(E4M3)
        new = _codes(x, e[:, None, :, None]).transpose(1, 2)               # rows from slot 0 on
        src = (i - e0[:, None]).clamp(min=0)[:, None, :, None].expand_as(codes)
        new = torch.gather(new.view(torch.uint8), 2, src)
        put = (i >= e0[:, None]) & (i < (e0 + m)[:, None])
        old_slot = (i < e0[:, None])[:, None, :, None]
        codes = torch.where(old_slot, moved.view(torch.uint8), codes)
        kv[page, which] = torch.where(put[:, None, :, None], new, codes)
    if c["stats"]:
        _statistics(s, k[rows], v[rows], live, page)
    out = _read(s, s["back_indptr"], s["back_rows"])
    return out + ((s["q"],) if c["rope"] else ()) + \
        ((s["meta"], s["log_norm"], s["mean"]) if c["stats"] else ())


def _statistics(s, k, v, live, page):
    """Of pages that begin empty; k, v [n, S, H, D]."""
    S = s["case"]["page"]
    at = s["plan"][:, 0]
    b = torch.searchsorted(s["indptr"][1:].contiguous(), at, right=True)
    p = at - s["indptr"][b]
    mp = s["md_indices"][(s["md_indptr"][b] + p // S).long()].long()
    mask = live[:, :, None, None]
    k32, v32 = k.float(), v.float()
    hi = torch.where(mask, k32, torch.full_like(k32, NEG)).amax(1).half()
    lo = torch.where(mask, k32, torch.full_like(k32, -NEG)).amin(1).half()
    mean = (torch.where(mask, v32, torch.zeros_like(v32)).sum(1) /
            live.sum(1)[:, None, None]).half()
    meta = s["meta"] if s["case"]["layout"] == 1 else s["meta"].transpose(2, 3)
    meta[mp, 0, :, p % S] = hi
    meta[mp, 1, :, p % S] = lo
    s["mean"][page] = mean
    s["log_norm"][page] = torch.log(
        torch.sqrt(mean.float().square().sum(-1)).half().float()).half()


def _rows(s, which):
    """K (0) or V (1) of the padded batch, [B, H, max_len, D] in fp32."""
    pos = torch.arange(s["max_len"], device=DEV).expand(s["case"]["batch"], -1)
    page, slot = _slots(s, pos)
    return _values(s, page[:, None], which, _heads(s, 1), slot[:, None])


def _scores(s):
    """Scores [B, H, group, max_new, max_len] of the padded batch, -inf where a
    query does not see a key (or there is none)."""
    c = s["case"]
    B, H, G, n = c["batch"], c["kv_heads"], c["heads"] // c["kv_heads"], s["max_new"]
    i = torch.arange(n, device=DEV)
    row = (s["tok_indptr"][:-1, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"][row.long()].float().view(B, n, H, G, -1).permute(0, 2, 3, 1, 4)
    t = torch.matmul(q.reshape(B, H, G * n, -1), _rows(s, 0).transpose(2, 3).contiguous())
    t = t.view(B, H, G, n, -1) / math.sqrt(c["dim"])
    if c["cap"]:
        t = c["cap"] * torch.tanh(t / c["cap"])
    count = s["tok_indptr"][1:] - s["tok_indptr"][:-1]
    pos = ((s["lens"] - count)[:, None] + i)[:, :, None]
    j = torch.arange(s["max_len"], device=DEV)
    if s["slopes"] is not None:
        t = t - s["slopes"].view(1, H, G, 1, 1) * (pos - j).abs()[:, None, None]
    sees = torch.ones_like(pos - j, dtype=torch.bool)
    if c["causal"]:
        sees = sees & (j <= pos)
    if c["window"]:
        sees = sees & (j > pos - c["window"])
    if s["prefix"] is not None:
        sees = sees | (j < s["prefix"].view(-1, 1, 1))
    sees = sees & (j < s["lens"].view(-1, 1, 1)) & (i.view(1, -1, 1) < count.view(-1, 1, 1))
    return t.masked_fill_(~sees[:, None, None], NEG)


def _flat(s, x):
    """Padded rows [B, H, group, max_new, ...] as the tokens of q, [T, heads, ...]."""
    b, _ = _sequence(s, s["tok_indptr"], s["rows"])
    t = torch.arange(s["rows"], device=DEV) - s["tok_indptr"][b]
    return x[b, :, :, t.long()].flatten(1, 2)


def _attention(s):
    t = _scores(s)
    top = t.amax(-1, keepdim=True)
    top = torch.where(top == NEG, torch.zeros_like(top), top)
    p = torch.exp(t - top)
    del t
    total = p.sum(-1, keepdim=True)
    B, H, G, n, _ = p.shape
    o = torch.matmul(p.view(B, H, G * n, -1), _rows(s, 1)).view(B, H, G, n, -1)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return _flat(s, o).half(), _flat(s, (top + torch.log(total)).squeeze(-1))


def _decode(s):
    c = s["case"]
    B, H, S, D = c["batch"], c["kv_heads"], c["page"], c["dim"]
    if s["picked"] is None:
        j = torch.arange(s["max_len"], device=DEV).expand(B, -1)
        j, inside = j[:, None], (j < s["lens"].view(-1, 1))[:, None]
    else:
        j = (s["picked"][..., None] * S + torch.arange(S, device=DEV)).flatten(2)
        inside = (j >= 0) & (j < s["lens"].view(-1, 1, 1))
    page, slot = _slots(s, j.clamp(min=0))
    h = _heads(s, 1)
    q = s["q"].float().view(B, H, -1, D)
    t = torch.matmul(q, _values(s, page, 0, h, slot).transpose(2, 3).contiguous()) / math.sqrt(D)
    t = t.masked_fill(~inside[:, :, None], NEG)
    p = torch.exp(t - t.amax(-1, keepdim=True))
    o = torch.matmul(p, _values(s, page, 1, h, slot)) / p.sum(-1, keepdim=True)
    s["o"].copy_(o.reshape(B, -1, D))
    return s["o"]


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if not own:
        if c["kind"] == "read":
            return _read(s, s["tok_indptr"], s["rows"])
        return {"append": _append, "attn": _attention, "decode": _decode}[c["kind"]](s)
    from aoakv import ops
    table = (s["kv"], s["exp"], s["indptr"], s["indices"], s["last"])
    if c["kind"] == "append":
        stats = dict(metadata_data=s["meta"], metadata_indptr=s["md_indptr"],
                     metadata_indices=s["md_indices"], v_log_norm=s["log_norm"],
                     v_mean=s["mean"]) if c["stats"] else {}
        if c["rope"]:
            ops.rope_append_kv_cache_fp8(s["q"], s["k"], s["v"], s["tok_indptr"], *table,
                                         c["layout"], rope_theta=c["theta"], **stats)
        else:
            ops.append_kv_cache_fp8(s["k"], s["v"], s["tok_indptr"], *table, c["layout"], **stats)
        out = ops.read_kv_cache_fp8(s["back_rows"], s["back_indptr"], *table, c["layout"])
        return out + ((s["q"],) if c["rope"] else ()) + \
            ((s["meta"], s["log_norm"], s["mean"]) if c["stats"] else ())
    if c["kind"] == "attn":
        return ops.chunk_attn_fp8(s["q"], s["tok_indptr"], *table, s["max_pages"], c["layout"],
                                  causal=c["causal"], window=c["window"], soft_cap=c["cap"],
                                  slopes=s["slopes"], prefix_len=s["prefix"], return_lse=True)
    if c["kind"] == "decode":
        if "workspace" not in s:  # (a program keeps one)
            pages = s["max_pages"] if s["sel"] is None else s["sel"].shape[-1]
            s["workspace"] = ops.decode_workspace(c["batch"], c["heads"], c["kv_heads"], pages,
                                                  DEV, head_dim=c["dim"])
        ops.decode_sparse_attn_fp8(s["q"], s["o"], *table, s["sel"], c["budget"], s["workspace"],
                                   s["max_pages"], c["layout"])
        return s["o"]
    return ops.read_kv_cache_fp8(s["rows"], s["tok_indptr"], *table, c["layout"])


# ------------------------------------------------------------------ what a pass needs
def _seen(case):
    """Over the batch: (query, key) pairs per query head, and keys that any query sees."""
    pairs = keys = 0
    W, p = case["window"], case["prefix"]
    for n, t in _lengths(case):
        pos = torch.arange(n - t, n, dtype=torch.int64)
        hi = pos + 1 if case["causal"] else torch.full_like(pos, n)
        lo = (pos + 1 - W).clamp(min=0) if W else torch.zeros_like(pos)
        a = min(p, n)
        pairs += int((a + (hi - lo.clamp(min=a)).clamp(min=0)).sum())
        keys += min(n, a + max(0, int(hi.max()) - max(a, int(lo.min()))))
    return pairs, keys


def work(case):
    H, D, Hq, S = case["kv_heads"], case["dim"], case["heads"], case["page"]
    lens = _lengths(case)
    new = sum(t for _, t in lens)
    if case["kind"] == "attn":
        pairs, keys = _seen(case)
        return {"bytes": new * Hq * (4 * D + 4) + keys * H * 2 * D, "flops": 4.0 * pairs * Hq * D}
    if case["kind"] == "decode":
        seen = sum(min(n, max(3, min(n, case["budget"]) // S) * S) if case["budget"] else n
                   for n, _ in lens)
        return {"bytes": seen * H * 2 * D + len(lens) * Hq * 4 * D, "flops": 4.0 * seen * Hq * D}
    if case["kind"] == "read":
        return {"bytes": new * H * 6 * D, "flops": 2.0 * new * H * D}
    # appended, and the touched pages' tokens read back as fp16
    back = sum(n - (n - t) // S * S for n, t in lens)
    pages = sum(-(-n // S) - (n - t) // S for n, t in lens)
    stats = pages * H * (6 * D + 2) if case["stats"] else 0
    turn = 4 * D * Hq if case["rope"] else 0
    return {"bytes": new * (H * 6 * D + turn) + stats + back * H * 6 * D,
            "flops": 3.0 * new * D * (2 * H + (Hq if case["rope"] else 0))}


# ------------------------------------------------------------------ in 64 bits
def _cached(s, b, which, h):
    """[L, D] of one head of a sequence, in fp64."""
    S, n, p = s["case"]["page"], int(s["lens"][b]), s["indptr"].tolist()
    pages = s["indices"][p[b]:p[b + 1]].long()
    x = s["kv"].view(torch.uint8)[pages, which]
    x = x[:, h] if s["case"]["layout"] == 1 else x[:, :, h]
    x = x.contiguous().view(E4M3).float().double() * _two_to(s["exp"][pages, which, h])[
        :, None, None]
    return x.reshape(-1, s["case"]["dim"])[:n]


def _two_to(x):
    """2^x of whole x in fp64, from a table."""
    at = torch.tensor([2.0 ** i for i in range(-64, 65)], dtype=torch.float64, device=DEV)
    return at[x.long() + 64]


def _held(x, e):
    """What a code holds of x at exponent e: four significant bits, none below 2^(e - 9)."""
    x = x.clamp(-MOST, MOST)
    step = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0 + e) - 3.0
    return torch.round(x / _two_to(step)) * _two_to(step)


def exact(case, seed):
    s = prepare(case, seed)
    H, D, G = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    lens = _lengths(case)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "read":
        return tuple(torch.cat([torch.stack([_cached(s, b, w, h)[n - t:] for h in range(H)], 1)
                                for b, (n, t) in enumerate(lens)]) for w in (0, 1))
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)
    at = 0
    for b, (n, t) in enumerate(lens):
        j = torch.arange(n, device=DEV)
        for h in range(H):
            k, v = _cached(s, b, 0, h).t().contiguous(), _cached(s, b, 1, h)
            if case["kind"] == "decode":
                z = s["q"][b, h * G:(h + 1) * G].double() @ k * (1.0 / math.sqrt(D))
                if s["picked"] is not None:
                    z.masked_fill_(~torch.isin(j // case["page"], s["picked"][b, h]), NEG)
                o[b, h * G:(h + 1) * G] = torch.softmax(z, 1) @ v
                continue
            for hq in range(h * G, h * G + G):
                for r in range(0, t, 4096):
                    q = s["q"][at + r:at + min(t, r + 4096), hq].double()
                    z = q @ k * (1.0 / math.sqrt(D))
                    if case["cap"]:
                        z = torch.tanh(z / case["cap"]) * case["cap"]
                    p = torch.arange(n - t + r, n - t + r + q.shape[0], device=DEV)[:, None]
                    if case["alibi"]:
                        z = z - float(s["slopes"][hq]) * (p - j).abs()
                    hide = torch.zeros_like(p - j, dtype=torch.bool)
                    if case["causal"]:
                        hide |= j > p
                    if case["window"]:
                        hide |= j <= p - case["window"]
                    hide &= j >= case["prefix"]
                    z.masked_fill_(hide, NEG)
                    e = torch.logsumexp(z, 1)
                    lse[at + r:at + r + q.shape[0], hq] = e
                    o[at + r:at + r + q.shape[0], hq] = torch.exp(z - e[:, None]) @ v
        at += t
    return o if case["kind"] == "decode" else (o, lse)


def _exact_append(s):
    """Page by page of a sequence, all heads at once."""
    case = s["case"]
    S, H, D, Hq = case["page"], case["kv_heads"], case["dim"], case["heads"]
    mp, md = s["md_indptr"].tolist(), s["md_indices"].tolist()
    ip, ids = s["indptr"].tolist(), s["indices"].tolist()
    turned, back = [], ([], [])
    stats = case["stats"]
    if stats:
        meta, norm, mean = s["meta"].double(), s["log_norm"].double(), s["mean"].double()
    at = 0
    for b, (n, t) in enumerate(_lengths(case)):
        k, v = s["k"][at:at + t].double(), s["v"][at:at + t].double()
        if case["rope"]:
            pos = torch.arange(n - t, n, device=DEV, dtype=torch.float64)
            turn = pos[:, None] * case["theta"] ** (
                -torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
            turn = torch.complex(torch.cos(turn), torch.sin(turn))[:, None]

            def rotated(x):
                z = torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn
                return torch.cat([z.real, z.imag], -1)

            k = rotated(k).half().double()
            turned.append(rotated(s["q"][at:at + t].double()))
        at += t
        first = (n - t) // S
        e0 = n - t - first * S
        for p in range(first, -(-n // S)):
            lo = max(p * S - (n - t), 0)
            hi = min((p + 1) * S - (n - t), t)
            page = ids[ip[b] + p]
            for which, x in ((0, k[lo:hi]), (1, v[lo:hi])):
                e = torch.ceil(torch.log2(x.abs().amax((0, 2)) / 448.0)).clamp(LOW, HIGH)
                if p == first and e0:
                    e = torch.maximum(e, s["exp"][page, which].double())
                    c = s["kv"].view(torch.uint8)[page, which]
                    c = c.transpose(0, 1) if case["layout"] == 1 else c
                    c = c[:e0].contiguous().view(E4M3).float().double()
                    c = c * _two_to(s["exp"][page, which])[:, None]
                    back[which].append(_held(c, e[:, None]))
                back[which].append(_held(x, e[:, None]))
            if stats:
                q = md[mp[b] + p // S]
                for which, x in ((0, k[lo:hi].amax(0)), (1, k[lo:hi].amin(0))):
                    if case["layout"] == 1:
                        meta[q, which, :, p % S] = x
                    else:
                        meta[q, which, p % S] = x
                mean[page] = v[lo:hi].mean(0)
                norm[page] = torch.log(mean[page].norm(dim=-1))
    return (torch.cat(back[0]), torch.cat(back[1])) + \
        ((torch.cat(turned),) if case["rope"] else ()) + \
        ((meta, norm, mean) if stats else ())
