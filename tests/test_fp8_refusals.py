"""What the calls over a cache held in 8 bits and their C entry points refuse, before
anything is launched (no GPU needed)."""
import re

import pytest
import torch

from aoakv import _lib, ops

H, I, F, B, C, E = (torch.float16, torch.int32, torch.float32, torch.uint8, torch.float8_e4m3fn,
                    torch.int8)
P = 1 << 12  # an address that no call gets to


def call(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    return rc, lib.aoakv_last_error().decode()


TABLE = dict(kv=P, exp=P, indptr=P, indices=P, last=P)
STATS = dict(meta=P, md_indptr=P, md_indices=P, log_norm=P, mean=P)
SHAPE = dict(batch=2, hkv=4, dim=128, page=16, layout=1)
APPEND = dict(k=P, v=P, tok_indptr=P, rows=4, **TABLE, **STATS, **SHAPE, stream=None)
# (q far from k and v: it may not share memory with them)
ROPE = dict(q=P << 20, k=P, v=P, tok_indptr=P, rows=4, hq=8, **TABLE, **STATS, **SHAPE, scale=1.0,
            theta=1e4, stream=None)
READ = dict(k=P, v=P, tok_indptr=P, rows=4, **TABLE, **SHAPE, stream=None)
CHUNK = dict(q=P, o=P, lse=P, q_indptr=P, rows=4, **TABLE, prefix=None, slopes=None, batch=2,
             max_pages=8, hq=8, hkv=4, dim=128, page=16, layout=1, causal=1, window=0, cap=0.0,
             ws=P, ws_bytes=1 << 40, error=None, stream=None)
DECODE = dict(q=P, o=P, **TABLE, sel=P, stride=16, budget=256, budgets=None, ws=P,
              ws_bytes=1 << 40, batch=2, max_pages=8, hq=8, hkv=4, dim=128, page=16, layout=1,
              flags=0, stream=None)
CALLS = {"aoakv_append_kv_cache_fp8": APPEND, "aoakv_rope_append_kv_cache_fp8": ROPE,
         "aoakv_read_kv_cache_fp8": READ, "aoakv_chunk_attn_fp8": CHUNK,
         "aoakv_decode_sparse_attn_fp8": DECODE}

BAD = [(dict(dim=96), "head_dim"), (dict(page=0), "page_size"), (dict(page=33), "page_size"),
       (dict(layout=2), "layout"), (dict(hq=0), "num_(qo_)?heads"),
       (dict(hq=512), "num_(qo_)?heads"), (dict(hkv=0), "multiple|num_heads"),
       (dict(hkv=257), "num_heads|multiple"), (dict(batch=0), "batch_size"),
       (dict(batch=65536), "batch_size"), (dict(max_pages=0), "max_pages"),
       (dict(max_pages=1 << 30), "max_pages"), (dict(rows=1 << 31), "rows|tokens"),
       (dict(scale=0.0), "rope_scale"), (dict(scale=float("inf")), "rope_scale"),
       (dict(theta=-1.0), "rope_theta"), (dict(theta=float("nan")), "rope_theta"),
       (dict(window=1 << 31), "window"), (dict(cap=-1.0), "soft_cap"),
       (dict(stride=2), "sel_stride"), (dict(ws_bytes=64), "workspace"),
       (dict(flags=16), "flags"), (dict(flags=2), "flags"),
       *[({k: P + 8}, "16 bytes") for k in ("k", "v", "kv", "meta", "mean")],
       *[({k: None}, "null") for k in ("k", "v", "q", "o", "tok_indptr", "q_indptr", "kv", "exp",
                                       "indptr", "indices", "last")],
       *[({k: None}, "all given or all NULL") for k in STATS]]


@pytest.mark.parametrize("name,bad,says", [(n, b, s) for n in CALLS for b, s in BAD
                                           if set(b) <= set(CALLS[n]) and
                                           not (n == "aoakv_chunk_attn_fp8" and "ws_bytes" in b)],
                         ids=lambda x: str(x) if isinstance(x, dict) else "")
def test_c_entry_points(name, bad, says):
    rc, msg = call(name, *{**CALLS[name], **bad}.values())
    assert rc in (_lib.AOAKV_ERR_INVALID, _lib.AOAKV_ERR_UNSUPPORTED) and re.search(says, msg), msg


def test_c_more():
    """Alignment of q, memory that q shares, groups, a workspace for the decode."""
    for name in ("aoakv_rope_append_kv_cache_fp8", "aoakv_chunk_attn_fp8",
                 "aoakv_decode_sparse_attn_fp8"):
        rc, msg = call(name, *{**CALLS[name], "q": (P << 20) + 8}.values())
        assert rc == _lib.AOAKV_ERR_INVALID and "16 bytes" in msg
    for k in ("k", "v"):
        rc, msg = call("aoakv_rope_append_kv_cache_fp8", *{**ROPE, "q": P, k: P + 1024}.values())
        assert rc == _lib.AOAKV_ERR_INVALID and "shares memory" in msg
    for hq in (9, 12, 64):
        rc, msg = call("aoakv_decode_sparse_attn_fp8", *{**DECODE, "hq": hq}.values())
        assert rc in (_lib.AOAKV_ERR_INVALID, _lib.AOAKV_ERR_UNSUPPORTED) and \
            re.search("multiple|group", msg)
    rc, msg = call("aoakv_decode_sparse_attn_fp8", *{**DECODE, "ws": None}.values())
    assert rc == _lib.AOAKV_ERR_INVALID and "null" in msg
    # more workgroups than a dispatch counts
    rc, msg = call("aoakv_decode_sparse_attn_fp8",
                   *{**DECODE, "batch": 65535, "hq": 256, "hkv": 256, "ws_bytes": 1 << 60,
                     "sel": None}.values())
    assert rc == _lib.AOAKV_ERR_INVALID and "batch_size" in msg
    rc, msg = call("aoakv_append_kv_cache_fp8", *{**APPEND, "rows": 1 << 25, "page": 1}.values())
    assert rc == _lib.AOAKV_ERR_INVALID and "tokens" in msg


def test_no_rows_is_a_call():
    """A batch without a row: nothing is launched."""
    for name in CALLS:
        if "rows" in CALLS[name]:
            none = {k: None for k in ("q", "k", "v", "o") if k in CALLS[name]}
            assert call(name, *{**CALLS[name], "rows": 0, **none}.values())[0] == 0


# entry point -> its arguments, a tensor as its dtype
WRAPPED = {
    "append_kv_cache_fp8": [H, H, I, C, E, I, I, I, 1],
    "rope_append_kv_cache_fp8": [H, H, H, I, C, E, I, I, I, 1],
    "read_kv_cache_fp8": [4, I, C, E, I, I, I, 1],
    "chunk_attn_fp8": [H, I, C, E, I, I, I, 8, 1],
    "decode_sparse_attn_fp8": [H, H, C, E, I, I, I, None, 0, B, 8, 1],
}


@pytest.mark.parametrize("name", WRAPPED)
def test_types_and_devices(name):
    f = getattr(ops, name)
    args = [torch.zeros(4, dtype=x) if isinstance(x, torch.dtype) else x for x in WRAPPED[name]]
    with pytest.raises(ValueError, match="must be a device tensor"):
        f(*args)
    for i, x in enumerate(WRAPPED[name]):
        if x is (C if "append" in name or "read" in name else H):  # the tensor looked at first
            for bad, error, says in (("x", TypeError, "must be a torch.Tensor"),
                                     (torch.zeros(4, dtype=torch.float64), TypeError,
                                      "got torch.float64")):
                with pytest.raises(error, match=says):
                    f(*args[:i], bad, *args[i + 1:])
            break


def _valid(d="cuda:0"):
    z = lambda *s, dtype=H: torch.zeros(s, dtype=dtype, device=d)  # noqa: E731
    i = lambda *v: torch.tensor(v, dtype=I, device=d)  # noqa: E731
    table = dict(kv_data=z(4, 2, 2, 16, 64, dtype=B).view(C), kv_exp=z(4, 2, 2, dtype=E),
                 kv_indptr=i(0, 1, 2), kv_indices=i(0, 1), kv_last_page_len=i(16, 3), layout=1)
    stats = dict(metadata_data=z(2, 2, 2, 16, 64), metadata_indptr=i(0, 1, 2),
                 metadata_indices=i(0, 1), v_log_norm=z(4, 2), v_mean=z(4, 2, 64))
    rows = dict(k=z(5, 2, 64), v=z(5, 2, 64), token_indptr=i(0, 2, 5))
    return {
        "append_kv_cache_fp8": dict(rows, **table, **stats),
        "rope_append_kv_cache_fp8": dict(rows, q=z(5, 4, 64), **table, **stats),
        "read_kv_cache_fp8": dict(rows, num_tokens=5, **table),
        "chunk_attn_fp8": dict(q=z(5, 4, 64), q_indptr=i(0, 2, 5), max_pages=1, **table,
                               slopes=z(4, dtype=F), prefix_len=i(0, 1), o=z(5, 4, 64),
                               workspace=z(64, dtype=B)),
        "decode_sparse_attn_fp8": dict(q=z(2, 4, 64), o=z(2, 4, 64), sel_pages=z(2, 2, 3, dtype=I),
                                       token_budget=48, token_budgets=i(48, 48), max_pages=1,
                                       workspace=z(1 << 20, dtype=B), **table),
    }


SHAPES = {  # argument -> a shape that does not go with the others
    "q": (5, 4, 128), "q_indptr": (2,), "kv_data": (4, 2, 2, 16), "kv_exp": (4, 2, 3),
    "kv_indptr": (2,), "kv_last_page_len": (3,), "slopes": (3,), "prefix_len": (3,),
    "o": (4, 4, 64), "k": (5, 3, 64), "v": (4, 2, 64), "token_indptr": (2,),
    "metadata_data": (2, 2, 3, 16, 64), "metadata_indptr": (2,), "v_log_norm": (3, 2),
    "v_mean": (4, 2, 32), "workspace": (8,), "sel_pages": (2, 3, 3), "token_budgets": (3,),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", WRAPPED)
def test_every_argument(name):
    """A call that runs; then each argument in turn of a wrong shape, type or place."""
    f = getattr(ops, name)
    f(**_valid()[name])
    for k, t in _valid()[name].items():
        if isinstance(t, torch.Tensor):
            if k in SHAPES:
                bad = torch.zeros(SHAPES[k], dtype=B if t.dtype is C else t.dtype,
                                  device="cuda:0")
                with pytest.raises((ValueError, _lib.AoakvError)):
                    f(**dict(_valid()[name], **{k: bad.view(C) if t.dtype is C else bad}))
            with pytest.raises(ValueError, match="device tensor"):
                f(**dict(_valid()[name], **{k: t.cpu()}))
            with pytest.raises(TypeError, match="torch.float64"):
                f(**dict(_valid()[name], **{k: t.float().double()}))
            if t.dim() > 1:
                wide = torch.zeros(t.shape[:-1] + (2 * t.shape[-1],),
                                   dtype=B if t.dtype is C else t.dtype, device="cuda:0")
                wide = (wide.view(C) if t.dtype is C else wide)[..., ::2]
                with pytest.raises(ValueError, match="contiguous"):
                    f(**dict(_valid()[name], **{k: wide}))
        else:
            for bad in (-1, 2**32 + 1, 2**70):
                with pytest.raises((ValueError, _lib.AoakvError)):
                    f(**dict(_valid()[name], **{k: bad}))
    if "append" in name:
        for k in ("metadata_data", "metadata_indptr", "metadata_indices", "v_log_norm", "v_mean"):
            with pytest.raises(ValueError, match="all given or all None"):
                f(**dict(_valid()[name], **{k: None}))
    torch.cuda.synchronize()
