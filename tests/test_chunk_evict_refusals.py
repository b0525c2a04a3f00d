"""What ops.chunk_attn, attn_weights, keep_tokens and compact_kv_cache and their C
entry points refuse, before anything is launched (no GPU needed)."""
import re

import pytest
import torch

from aoakv import _lib, ops

H, I, F, B = torch.float16, torch.int32, torch.float32, torch.uint8
P = 1 << 12  # an address that no call gets to


def call(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    return rc, lib.aoakv_last_error().decode()


CHUNK = dict(q=P, o=P, lse=P, q_indptr=P, rows=4, kv=P, indptr=P, indices=P, last=P, prefix=None,
             slopes=None, batch=2, max_pages=8, hq=8, hkv=4, dim=128, page=16, layout=1, causal=1,
             window=0, cap=0.0, ws=P, ws_bytes=1 << 40, error=None, stream=None)
WEIGHTS = dict(q=P, lse=P, q_indptr=P, start=None, weights=P, rows=4, kv=P, indptr=P, indices=P,
               last=P, prefix=None, slopes=None, batch=2, max_pages=8, hq=8, hkv=4, dim=128,
               page=16, layout=1, causal=1, window=0, cap=0.0, ws=P, ws_bytes=1 << 40, error=None,
               stream=None)
KEEP = dict(weights=P, indptr=P, indices=P, last=P, kept=P, stride=64, keep=64, sink=4, recent=4,
            batch=2, max_pages=8, hkv=4, page=16, error=None, stream=None)
COMPACT = dict(kept=P, stride=64, keep=64, kv=P, indptr=P, indices=P, last=P, new_indptr=P,
               new_indices=P, meta=P, md_indptr=P, md_indices=P, log_norm=P, mean=P, weights=None,
               batch=2, max_pages=8, hkv=4, dim=128, page=16, layout=1, error=None, stream=None)
CALLS = {"aoakv_chunk_attn": CHUNK, "aoakv_attn_weights": WEIGHTS, "aoakv_keep_tokens": KEEP,
         "aoakv_compact_kv_cache": COMPACT}

BAD = [(dict(dim=96), "head_dim"), (dict(page=0), "page_size"), (dict(page=33), "page_size"),
       (dict(layout=2), "layout"), (dict(hq=9), "multiple"), (dict(hkv=0), "multiple|num_heads"),
       (dict(hq=0), "num_heads"), (dict(hq=512), "num_heads"), (dict(hkv=257), "num_heads"),
       (dict(batch=0), "batch_size"), (dict(batch=65536), "batch_size"),
       (dict(max_pages=0), "max_pages"), (dict(max_pages=1 << 30), "max_pages"),
       (dict(window=1 << 31), "window"), (dict(cap=-1.0), "soft_cap"),
       (dict(cap=float("nan")), "soft_cap"), (dict(cap=float("inf")), "soft_cap"),
       (dict(cap=1025.0), "soft_cap"), (dict(cap=1e-7), "soft_cap"),
       (dict(rows=1 << 31), "rows"),
       *[({k: P + 8}, "16 bytes") for k in ("ws", "q", "o", "kv", "meta", "mean")],
       (dict(keep=0), "keep"), (dict(keep=65), "keep"), (dict(sink=40, recent=40), "sink"),
       (dict(new_indptr=None), "both"), (dict(new_indices=None), "both"),
       *[({k: None}, "null") for k in ("q", "q_indptr", "kv", "indptr", "indices", "last", "kept",
                                       "meta", "md_indptr", "md_indices", "log_norm", "mean")]]


@pytest.mark.parametrize("name,bad,says", [(n, b, s) for n in CALLS for b, s in BAD
                                           if set(b) <= set(CALLS[n])],
                         ids=lambda x: str(x) if isinstance(x, dict) else "")
def test_c_entry_points(name, bad, says):
    args = CALLS[name]
    if "hkv" in bad and bad["hkv"] == 257 and "hq" in args:
        bad = dict(bad, hq=257)
    rc, msg = call(name, *{**args, **bad}.values())
    assert rc in (_lib.AOAKV_ERR_INVALID, _lib.AOAKV_ERR_UNSUPPORTED) and re.search(says, msg), msg


def test_c_results_are_needed():
    assert call("aoakv_chunk_attn", *{**CHUNK, "o": None}.values())[0] == _lib.AOAKV_ERR_INVALID
    for k in ("lse", "weights"):
        rc, msg = call("aoakv_attn_weights", *{**WEIGHTS, k: None}.values())
        assert rc == _lib.AOAKV_ERR_INVALID and "null" in msg
    rc, msg = call("aoakv_keep_tokens", *{**KEEP, "weights": None}.values())
    assert rc == _lib.AOAKV_ERR_INVALID and "null" in msg


def test_no_rows_is_a_call():
    """A batch without a row has no attention to compute: nothing is launched."""
    assert call("aoakv_chunk_attn", *{**CHUNK, "rows": 0, "q": None, "o": None}.values())[0] == 0


# entry point -> its arguments, a tensor as its dtype
WRAPPED = {
    "chunk_attn": [H, I, H, I, I, I, 8, 1],
    "attn_weights": [H, F, I, F, H, I, I, I, 8, 1],
    "keep_tokens": [F, I, I, I, 64, I, 8],
    "compact_kv_cache": [I, 64, H, I, I, I, I, I, H, I, I, H, H, 8, 1],
}


def _args(spec, device="cpu"):
    return [torch.zeros(4, dtype=x, device=device) if isinstance(x, torch.dtype) else x
            for x in spec]


@pytest.mark.parametrize("name", WRAPPED)
def test_types_and_devices(name):
    f, spec = getattr(ops, name), WRAPPED[name]
    with pytest.raises(ValueError, match="must be a device tensor"):
        f(*_args(spec))
    first = spec.index(H) if name == "compact_kv_cache" else 0  # the tensor looked at first
    bad = _args(spec)
    bad[first] = "x"
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        f(*bad)
    bad[first] = torch.zeros(4, dtype=torch.float64)
    with pytest.raises(TypeError, match="got torch.float64"):
        f(*bad)


def _valid(d="cuda:0"):
    z = lambda *s, dtype=H: torch.zeros(s, dtype=dtype, device=d)
    i = lambda *v: torch.tensor(v, dtype=I, device=d)
    kv = z(4, 2, 2, 16, 64)
    table = (i(0, 1, 2), i(0, 1), i(16, 3))
    return {
        "chunk_attn": dict(q=z(5, 4, 64), q_indptr=i(0, 2, 5), kv_data=kv, kv_indptr=table[0],
                           kv_indices=table[1], kv_last_page_len=table[2], max_pages=1, layout=1,
                           slopes=z(4, dtype=F), prefix_len=i(0, 1), o=z(5, 4, 64),
                           workspace=z(64, dtype=B)),
        "attn_weights": dict(q=z(5, 4, 64), lse=z(5, 4, dtype=F), q_indptr=i(0, 2, 5),
                             weights=z(4, 2, 16, dtype=F), kv_data=kv, kv_indptr=table[0],
                             kv_indices=table[1], kv_last_page_len=table[2], max_pages=1,
                             layout=1, slopes=z(4, dtype=F), prefix_len=i(0, 1), start=i(0, 0),
                             workspace=z(64, dtype=B)),
        "keep_tokens": dict(weights=z(4, 2, 16, dtype=F), kv_indptr=table[0], kv_indices=table[1],
                            kv_last_page_len=table[2], keep=8, kept=z(2, 2, 8, dtype=I),
                            max_pages=1, workspace=z(64, dtype=B)),
        "compact_kv_cache": dict(kept=z(2, 2, 8, dtype=I), keep=8, kv_data=kv, kv_indptr=table[0],
                                 kv_indices=table[1], kv_last_page_len=table[2],
                                 new_indptr=i(0, 1, 2), new_indices=i(2, 3),
                                 metadata_data=z(2, 2, 2, 16, 64), metadata_indptr=i(0, 1, 2),
                                 metadata_indices=i(0, 1), v_log_norm=z(4, 2), v_mean=z(4, 2, 64),
                                 max_pages=1, layout=1, weights=z(4, 2, 16, dtype=F),
                                 workspace=z(64, dtype=B)),
    }


SHAPES = {  # argument -> a shape that does not go with the others
    "q": (5, 4, 128), "q_indptr": (2,), "kv_data": (4, 2, 2, 16), "kv_indptr": (2,),
    "kv_last_page_len": (3,), "slopes": (3,), "prefix_len": (3,), "o": (4, 4, 64), "lse": (5, 3),
    "weights": (4, 2, 8), "start": (1,), "kept": (2, 3, 8), "new_indptr": (2,),
    "metadata_data": (2, 2, 3, 16, 64), "metadata_indptr": (2,), "v_log_norm": (3, 2),
    "v_mean": (4, 2, 32), "workspace": (8,),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", WRAPPED)
def test_every_argument(name):
    """A call that runs; then each argument in turn of a wrong shape, type or
    place."""
    f = getattr(ops, name)
    f(**_valid()[name])
    for k, t in _valid()[name].items():
        if isinstance(t, torch.Tensor):
            if k in SHAPES and not (name == "keep_tokens" and k == "weights"):
                with pytest.raises((ValueError, _lib.AoakvError)):
                    f(**dict(_valid()[name], **{k: torch.zeros(SHAPES[k], dtype=t.dtype,
                                                               device="cuda:0")}))
            with pytest.raises(ValueError, match="device tensor"):
                f(**dict(_valid()[name], **{k: t.cpu()}))
            with pytest.raises(TypeError, match="torch.float64"):
                f(**dict(_valid()[name], **{k: t.double()}))
            if t.dim() > 1:
                wide = torch.zeros(t.shape[:-1] + (2 * t.shape[-1],), dtype=t.dtype,
                                   device="cuda:0")[..., ::2]
                with pytest.raises(ValueError, match="contiguous"):
                    f(**dict(_valid()[name], **{k: wide}))
        else:
            for bad in (-1, 2**32 + 1, 2**70):
                with pytest.raises((ValueError, _lib.AoakvError)):
                    f(**dict(_valid()[name], **{k: bad}))
    if name == "keep_tokens":
        for k in ("sink", "recent"):
            for bad in (-1, 9, 2**32):
                with pytest.raises((ValueError, _lib.AoakvError)):
                    f(**_valid()[name], **{k: bad})
    elif name != "compact_kv_cache":
        for bad in (-1, 2**31, 2**32):
            with pytest.raises((ValueError, _lib.AoakvError)):
                f(**_valid()[name], window=bad)
        with pytest.raises(_lib.AoakvError, match="soft_cap"):
            f(**_valid()[name], soft_cap=-2.0)
    torch.cuda.synchronize()
