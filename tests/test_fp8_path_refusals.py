"""What the controller, the shim and the latency driver take and refuse of a cache held in
8 bits (CPU: nothing is launched)."""
import pytest
import torch


def test_cache_types():
    from aoakv.utils import InferenceController
    for bad in (torch.float32, torch.int8, torch.float8_e5m2):
        with pytest.raises(TypeError, match="kv_dtype"):
            InferenceController(1, 4, 64, 16, 4, 100, torch.float16, "cpu", kv_dtype=bad)
    with pytest.raises(TypeError, match="float16"):
        InferenceController(1, 4, 64, 16, 4, 100, torch.float8_e4m3fn, "cpu")


def test_latency_flag():
    from aoakv import latency
    assert latency.parse_args([]).kv_dtype == "fp16"
    assert latency.parse_args(["--kv_dtype", "fp8", "--graph"]).kv_dtype == "fp8"
    with pytest.raises(SystemExit):
        latency.parse_args(["--kv_dtype", "int4"])


def test_no_eviction_in_the_shim():
    from aoakv.shim import LlamaShape, QuestLlamaModel
    m = QuestLlamaModel(LlamaShape(256, 4, 4, 1, 256))
    with pytest.raises(ValueError, match="fp16"):
        m.quest_init(16, 100, evict_keep=64, device="cpu", kv_dtype=torch.float8_e4m3fn)
