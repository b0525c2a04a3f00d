"""The kernels of the 8-bit cache keep all their values in vector registers, as those of
the chunk attention do (test_chunk_registers.py says why), by the built library's metadata."""
import pytest

from test_chunk_registers import LIB, code_objects, kernels

KERNELS = ("append_fp8_kernel", "read_fp8_kernel", "decode_fp8_kernel")


def test_no_vector_register_is_spilled():
    if not LIB.exists():
        pytest.skip("the library is not built")
    seen = {k: 0 for k in KERNELS}
    chunk = 0
    for elf in code_objects(LIB.read_bytes()):
        for k in kernels(elf):
            for name in KERNELS:
                if name in k[".name"]:
                    seen[name] += 1
                    assert k[".vgpr_spill_count"] == 0, k[".name"]
                    assert k[".private_segment_fixed_size"] == 0, k[".name"]
            # the attention over codes: its last template argument
            chunk += "chunk_attn_kernel" in k[".name"] and "ELb1EEE" in k[".name"]
    assert all(seen.values()) and chunk, (seen, chunk)
