"""The prefill's matrix kernels hold the same 128-bit fragments as the chunk
attention's, one of whose spilled ones lost a dword: they spill none either."""
import pytest

from test_chunk_registers import LIB, code_objects, kernels


def test_no_vector_register_is_spilled():
    if not LIB.exists():
        pytest.skip("the library is not built")
    seen = 0
    for elf in code_objects(LIB.read_bytes()):
        for k in kernels(elf):
            if "prefill_kernelILi" in k[".name"] or "prefill_merge_kernel" in k[".name"]:
                seen += 1
                assert k[".vgpr_spill_count"] == 0, k[".name"]
    assert seen >= 21, seen
