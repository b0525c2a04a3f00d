"""The attention kernels of the 8-bit cache leave room for the workgroups per CU that their
launches count on, by the built library's metadata: of the 512 registers of a lane on each of
a CU's 4 SIMDs, and of its 160 KB of LDS."""
import re

import pytest

from test_chunk_registers import LIB, code_objects, kernels

SIMDS, REGISTERS, STEP, LDS = 4, 512, 8, 160 * 1024


def workgroups(k):
    """Workgroups of kernel k that a CU holds."""
    waves = k[".max_flat_workgroup_size"] // 64 // SIMDS  # of a workgroup per SIMD
    registers = -(-k[".vgpr_count"] // STEP) * STEP
    return min(REGISTERS // registers // waves, LDS // max(1, k[".group_segment_fixed_size"]))


def test_workgroups_per_cu():
    if not LIB.exists():
        pytest.skip("the library is not built")
    seen = {}
    for elf in code_objects(LIB.read_bytes()):
        for k in kernels(elf):
            m = re.search(r"(chunk_attn|decode_fp8)_kernelILi(\d+)E(.*)", k[".name"])
            if m is None or m[1] == "chunk_attn" and "ELb1EEE" not in k[".name"]:
                continue
            assert k[".vgpr_count"] >= k[".agpr_count"]  # (one file: all of a lane's registers)
            want = 2 if m[1] == "chunk_attn" and m[2] != "256" else 1
            assert workgroups(k) >= want, (k[".name"], k[".vgpr_count"])
            seen[m[1], int(m[2])] = seen.get((m[1], int(m[2])), 0) + 1
    dims = (64, 128, 256)
    # 4 scores, page kinds and both forms; runs of 16, 4 and 1 tokens per page
    assert seen == {**{("chunk_attn", d): 16 for d in dims}, **{("decode_fp8", d): 3 for d in dims}}
