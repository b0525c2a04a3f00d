"""The kernels of chunks and eviction keep all their values in registers: where
the register allocator spilled some of the head dim 256 attention's, it left a
query's fourth dword in a register that nothing read.  Read from the metadata
(msgpack, in the code objects' notes) of the library as it is built."""
import struct
from pathlib import Path

import pytest

LIB = Path(__file__).resolve().parent.parent / "aoa-kv_amd" / "aoakv" / "libaoakv.so"
BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"
KERNELS = ("chunk_attn_kernel", "chunk_list_kernel", "chunk_join_kernel", "attn_weights_kernel",
           "weights_join_kernel", "keep_", "compact_")


def code_objects(data):
    """The gfx950 ELF images of the bundles in a host library."""
    at = data.find(BUNDLE)
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + len(BUNDLE))
        p = at + len(BUNDLE) + 8
        for _ in range(n):
            off, size, chars = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24:p + 24 + chars]
            p += 24 + chars
            if b"gfx950" in name and size:
                yield data[at + off:at + off + size]
        at = data.find(BUNDLE, p)


def kernels(elf):
    """The kernels' metadata: note type 32 of name AMDGPU."""
    msgpack = pytest.importorskip("msgpack")
    phoff, = struct.unpack_from("<Q", elf, 32)
    size, count = struct.unpack_from("<HH", elf, 54)
    for i in range(count):
        kind, = struct.unpack_from("<I", elf, phoff + i * size)
        if kind != 4:  # PT_NOTE
            continue
        off, = struct.unpack_from("<Q", elf, phoff + i * size + 8)
        length, = struct.unpack_from("<Q", elf, phoff + i * size + 32)
        p = off
        while p < off + length:
            ns, ds, note = struct.unpack_from("<III", elf, p)
            name, desc = p + 12, p + 12 + (ns + 3) // 4 * 4
            if note == 32 and elf[name:name + 6] == b"AMDGPU":
                yield from msgpack.unpackb(elf[desc:desc + ds])["amdhsa.kernels"]
            p = desc + (ds + 3) // 4 * 4


def test_no_vector_register_is_spilled():
    if not LIB.exists():
        pytest.skip("the library is not built")
    seen = {k: 0 for k in KERNELS}
    for elf in code_objects(LIB.read_bytes()):
        for k in kernels(elf):
            for name in KERNELS:
                if name in k[".name"]:
                    seen[name] += 1
                    assert k[".vgpr_spill_count"] == 0, k[".name"]
    assert all(seen.values()), seen
