"""What the built library says of its kernels' registers (the metadata that the compiler writes beside them)."""
import struct

import pytest

import tensorrt_amd

msgpack = pytest.importorskip("msgpack")


def code_objects(data):
    """The gfx950 ELF files of the offload bundles in a library."""
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = data.find(magic)
    while at >= 0:
        pos = at + len(magic)
        (entries,) = struct.unpack_from("<Q", data, pos)
        pos += 8
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, pos)
            name = data[pos + 24:pos + 24 + length]
            pos += 24 + length
            if b"gfx950" in name and size:
                yield data[at + offset:at + offset + size]
        at = data.find(magic, pos)


def kernels(elf):
    """The kernels' metadata: the msgpack of the AMDGPU note."""
    assert elf[:5] == b"\x7fELF\x02"
    (headers,) = struct.unpack_from("<Q", elf, 0x20)
    size, count = struct.unpack_from("<HH", elf, 0x36)
    for i in range(count):
        kind, _, offset, _, _, length = struct.unpack_from("<IIQQQQ", elf, headers + i * size)
        pos = offset
        while kind == 4 and pos < offset + length:
            name, desc, note = struct.unpack_from("<III", elf, pos)
            at = pos + 12 + (name + 3) // 4 * 4
            if note == 32:
                yield from msgpack.unpackb(elf[at:at + desc])["amdhsa.kernels"]
            pos = at + (desc + 3) // 4 * 4


def test_no_linear_layer_spills():
    found = {}
    with open(tensorrt_amd.library_path(), "rb") as f:
        for elf in code_objects(f.read()):
            found.update((k[".name"], k) for k in kernels(elf))
    layers = [k for n, k in found.items() if "linear" in n or "dynamic_few" in n]
    assert len(layers) > 100
    spilling = {k[".name"]: k[".vgpr_spill_count"] for k in layers if k[".vgpr_spill_count"] or k[".private_segment_fixed_size"]}
    assert not spilling
