"""What the compiler made of the feature operators' kernels, from the code objects in the built library."""
import struct

import pytest


msgpack = pytest.importorskip("msgpack")


def kernels(path):
    """The metadata of every kernel: .name, .vgpr_count, .vgpr_spill_count, ..."""
    blob, magic, at = open(path, "rb").read(), b"__CLANG_OFFLOAD_BUNDLE__", -1
    while (at := blob.find(magic, at + 1)) >= 0:
        p = at + len(magic)
        count, = struct.unpack_from("<Q", blob, p)
        p += 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", blob, p)
            target, p = blob[p + 24:p + 24 + length], p + 24 + length
            elf = blob[at + offset:at + offset + size]
            if b"gfx950" in target and elf[:4] == b"\x7fELF":
                yield from notes(elf)


def notes(elf):
    table, = struct.unpack_from("<Q", elf, 0x20)
    size, count = struct.unpack_from("<HH", elf, 0x36)
    for i in range(count):
        kind, _, start, _, _, length = struct.unpack_from("<IIQQQQ", elf, table + i * size)
        if kind != 4:  # PT_NOTE
            continue
        p = start
        while p < start + length:
            name, desc, what = struct.unpack_from("<III", elf, p)
            body = p + 12 + (name + 3) // 4 * 4
            if what == 32 and elf[p + 12:p + 12 + name].rstrip(b"\0") == b"AMDGPU":
                yield from msgpack.unpackb(elf[body:body + desc], raw=False)["amdhsa.kernels"]
            p = body + (desc + 3) // 4 * 4


def test_no_vector_register_is_spilled(hip_library):
    """A register that is spilled in the tiles or in the rows that lanes hold is written to memory and read back where registers were counted on."""
    ours = {k[".name"]: k for k in kernels(hip_library) if any(n in k[".name"] for n in ("linear_", "preference_", "dropout_kernel", "pack_kernel"))}
    assert len(ours) > 40
    assert not {n: k[".vgpr_spill_count"] for n, k in ours.items() if k[".vgpr_spill_count"]}
