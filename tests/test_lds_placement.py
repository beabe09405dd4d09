"""Where kernels with dynamic LDS have it: right after the static LDS whose size the built library's metadata gives."""

from __future__ import annotations

import struct

import pytest

msgpack = pytest.importorskip("msgpack")


def _code_objects(data: bytes):
    """The gfx950 ELF images in the library's offload bundles."""

    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = data.find(magic)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(magic))
        entry = at + len(magic) + 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            if size and b"gfx950" in data[entry + 24:entry + 24 + length]:
                yield data[at + offset:at + offset + size]
            entry += 24 + length
        at = data.find(magic, at + len(magic))


def _kernels(elf: bytes):
    """The kernels' metadata from an image's note segments (note type 32, msgpack)."""

    table, = struct.unpack_from("<Q", elf, 32)
    size, count = struct.unpack_from("<HH", elf, 54)
    for header in range(table, table + size * count, size):
        if struct.unpack_from("<I", elf, header)[0] != 4:
            continue
        at, = struct.unpack_from("<Q", elf, header + 8)
        end = at + struct.unpack_from("<Q", elf, header + 32)[0]
        while at < end:
            names, length, kind = struct.unpack_from("<III", elf, at)
            start = at + 12 + (names + 3) // 4 * 4
            if kind == 32:
                yield from msgpack.unpackb(elf[start:start + length])["amdhsa.kernels"]
            at = start + (length + 3) // 4 * 4


def test_rows_kept_in_lds_are_aligned():
    """The distillation keeps 16-byte runs of a row at the start of its dynamic LDS."""

    from qste_amd.kernels import _lib

    sizes = {k[".name"]: k[".group_segment_fixed_size"]
             for image in _code_objects(_lib.LIB_PATH.read_bytes()) for k in _kernels(image)
             if "7distill14forward_kernel" in k[".name"]}
    assert sizes
    assert {name: size for name, size in sizes.items() if size % 16} == {}
