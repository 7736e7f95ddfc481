"""Register spills of the built kernels, as the code objects in the library state them."""
import struct

import pytest

from nextou_amd import _lib

msgpack = pytest.importorskip("msgpack")
_BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"


def _metadata(elf):
    (table,), (count,) = struct.unpack_from("<Q", elf, 0x28), struct.unpack_from("<H", elf, 0x3C)
    for i in range(count):
        (kind,), (at, size) = struct.unpack_from("<I", elf, table + 64 * i + 4), struct.unpack_from("<QQ", elf, table + 64 * i + 24)
        end = at + size
        while kind == 7 and at < end:                      # notes
            name, desc, what = struct.unpack_from("<III", elf, at)
            at += 12 + (name + 3) // 4 * 4
            if what == 32:                                 # AMDGPU metadata
                yield msgpack.unpackb(elf[at:at + desc])
            at += (desc + 3) // 4 * 4


def _kernels():
    """{mangled name: bytes of scratch memory a lane}"""
    data = open(_lib.LIB_PATH, "rb").read()
    out, at = {}, data.find(_BUNDLE)
    while at >= 0:
        (entries,), p = struct.unpack_from("<Q", data, at + 24), at + 32
        for _ in range(entries):
            off, size, n = struct.unpack_from("<QQQ", data, p)
            if b"gfx950" in data[p + 24:p + 24 + n]:
                for meta in _metadata(data[at + off:at + off + size]):
                    out.update((k[".name"], k[".private_segment_fixed_size"]) for k in meta["amdhsa.kernels"])
            p += 24 + n
        at = data.find(_BUNDLE, at + 1)
    return out


def test_the_stationary_output_weight_gradients_do_not_spill():
    """Their loop reads a spilled register behind the slab's loads from memory, which doubles their time."""
    kernels = {name: size for name, size in _kernels().items() if "pw_wgrad_so_kernel" in name}
    assert len(kernels) == 8 and not any(kernels.values()), kernels
