"""CPU: what the compiler reports of the registers of the library's own kernels.

Where a kernel's registers run out, a value of several registers may go partly to accumulation registers and partly to memory; the compiler
here has been seen to bring such a value back with a piece missing (a fragment of Q of the attention's form with two tiles of 256 channels in
8 bits, whose first tile came out wrong).  No kernel of the library is near that: those that use accumulation registers spill nothing."""
import struct

import pytest

from framefusion_amd import _lib

msgpack = pytest.importorskip("msgpack")
EM_AMDGPU, NT_AMDGPU_METADATA = 224, 32


def code_objects(blob):
    at = blob.find(b"\x7fELF", 4)
    while at >= 0:
        if blob[at + 4] == 2 and struct.unpack_from("<H", blob, at + 18)[0] == EM_AMDGPU:
            yield at
        at = blob.find(b"\x7fELF", at + 4)


def kernels():
    """The metadata of every kernel in the library file (ELF notes of its device code)."""
    _lib.load()
    blob = open(_lib.LIB_PATH, "rb").read()
    for base in code_objects(blob):
        phoff, = struct.unpack_from("<Q", blob, base + 32)
        phentsize, phnum = struct.unpack_from("<HH", blob, base + 54)
        for i in range(phnum):
            kind, _, offset, _, _, size = struct.unpack_from("<IIQQQQ", blob, base + phoff + i * phentsize)
            if kind != 4:                                                     # PT_NOTE
                continue
            at, end = base + offset, base + offset + size
            while at < end:
                namesz, descsz, ntype = struct.unpack_from("<III", blob, at)
                desc = at + 12 + (namesz + 3) // 4 * 4
                if ntype == NT_AMDGPU_METADATA:
                    yield from msgpack.unpackb(blob[desc:desc + descsz], strict_map_key=False)["amdhsa.kernels"]
                at = desc + (descsz + 3) // 4 * 4


def test_spilled_registers_go_to_memory_alone():
    found = {k[".name"]: k for k in kernels()}
    assert sum("k_cache_attention" in name for name in found) >= 2 * 24 and len(found) > 200
    for name, k in found.items():
        assert k[".vgpr_spill_count"] == 0 or k[".agpr_count"] == 0, (name, k[".vgpr_spill_count"], k[".agpr_count"])
        assert k[".vgpr_spill_count"] <= 8, (name, k[".vgpr_spill_count"])
