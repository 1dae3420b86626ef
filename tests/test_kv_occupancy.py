"""CPU: how many waves a SIMD the built library's attention over the KV cache
leaves room for, from the notes that the compiler writes beside each kernel.

A SIMD has 512 registers a lane: 168 a wave are three waves, 256 two.  The body
of 16 rows for heads of up to 64 channels is built for three but for f32 queries
beside a prefix by 64 rows (at two, 512 sequences of 500 rows of fp8 heads took
52 us for 41), for heads of up to 128 for two; no vector register spills."""
import os
import re
import struct

import pytest

from conftest import ROOT

msgpack = pytest.importorskip("msgpack")


def kernels():
    """Name -> notes of every kernel in libqbk.so."""
    blob, out, at = open(os.path.join(ROOT, "quantibbler_amd", "libqbk.so"), "rb").read(), {}, 0
    while True:
        at = blob.find(b"AMDGPU\0\0", at + 1)
        if at < 0:
            return out
        name, size, kind = struct.unpack("<III", blob[at - 12:at])
        if name == 7 and kind == 32:
            notes = msgpack.unpackb(blob[at + 8:at + 8 + size], strict_map_key=False)
            out.update({k[".name"]: k for k in notes["amdhsa.kernels"]})


@pytest.fixture(scope="module")
def items():
    """(format, channels / 64, prefix by 64 rows, body of own rows, type of queries) -> notes of kva_items."""
    out = {}
    for name, notes in kernels().items():
        m = re.fullmatch(r"_ZN3qbk9kva_itemsILi(\d)ELi(\d)ELb(\d)ELi(\d)E([ft])EEvNS_9KvAttArgsE", name)
        if m:
            out[tuple(int(x) for x in m.groups()[:4]) + (m.group(5),)] = notes
    return out


def test_the_kernels_are_there(items):
    assert len([k for k in items if k[0] == 0]) == len([k for k in items if k[0] == 1]) == 18
    assert len([k for k in items if k[0] == 4]) >= 20


def test_no_vector_register_spills(items):
    for key, notes in items.items():
        assert notes[".vgpr_spill_count"] == 0, key


def test_waves_a_simd(items):
    """Vector registers in all, those of the matrix results among them."""
    for (fmt, dc, widep, own, t), notes in items.items():
        if dc == 4:
            continue
        three = dc == 1 and not (fmt != 4 and t == "f" and widep and own == 0)
        most = 168 if three else 256
        assert notes[".vgpr_count"] <= most, f"{(fmt, dc, widep, own, t)}: {notes['.vgpr_count']} registers for {most}"
