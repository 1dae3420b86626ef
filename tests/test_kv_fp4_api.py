"""CPU: the 4-bit KV cache's sizes, and what its calls refuse before any device
use, as the 8-bit formats do."""
import ctypes as C

import pytest

from quantibbler_amd import KernelError, KvCache
from quantibbler_amd._lib import KvShape, check, load
from quantibbler_amd._lib import QBK_KV_FP4

BUF = 0x1000  # never dereferenced: every call below is refused first


@pytest.mark.parametrize("seqs,cap,kv,d,row", [(4, 100, 2, 64, 32 + 2 + 4), (1, 1, 1, 256, 128 + 8 + 4),
                                               (2, 65, 8, 128, 64 + 4 + 4)])
def test_sizes(seqs, cap, kv, d, row):
    assert KvCache.size("fp4", seqs, cap, kv, d) == seqs * kv * (-(-cap // 64) * 64) * 2 * row


def test_size_of_a_last_group_of_sixteen():
    # codes of 80 channels, values filled up to 96, three multipliers each
    assert KvCache.size("fp4", 1, 64, 1, 80) == 64 * (40 + 48 + 2 * 3 + 2 * 4)


@pytest.mark.parametrize("d", [0, 8, 24, 272])
def test_head_dims_that_are_refused(d):
    with pytest.raises(KernelError, match=f"multiple of 16 up to 256, got {d}"):
        KvCache.size("fp4", 1, 64, 1, d)


def test_formats_do_not_mix():
    shape, other = KvShape(QBK_KV_FP4, 4, 100, 2, 64), KvShape(0, 2, 50, 2, 64)
    args = (None, C.byref(shape), BUF, 0, 4, BUF, 100, C.byref(other), BUF, 0, 5, 4, 1, BUF, 1, BUF, BUF, 1 << 30, None)
    with pytest.raises(KernelError, match="must have the format"):
        check(load().qbk_attention_kv_dev(*args))


@pytest.mark.parametrize("fmt", [2, 3, 5, -1])
def test_other_formats(fmt):
    with pytest.raises(KernelError, match="format must be int8 .*fp4"):
        check(load().qbk_kv_cache_write_dev(None, C.byref(KvShape(fmt, 1, 8, 1, 64)), BUF, BUF, BUF, 1, 64, 1, None, BUF,
                                            0, 1, None))
