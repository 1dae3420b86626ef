"""CPU: the largest calls of the 8-bit KV cache, its attention and the log
probabilities: what one launch cannot hold is refused before any device use."""
import ctypes as C

import pytest

from quantibbler_amd import KernelError
from quantibbler_amd._lib import KvShape, check, load

BUF = 0x1000  # never dereferenced: every call below is refused first


def _err(rc, words):
    with pytest.raises(KernelError, match=words):
        check(rc)


def test_launches_of_more_than_two_to_the_32_threads():
    """What no grid of 256 threads a workgroup can hold is refused, not left to the launch."""
    lib = load()
    rows = getattr(lib, "qbk_kv_cache_write_dev")
    many = KvShape(0, 1 << 23, 16, 64, 16)  # by rows: three a sequence, four rows and heads a workgroup
    _err(rows(None, C.byref(many), BUF, BUF, BUF, 1, 1024, 3 << 23, None, BUF, 0, 1 << 23, None), "too many rows")
    one = KvShape(0, 1, 1 << 30, 64, 16)  # by tiles: 64 rows of a head a workgroup
    _err(rows(None, C.byref(one), BUF, BUF, BUF, 1, 1024, 1 << 28, None, BUF, 0, 1, None), "too many rows")
    x = lib.qbk_logprobs_dev
    _err(x(None, BUF, 1, 1 << 24, 100, 100, BUF, BUF, BUF, 0, None, None, BUF, 1 << 40, None), "too many rows")
    _err(x(None, BUF, 1, 1 << 20, 1 << 17, 1 << 17, BUF, BUF, BUF, 0, None, None, BUF, 1 << 40, None), "too many rows")
    seqs = KvShape(0, 1 << 22, 16, 8, 16)
    _err(lib.qbk_attention_kv_dev(None, C.byref(seqs), BUF, 0, 1 << 22, BUF, 16, None, None, 0, 0, 8, 1, BUF, 1, BUF, BUF,
                                  1 << 40, None), "too many query rows")
    assert lib.qbk_attention_kv_workspace_size(C.byref(seqs), 8, 1 << 22, 1, 16, 0) == 0
    long = KvShape(0, 1, 1 << 20, 8, 16)  # few items, whose partial rows the join would take four a workgroup
    _err(lib.qbk_attention_kv_dev(None, C.byref(long), BUF, 0, 1, BUF, 1 << 20, C.byref(long), BUF, 0, 1 << 20, 8, 1 << 23,
                                  BUF, 1, BUF, BUF, 1 << 62, None), "too many query rows")
