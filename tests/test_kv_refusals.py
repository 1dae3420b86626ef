"""CPU: calls of the 8-bit KV cache, its attention and the log probabilities
that are refused before any device use: launches that cannot be, tensors that
are not what a call takes them for, devices that are not the context's."""
import ctypes as C

import pytest

from quantibbler_amd import KernelError
from quantibbler_amd._lib import KvShape, check, load

BUF = 0x1000  # never dereferenced: every call below is refused first, at the latest for its null context


def _err(rc, words):
    with pytest.raises(KernelError, match=words):
        check(rc)


def test_rows_of_nothing_are_bound_by_the_launch_too():
    """No own rows and no prefix: no workspace, and still one launch over all outputs."""
    lib, shape = load(), KvShape(0, 1 << 20, 16, 8, 16)

    def call(sq):
        return lib.qbk_attention_kv_dev(None, C.byref(shape), BUF, 0, 1 << 20, BUF, 0, None, None, 0, 0, 8, sq, BUF, 1, BUF,
                                        None, 0, None)

    _err(call(8), "too many query rows")
    _err(call(7), "null qbk_ctx")
