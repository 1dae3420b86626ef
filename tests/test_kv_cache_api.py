"""CPU: the 8-bit KV cache, its attention and the log probabilities refuse bad
calls before any device use, with the library's own error type and words."""
import ctypes as C

import pytest

from quantibbler_amd import KernelError, KvCache
from quantibbler_amd._lib import KvShape, check, load
from quantibbler_amd.gpu import logprobs_workspace_size


def _err(rc, words):
    with pytest.raises(KernelError, match=words):
        check(rc)


SHAPE = KvShape(0, 4, 100, 2, 64)
BUF = 0x1000  # never dereferenced: every call below is refused first


def test_sizes():
    # 100 rows round up to 128; key and value codes and one f32 scale each
    assert KvCache.size("int8", 4, 100, 2, 64) == 4 * 128 * 2 * 2 * (64 + 4)
    assert KvCache.size("fp8", 1, 1, 1, 256) == 64 * 2 * 260
    assert logprobs_workspace_size(0, 10, 3) == 0
    assert logprobs_workspace_size(3, 8193, 5) >= 3 * 2 * (16 + 8 * 5)


@pytest.mark.parametrize("args,words", [
    (("int4", 1, 8, 1, 64), "format must be one of"),
    (("int8", 0, 8, 1, 64), "non-empty"),
    (("int8", 1, 0, 1, 64), "non-empty"),
    (("int8", 1, 8, 1, 72), "multiple of 16 up to 256, got 72"),
    (("int8", 1, 8, 1, 272), "multiple of 16 up to 256, got 272"),
    (("int8", 1, 8, 1, 0), "multiple of 16 up to 256, got 0"),
    (("int8", 1, 1 << 31, 1, 64), "below 2\\^31"),
    (("int8", 1, 8, (1 << 16) + 1, 64), "heads must be at most 65536"),
    (("int8", 1 << 20, 1 << 20, 64, 64), "2\\^48"),
    (("int8", -1, 8, 1, 64), "negative"),
])
def test_shape_refusals(args, words):
    with pytest.raises(KernelError, match=words):
        KvCache.size(*args)


def test_small_buffer_is_refused():
    import numpy as np

    with pytest.raises(KernelError, match="smaller than the"):
        KvCache(None, "int8", 1, 64, 1, 64, np.zeros(64 * 2 * 68 - 1, np.uint8))


@pytest.mark.parametrize("name", ["qbk_kv_cache_write_dev", "qbk_kv_cache_read_dev"])
def test_row_refusals(name):
    fn = getattr(load(), name)

    def call(shape=SHAPE, cache=BUF, k=BUF, v=BUF, dtype=1, stride=128, rows=4, start=None, pos=BUF, first=0, n=4):
        return fn(None, C.byref(shape), cache, k, v, dtype, stride, rows, start, pos, first, n, None)

    _err(call(shape=KvShape(2, 4, 100, 2, 64)), "format must be int8")
    _err(call(dtype=0), "float32 or bfloat16")
    _err(call(first=1), "sequences 1 .. 5 of a kv cache holding 4")
    _err(call(first=5, n=0, rows=0), "sequences 5 .. 5")
    _err(call(first=2 ** 64 - 1, n=2), "of a kv cache holding 4")
    _err(call(stride=127), "row_stride 127 is smaller than a row of 128")
    _err(call(rows=6), "6 rows do not split evenly over 4")
    _err(call(n=0), "rows for no sequence")
    _err(call(rows=2 ** 32, n=1), "too many rows")
    _err(call(stride=1 << 41), "too many rows")
    for hole in ("cache", "k", "v", "pos"):
        _err(call(**{hole: None}), "null argument")
    _err(call(cache=BUF + 8), "16-byte aligned")
    _err(call(), "null qbk_ctx")
    assert call(rows=0, k=None, v=None, pos=None) == 0  # nothing to do


def test_attention_refusals():
    lib = load()
    other = KvShape(0, 2, 50, 2, 64)

    def call(shape=SHAPE, cache=BUF, first=0, n=4, lens=BUF, most=100, pshape=None, prefix=None, pseq=0, plen=0, heads=4,
             sq=1, q=BUF, dtype=1, out=BUF, ws=BUF, size=1 << 30):
        return lib.qbk_attention_kv_dev(None, C.byref(shape), cache, first, n, lens, most,
                                        None if pshape is None else C.byref(pshape), prefix, pseq, plen, heads, sq, q,
                                        dtype, out, ws, size, None)

    _err(call(shape=KvShape(7, 4, 100, 2, 64)), "format must be int8")
    _err(call(heads=5), "n_kv_heads must divide n_heads: n_heads=5, n_kv_heads=2")
    _err(call(heads=0), "n_kv_heads must divide n_heads")
    _err(call(heads=8194), "up to 8192 heads")
    _err(call(sq=0), "at least one query")
    _err(call(most=101), "max_len 101 is past the kv cache's capacity of 100")
    _err(call(dtype=0), "float32 or bfloat16 queries")
    _err(call(first=3, n=2), "sequences 3 .. 5 of a kv cache holding 4")
    _err(call(plen=5), "null shape")
    _err(call(plen=5, pshape=KvShape(1, 2, 50, 2, 64), prefix=BUF), "must have the format")
    _err(call(plen=5, pshape=KvShape(0, 2, 50, 1, 64), prefix=BUF), "must have the format")
    _err(call(plen=5, pshape=KvShape(0, 2, 50, 2, 128), prefix=BUF), "must have the format")
    _err(call(plen=51, pshape=other, prefix=BUF), "prefix of 51 rows of sequence 0")
    _err(call(plen=5, pseq=2, pshape=other, prefix=BUF), "of sequence 2 in a kv cache of 2 sequences")
    _err(call(plen=5, pshape=other), "null argument")
    for hole in ("cache", "lens", "q", "out"):
        _err(call(**{hole: None}), "null argument")
    _err(call(cache=BUF + 4), "kv cache buffer must be 16-byte aligned")
    _err(call(plen=5, pshape=other, prefix=BUF + 4), "kv cache buffer must be 16-byte aligned")
    _err(call(n=4, sq=1 << 40), "too many query rows")
    need = lib.qbk_attention_kv_workspace_size(C.byref(SHAPE), 4, 4, 1, 100, 50)
    assert need > 0
    _err(call(plen=50, pshape=other, prefix=BUF, size=need - 1), f"smaller than the {need} needed")
    _err(call(plen=50, pshape=other, prefix=BUF, ws=None), f"workspace of 0 bytes is smaller than the {need}")
    _err(call(plen=50, pshape=other, prefix=BUF, ws=BUF + 8), "workspace must be 16-byte aligned")
    _err(call(), "null qbk_ctx")
    assert call(n=0, q=None, out=None, lens=None) == 0
    assert lib.qbk_attention_kv_workspace_size(C.byref(SHAPE), 4, 0, 1, 100, 50) == 0
    assert lib.qbk_attention_kv_workspace_size(C.byref(SHAPE), 3, 4, 1, 100, 50) == 0


def test_attention_words_need_not_be_on_the_host():
    """The Python face refuses host lengths, positions and row starts."""
    import torch

    cache = KvCache.__new__(KvCache)
    cache.n_seqs, cache.capacity, cache.n_kv_heads, cache.head_dim = 2, 8, 1, 16
    cache.buffer, cache._shape = BUF, KvShape(0, 2, 8, 1, 16)
    cache._shape_ref, cache._base, cache.ctx = C.byref(cache._shape), BUF, None
    host = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(KernelError, match="lengths must be a contiguous 32-bit device tensor"):
        cache.attention_dev(BUF, "float32", 1, host, BUF, BUF, 1 << 20)
    with pytest.raises(KernelError, match="positions must be"):
        cache.write_dev(BUF, BUF, "float32", host, 2)
    with pytest.raises(KernelError, match="row starts must be"):
        cache.read_dev(BUF, BUF, "float32", BUF, 2, row_start=host)
    with pytest.raises(KernelError, match="must not be negative"):
        cache.attention_dev(BUF, "float32", 1, BUF, BUF, BUF, 1 << 20, max_len=-1)
    with pytest.raises(KernelError, match="needs the cache that holds the prefix"):
        cache.attention_dev(BUF, "float32", 1, BUF, BUF, BUF, 1 << 20, prefix_len=3)
    with pytest.raises(KernelError, match="'float32' or 'bfloat16' queries, got 'float64'"):
        cache.attention_dev(BUF, "float64", 1, BUF, BUF, BUF, 1 << 20)


def test_logprobs_refusals():
    lib = load()

    def call(x=BUF, dtype=1, rows=2, vocab=100, stride=100, targets=BUF, logp=BUF, ent=BUF, top=3, ids=BUF, tops=BUF,
             ws=BUF, size=1 << 20):
        return lib.qbk_logprobs_dev(None, x, dtype, rows, vocab, stride, targets, logp, ent, top, ids, tops, ws, size,
                                    None)

    _err(call(vocab=0), "1 <= vocab")
    _err(call(vocab=1 << 31), "1 <= vocab")
    _err(call(top=65), "top_k must be at most 64")
    _err(call(vocab=2, stride=2), "top_k must be at most 64 and the vocabulary of 2, got 3")
    _err(call(rows=1 << 31), "too many rows")
    _err(call(dtype=0), "float32 or bfloat16 logits")
    _err(call(stride=99), "row_stride 99 does not fit rows of 100")
    _err(call(targets=None), "come together")
    _err(call(logp=None), "come together")
    _err(call(ids=None), "needs top_ids and top_logprobs")
    _err(call(tops=None), "needs top_ids and top_logprobs")
    _err(call(x=None), "null argument")
    need = lib.qbk_logprobs_workspace_size(2, 10000, 3)
    wide = dict(vocab=10000, stride=10000)
    _err(call(size=need - 1, **wide), f"smaller than the {need} needed")
    _err(call(ws=None, **wide), "workspace of 0 bytes")
    _err(call(ws=BUF + 8, **wide), "16-byte aligned")
    assert lib.qbk_logprobs_workspace_size(2, 100, 3) == 0  # short rows need none
    _err(call(), "null qbk_ctx")
    assert call(rows=0, x=None, ws=None, size=0) == 0
