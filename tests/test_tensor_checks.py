"""CPU: the tensors that the serving operators are given are looked at before
their addresses are taken: type, device, layout and room.  A stand-in says what
a device tensor of its shape would; a call whose tensors are right comes as far
as its context, which is null here."""
import pytest

torch = pytest.importorskip("torch")

from quantibbler_amd import DecoderBlock, KernelError, KvCache
from quantibbler_amd.gpu import embed_dev, logprobs_dev, logprobs_workspace_size


class OnDevice:
    """A tensor's type, layout and device, without its memory."""

    is_cuda = True

    def __init__(self, meta, index=0):
        self.meta, self.index, self.device = meta, index, f"cuda:{index}"

    def __getattr__(self, name):
        return getattr(self.meta, name)

    def __getitem__(self, at):
        return OnDevice(self.meta[at], self.index)

    def get_device(self):
        return self.index

    def data_ptr(self):
        return 4096


def dev(*shape, dtype=torch.float32, index=0):
    return OnDevice(torch.empty(shape, dtype=dtype, device="meta"), index)


class Context:
    handle, device_index = None, 0


CTX = Context()


def refused(words, call, **kw):
    with pytest.raises(KernelError, match=words):
        call(**kw)


ROWS, VOCAB, TOP = 3, 9000, 4
NEED = logprobs_workspace_size(ROWS, VOCAB, TOP)


def logprobs(**kw):
    a = dict(logits=dev(ROWS, VOCAB), rows=ROWS, vocab=VOCAB, targets=dev(ROWS, dtype=torch.int32), logprobs=dev(ROWS),
             entropy=dev(ROWS), workspace=dev(NEED, dtype=torch.uint8), workspace_size=NEED, top_k=TOP,
             top_ids=dev(ROWS, TOP, dtype=torch.int32), top_logprobs=dev(ROWS, TOP))
    a.update(kw)
    logprobs_dev(CTX, **a)


def test_logprobs_takes_what_it_says():
    right = "null qbk_ctx"
    refused(right, logprobs)
    refused(right, logprobs, logits=dev(ROWS, VOCAB, dtype=torch.bfloat16), dtype="bfloat16")
    refused(right, logprobs, logits=dev(ROWS, 9011)[:, :VOCAB], row_stride=9011)
    refused(right, logprobs, logits=dev(ROWS, 9011), row_stride=9011)
    refused(right, logprobs, logits=dev(ROWS * VOCAB), targets=None, logprobs=None, entropy=None)
    refused(right, logprobs, logits=4096, targets=4096, logprobs=4096, workspace=4096, top_ids=4096, top_logprobs=4096)
    refused(right, logprobs, workspace=dev(NEED // 4 + 1))


@pytest.mark.parametrize("name,bad", [
    ("targets", dev(ROWS, dtype=torch.int64)), ("targets", dev(ROWS - 1, dtype=torch.int32)), ("targets", dev(ROWS)),
    ("targets", torch.zeros(ROWS, dtype=torch.int32)), ("targets", dev(ROWS, dtype=torch.int32, index=1)),
    ("targets", dev(ROWS, 2, dtype=torch.int32)[:, 0]),
    ("logits", dev(ROWS, VOCAB, dtype=torch.bfloat16)), ("logits", dev(ROWS, VOCAB, dtype=torch.float64)),
    ("logits", dev(ROWS, VOCAB - 1)), ("logits", dev(ROWS, 9011)[:, :VOCAB]), ("logits", dev(ROWS, VOCAB, index=1)),
    ("logits", torch.zeros(ROWS, VOCAB)), ("logits", torch.zeros(ROWS, VOCAB).numpy()), ("logits", "logits"),
    ("logprobs", dev(ROWS - 1)), ("logprobs", dev(ROWS, dtype=torch.float64)), ("logprobs", dev(2 * ROWS)[::2]),
    ("entropy", dev(ROWS, dtype=torch.bfloat16)), ("entropy", torch.zeros(ROWS)),
    ("top_ids", dev(ROWS, TOP, dtype=torch.int64)), ("top_ids", dev(ROWS, TOP - 1, dtype=torch.int32)),
    ("top_logprobs", dev(ROWS, TOP, dtype=torch.float16)), ("top_logprobs", dev(ROWS, TOP - 1)),
    ("workspace", dev(NEED - 1, dtype=torch.uint8)), ("workspace", torch.zeros(NEED, dtype=torch.uint8)),
    ("workspace", dev(NEED, dtype=torch.uint8, index=1))])
def test_logprobs_refuses_other_tensors(name, bad):
    refused(f"^{'' if name in ('targets', 'top_ids') else 'logprobs: '}{name} must be", logprobs, **{name: bad})


def test_logprobs_refuses_strides_past_the_memory():
    refused("logits must be", logprobs, logits=dev(ROWS, 9011)[:, 12:], vocab=VOCAB, row_stride=9012)
    refused("logits must be", logprobs, logits=dev(ROWS, VOCAB), row_stride=VOCAB + 1)
    refused("'float32' or 'bfloat16' logits, got 'float16'", logprobs, dtype="float16")


SEQS, CAP, KV, HD, HEADS, N, WIDE = 4, 100, 2, 64, 8, 12, 400


def make(ctx=CTX, index=0, fmt="int8", cap=CAP):
    size = KvCache.size(fmt, SEQS, cap, KV, HD)
    return KvCache(ctx, fmt, SEQS, cap, KV, HD, dev(size, dtype=torch.uint8, index=index))


def words(n):
    return dev(n, dtype=torch.int32)


def rows(name, **kw):
    a = dict(k=dev(N, KV, HD), v=dev(N, KV, HD), dtype="float32", pos=words(SEQS), n_rows=N)
    a.update(kw)
    getattr(make(), name)(**a)


@pytest.mark.parametrize("name", ["write_dev", "read_dev"])
def test_rows_are_what_they_are_said_to_be(name):
    right, wide = "null qbk_ctx", dev(N, WIDE)
    refused(right, rows, name=name)
    refused(right, rows, name=name, k=dev(N * KV * HD), v=dev(N + 5, KV * HD))
    refused(right, rows, name=name, k=4096, v=4096)
    refused(right, rows, name=name, k=wide[:, 3:131], v=wide[:, WIDE - 128:], row_stride=WIDE)
    refused(right, rows, name=name, k=wide[0, 3:131], v=wide[:, 131:], row_stride=WIDE)
    refused(right, rows, name=name, k=dev(1, WIDE)[:, :128], v=dev(1, 128), n_rows=1, n_seqs=1, row_stride=WIDE)
    for at in ("k", "v"):
        for bad in (dev(N, KV, HD, dtype=torch.bfloat16), dev(N, KV, HD, dtype=torch.float64), dev(N - 1, KV, HD),
                    dev(N, KV, HD, index=1), torch.zeros(N, KV, HD), torch.zeros(N, KV, HD).numpy(), wide[:, :128]):
            refused(f"kv cache: {'keys' if at == 'k' else 'values'} must be", rows, name=name, **{at: bad})
    refused("kv cache: values must be", rows, name=name, k=wide[:, :128], v=wide[:, WIDE - 127:], row_stride=WIDE)
    refused("kv cache: keys must be", rows, name=name, k=wide[1:, :128], v=wide[:, :128], row_stride=WIDE)
    refused("positions must be", rows, name=name, pos=dev(SEQS, dtype=torch.int32, index=1))
    refused("row starts must be", rows, name=name, row_start=words(SEQS))


def test_the_buffer_is_the_devices():
    size = KvCache.size("int8", SEQS, CAP, KV, HD)
    for bad in (dev(size, dtype=torch.uint8, index=1), torch.zeros(size, dtype=torch.uint8),
                torch.zeros(size, dtype=torch.uint8).numpy(), dev(2 * size, dtype=torch.uint8)[::2]):
        refused("kv cache buffer must be", KvCache, ctx=CTX, fmt="int8", n_seqs=SEQS, capacity=CAP, n_kv_heads=KV,
                head_dim=HD, buffer=bad)


def attend(cache=None, **kw):
    cache = cache or make()
    sq, plen = kw.get("seq_q", 1), kw.get("prefix_len", 0)
    need = cache.attention_workspace_size(HEADS, seq_q=sq, prefix_len=plen)
    a = dict(q=dev(SEQS, sq, HEADS, HD), dtype="float32", n_heads=HEADS, lens=words(SEQS), out=dev(SEQS, sq, HEADS, HD),
             workspace=dev(max(need, 16), dtype=torch.uint8), workspace_size=need)
    a.update(kw)
    cache.attention_dev(**a)


def test_attention_takes_what_it_says():
    right = "null qbk_ctx"
    refused(right, attend)
    refused(right, attend, seq_q=3, prefix=make(), prefix_len=90)
    refused(right, attend, q=dev(SEQS * HEADS * HD), out=4096)
    for at, what in (("q", "queries"), ("out", "out")):
        for bad in (dev(SEQS, 1, HEADS, HD, dtype=torch.bfloat16), dev(SEQS, 1, HEADS, HD - 1),
                    dev(SEQS, 1, HEADS, 2 * HD)[..., :HD], dev(SEQS, HEADS, HD, index=1), torch.zeros(SEQS, HEADS, HD)):
            refused(f"kv attention: {what} must be", attend, **{at: bad})
    need = make().attention_workspace_size(HEADS, seq_q=1, prefix_len=90)
    for bad in (dev(need - 1, dtype=torch.uint8), dev(need, dtype=torch.uint8, index=1),
                torch.zeros(need, dtype=torch.uint8)):
        refused("kv attention: workspace must be", attend, prefix=make(), prefix_len=90, workspace=bad)
    other = type("Other", (), {"handle": None, "device_index": 1})()
    refused("prefix's cache is on device 1, the sequences' on 0", attend, prefix=make(other, 1), prefix_len=90)


def test_a_blocks_step_takes_what_it_says():
    block = DecoderBlock.__new__(DecoderBlock)
    block.ctx, block._h, block.d_model = CTX, None, 256
    other = type("Other", (), {"handle": None, "device_index": 1})()

    def step(**kw):
        a = dict(h=dev(SEQS, 256), pos=words(SEQS), n=SEQS, cache=make(), workspace=dev(1000, dtype=torch.uint8),
                 workspace_size=1000)
        a.update(kw)
        block.decode_kv_dev(**a)

    refused("null argument", step)  # the block itself
    refused("kv decode: workspace must be", step, workspace=dev(999, dtype=torch.uint8))
    refused("kv decode: workspace must be", step, workspace=torch.zeros(1000, dtype=torch.uint8))
    refused("kv cache is on device 1, the block on 0", step, cache=make(other, 1))
    refused("prefix's cache is on device 1, the sequences' on 0", step, prefix=make(other, 1), prefix_len=3)
    refused("positions must be", step, pos=dev(SEQS, dtype=torch.int32, index=1))
    refused("batched decode input must be", step, h=dev(SEQS, 256, index=1))


def test_token_ids_are_32_bits():
    """What argmax of torch gives is 64 bits, and was read as pairs of ids."""
    def ids(tokens):
        embed_dev(CTX, 4096, VOCAB, 64, tokens, ROWS, 4096)

    refused("null qbk_ctx", ids, tokens=dev(ROWS, dtype=torch.int32))
    refused("null qbk_ctx", ids, tokens=4096)
    for bad in (dev(ROWS, dtype=torch.int64), dev(ROWS - 1, dtype=torch.int32), dev(ROWS),
                torch.zeros(ROWS, dtype=torch.int32), dev(ROWS, dtype=torch.int32, index=1)):
        refused("^token ids must be", ids, tokens=bad)
