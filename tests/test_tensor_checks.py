"""CPU: the tensors that the serving operators are given are looked at before
their addresses are taken: type, device, layout and room.  A stand-in says what
a device tensor of its shape would; a call whose tensors are right comes as far
as its context, which is null here."""
import pytest

torch = pytest.importorskip("torch")

from quantibbler_amd import KernelError
from quantibbler_amd.gpu import logprobs_dev, logprobs_workspace_size


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
