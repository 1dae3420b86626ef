"""CPU: whose memory a model's calls on a stream of their own work in.  The
device's calls are stand-ins that note what was asked for and when; torch's
allocations note the stream whose pool they come from.  Memory of another
stream's pool may still be read and written by that stream's work when it is
handed out, and may be handed out again there while this stream's work is
under way."""
import contextlib

import pytest

torch = pytest.importorskip("torch")

from quantibbler_amd import gpu, model

CURRENT = "the caller's current stream"


class Memory:
    """What a call does with a device tensor, without one."""

    dtype = torch.uint8

    def __init__(self, size):
        self.size = size

    def __getitem__(self, at):
        return self

    def data_ptr(self):
        return 4096

    def element_size(self):
        return 4

    def numel(self):
        return 1 << 40

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True


class Stream:
    cuda_stream = 77

    def synchronize(self):
        pass


class Block:
    def __init__(self, log):
        self.log = log

    def prefill_workspace_size(self, n):
        return 1000

    def prefill_seq_dev(self, seq, h, n, ws, need, stream):
        self.log.append(("work", stream))

    def cache_ptrs(self):
        return 4096, 4096

    def decode_kv_workspace_size(self, *a, **kw):
        return 1000

    def decode_batch_workspace_size(self, n):
        return 1000

    def decode_batch_dev(self, h, pos, ws, need, stream):
        self.log.append(("work", stream))

    def reset(self):
        pass


@pytest.fixture
def small(monkeypatch):
    """A model of two blocks, its log, and the stream that its calls run on."""
    log, stream, now = [], Stream(), [CURRENT]

    def allocate(*a, **kw):
        log.append(("memory", now[-1]))
        return Memory(a)

    @contextlib.contextmanager
    def on(s):
        now.append(s)
        yield
        now.pop()

    for name in ("empty", "zeros"):
        monkeypatch.setattr(torch, name, allocate)
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: log.append(("wait", "everything")))
    for name in ("embed", "embed_dev", "rms_norm_dev"):
        monkeypatch.setattr(gpu, name, lambda *a, **kw: log.append(("work", stream)))
    monkeypatch.setattr(gpu.KvCache, "write_dev", lambda *a, **kw: log.append(("work", kw["stream"])))
    m = model.DeviceModel.__new__(model.DeviceModel)
    m.ctx = type("Context", (), {"device_index": 0})()
    m.md = type("Sizes", (), dict(vocab_size=100, d_model=64, n_kv_heads=2, head_dim=32, n_heads=2, rms_norm_eps=1e-5))()
    m.blocks, m.head = [Block(log), Block(log)], type("Head", (), {"logits_dev": lambda *a: None})()
    m.capacity, m.serving, m.n_seqs, m.positions, m.pos, m._shared, m._batch = 100, "bf16", 4, [0] * 4, 0, None, {}
    m.embedding = m.final_norm = m.hn = m.logits = Memory(1)
    return m, log, stream


def pools(log):
    return {where for what, where in log if what == "memory"}


def test_memory_is_of_the_stream_that_works_in_it(small):
    m, log, stream = small
    m.prefill([1, 2, 3], stream=stream)
    assert pools(log) == {stream}
    log.clear()
    m.share_prefix([1, 2, 3], 4, 20, stream=stream)
    assert len([x for x in log if x[0] == "memory"]) > 8 and pools(log) == {stream}
    log.clear()
    m.step_batch([1, 2], stream=stream)
    assert pools(log) == {stream}


def test_steps_under_way_are_waited_for_before_their_memory_goes(small):
    m, log, stream = small
    m.share_prefix([1, 2, 3], 4, 20, stream=stream)
    assert ("wait", "everything") not in log
    log.clear()
    first = m._shared
    m.share_prefix([1, 2, 3], 4, 20, stream=stream)
    assert ("wait", "everything") in log and m._shared is not first
    log.clear()
    m.reset()
    assert log == [("wait", "everything")] and m._shared is None
    m.reset()
    assert len(log) == 1
