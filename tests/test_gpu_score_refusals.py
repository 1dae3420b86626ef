"""GPU: what DeviceModel.score refuses, it refuses before the sequence is
replaced: the model goes on as if it had not been asked."""
import os

import pytest

from conftest import GOLDEN

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from quantibbler_amd import GpuContext, KernelError


def test_a_refused_score_leaves_the_model_as_it_was():
    from quantibbler_amd.model import DeviceModel, ModelDir

    m = DeviceModel(GpuContext(0), ModelDir.load(os.path.join(GOLDEN, "parity_tiny")), capacity=16, attention="exact")
    for t in (5, 6, 7):
        m.step(t)
    want = m.step(9).clone()
    m.reset()
    for t in (5, 6, 7):
        m.step(t)
    for ids, kw in (([1, 2], {"top_k": 65}), ([1, 2], {"top_k": -1}), ([1], {}), ([], {}), ([1, 128], {}),
                    ([1, -1], {}), (list(range(17)), {}), ([1, 2], {"seq": 1}), ([1, 2], {"seq": -1})):
        with pytest.raises((ValueError, KernelError)):
            m.score(ids, **kw)
        assert m.pos == 3 and m.positions == [3]
    assert torch.equal(m.step(9), want)
    with pytest.raises(KernelError, match="top_k must be at most 64 and the vocabulary of 128, got 65"):
        m.score([1, 2], top_k=65)
    m.close()
