"""GPU: DeviceModel.score -- the log probabilities of a sequence's own tokens --
against float64 on the logits the model gives at each position."""
import os

import numpy as np
import pytest

from conftest import GOLDEN

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

EPS = 2.0 ** -24
IDS = [3, 17, 90, 90, 4, 127, 0, 55, 61, 2, 33]


@pytest.fixture(scope="module")
def ctx():
    from quantibbler_amd import GpuContext

    return GpuContext(0)


def check(logits, ids, got, top):
    """Logits (float64) of magnitude below 64: sums, differences and the exponentials' arguments are off by at most
    their roundings, 128 of 2^-24 of 64."""
    ref = torch.log_softmax(logits, -1)
    want = ref.gather(1, torch.tensor(ids[1:], device=ref.device)[:, None])[:, 0]
    tol = 128 * 64 * EPS
    assert float(logits.abs().max()) < 64
    assert float((got[0].double() - want).abs().max()) <= tol
    assert float((got[1].double() + (ref.exp() * ref).sum(-1)).abs().max()) <= tol
    if top:
        order = torch.argsort(logits, dim=-1, descending=True, stable=True)[:, :top]
        assert torch.equal(got[2].long(), order)
        assert float((got[3].double() - ref.gather(1, order)).abs().max()) <= tol


@pytest.mark.parametrize("serving", ["bf16", "fp32"])
@pytest.mark.parametrize("top", [0, 5])
def test_score_of_a_small_model(ctx, serving, top):
    """Token by token on the exact face: the logits are those of step(), bit for bit, so the score is theirs; and a
    model that has scored goes on from where the sequence ends."""
    from quantibbler_amd.model import DeviceModel, ModelDir

    md = ModelDir.load(os.path.join(GOLDEN, "parity_tiny"))
    m = DeviceModel(ctx, md, capacity=32, attention="exact", serving=serving)
    rows = torch.stack([m.step(t).clone() for t in IDS]).double()
    m.reset()
    m.SCORE_ROWS = 4  # more than one batch of rows, the last one short
    check(rows[:-1], IDS, m.score(IDS, top_k=top), top)
    assert m.pos == len(IDS)
    after = m.step(9).clone()
    m.reset()
    for t in IDS:
        m.step(t)
    assert torch.equal(after, m.step(9))
    m.close()


def test_score_on_a_stream_of_its_own(ctx):
    from quantibbler_amd.model import DeviceModel, ModelDir

    md = ModelDir.load(os.path.join(GOLDEN, "parity_tiny"))
    m = DeviceModel(ctx, md, capacity=32, attention="exact")
    want = m.score(IDS, top_k=3)
    s = torch.cuda.Stream()
    m.reset()
    got = m.score(IDS, stream=s, top_k=3)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    m.close()


def test_score_of_a_prompt_in_one_pass(ctx, orc):
    """The one-pass prefill: against the logits of the same rows, formed one at a time."""
    from test_gpu_trunk import synthetic_model

    from quantibbler_amd.gpu import rms_norm_dev
    from quantibbler_amd.model import DeviceModel

    md = synthetic_model(orc, 808)
    ids = np.random.default_rng(11).integers(0, md.vocab_size, 70).tolist()
    m = DeviceModel(ctx, md, capacity=128)
    got = m.score(ids, top_k=2)
    h, n, ws = m._prefill_rows(ids, None, 0)
    rows = []
    for i in range(n - 1):
        rms_norm_dev(ctx, h[i], 1, md.d_model, m.final_norm, md.rms_norm_eps, m.hn)
        m.head.logits_dev(m.hn, 1, m.logits)
        rows.append(m.logits.clone())
    check(torch.stack(rows).double(), ids, got, 2)
    m.close()


def test_score_refuses_what_it_cannot_score(ctx):
    from quantibbler_amd import KernelError
    from quantibbler_amd.model import DeviceModel, ModelDir

    md = ModelDir.load(os.path.join(GOLDEN, "parity_tiny"))
    m = DeviceModel(ctx, md, capacity=8, attention="exact")
    with pytest.raises(ValueError, match="at least two tokens, got 1"):
        m.score([5])
    with pytest.raises(KernelError, match="token id 128 is outside the vocabulary"):
        m.score([5, 128])
    with pytest.raises(KernelError, match="exceeds the block's cache capacity of 8"):
        m.score(list(range(9)))
    with pytest.raises(KernelError, match="top_k must be at most 64"):
        m.score([5, 6], top_k=65)
    m.close()
