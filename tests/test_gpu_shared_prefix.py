"""GPU: share_prefix and step_shared against the oracle's trunk, which decodes
each request by itself behind the prompt on rows rounded as the cache rounds
them: the reference's gate for logits, which the meanings that this could be
mistaken for do not pass (test_oracle_shared_prefix)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import test_oracle_shared_prefix as meaning
from quantibbler_amd import GpuContext


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


@pytest.mark.parametrize("face", ["sage", "exact"])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_requests_behind_a_prompt_decode_as_by_themselves(ctx, orc, fmt, face):
    from quantibbler_amd.model import DeviceModel

    md, n = meaning.synthetic(orc), 3
    prompt, ids = meaning.tokens(md, n)
    want = [meaning.Requests(orc, md, prompt, face).logits(seq, fmt) for seq in ids]
    m = DeviceModel(ctx, md, capacity=meaning.PROMPT + meaning.STEPS, attention=face)
    m.share_prefix(prompt, n, meaning.STEPS, fmt=fmt)
    for step in range(meaning.STEPS):
        got = m.step_shared([seq[step] for seq in ids]).cpu().numpy().astype(np.float64)
        for i in range(n):
            a, b = got[i], want[i][step]
            assert meaning.apart(a, b) <= 0.02 and a @ b >= 0.999 * np.linalg.norm(a) * np.linalg.norm(b), \
                f"request {i}, step {step}: {meaning.apart(a, b):.4f} apart"
    m.close()
