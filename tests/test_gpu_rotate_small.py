"""GPU: heads so small that their mean square is a subnormal number, normed with
an eps of 0: values of ordinary size, by runs of channels and by pairs, against
float64.

Squares below 2^-126 are multiples of 2^-149, half a step off each, and so is
their mean; sums of multiples of 2^-149 below 2^-125 are exact.  So a mean square
m is off by 2^-149 at most, and its root's reciprocal by 2^-150 / m of itself,
besides what test_gpu_rotate allows."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import test_gpu_rotate as rot
from quantibbler_amd import GpuContext
from quantibbler_amd.gpu import Rope, rotate_heads_dev


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,rotary", [(128, 128), (64, 16), (128, 20), (16, 16), (256, 64)])
@pytest.mark.parametrize("size", [3e-21, 2e-20, 9e-20, 1e-10])
def test_heads_of_next_to_nothing(ctx, dtype, d, rotary, size, monkeypatch):
    monkeypatch.setattr(rot, "NORM_EPS", 0.0)
    rows, heads = 5, 3
    rng = np.random.default_rng(d + rotary)
    x = torch.from_numpy(size * rng.choice([-1.0, 1.0], (rows, heads, d)) * rng.uniform(0.7, 1.5, (rows, heads, d)))
    x = x.to(getattr(torch, dtype)).cuda()
    w = rng.uniform(0.5, 1.5, d).astype(np.float32)
    out = torch.empty_like(x)
    rotate_heads_dev(ctx, Rope(d, 10000.0, rotary_dim=rotary), x, None, dtype, rows, heads, 0, rot.words([3]), out, None,
                     q_norm=torch.from_numpy(w).cuda(), eps=0.0)
    torch.cuda.synchronize()
    old = x.double().cpu().numpy()
    want, tol = rot.reference(old, w, range(3, 3 + rows), 10000.0, rotary, False, None)
    least = (old * old).mean(-1).min()
    tol = tol + 2.0 ** -150 / least * 2 * np.abs(want).max()
    rot.check(out, want, tol)
