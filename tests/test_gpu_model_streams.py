"""GPU: a model's calls on a stream of their own, while the current stream
allocates, fills and frees memory of the sizes that they use: the results are
those of the default stream, bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from quantibbler_amd import GpuContext


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


def stir(md, n):
    """Memory of the current stream's pool taken, filled and given back: rows, workspaces, positions, caches."""
    for size in (n * md.d_model * 4, 4 * md.d_model * 4, 4 * md.vocab_size * 4, 16, 1 << 16, 1 << 19, 1 << 22):
        torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")


def serve(m, md, prompt, ids, stream, busy):
    out = []
    for again in range(2):  # the second prefix replaces the first while its last step may still run
        out.append(m.share_prefix(prompt, 3, 6, stream=stream))
        if busy:
            stir(md, len(prompt))
        for step in range(4):
            got = m.step_shared(ids[step], stream=stream)
            if busy:
                stir(md, len(prompt))
            if stream is not None:
                stream.synchronize()
            out.append(got.clone())
    out.append(m.prefill(prompt[:40], stream=stream))
    if busy:
        stir(md, 40)
    out.append(m.step_batch([7], stream=stream))
    if busy:
        stir(md, 40)
    m.reset()
    torch.cuda.synchronize()
    return [x.clone() for x in out]


def test_shared_prefix_on_a_stream_of_its_own(ctx, orc):
    from test_gpu_trunk import synthetic_model

    from quantibbler_amd.model import DeviceModel

    md = synthetic_model(orc, 808)
    rng = np.random.default_rng(21)
    prompt = rng.integers(0, md.vocab_size, 65).tolist()
    ids = [rng.integers(0, md.vocab_size, 3).tolist() for _ in range(4)]
    m = DeviceModel(ctx, md, capacity=80)
    want = serve(m, md, prompt, ids, None, False)
    got = serve(m, md, prompt, ids, torch.cuda.Stream(), True)
    for i, (a, b) in enumerate(zip(got, want)):
        assert bool(b.isfinite().all()) and torch.equal(a, b), f"result {i}"
    m.close()
