"""GPU: drafted tokens where a request's rows end."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import test_gpu_attention_kv as att
import test_gpu_block_kv as bkv
from quantibbler_amd import DecoderBlock, GpuContext

words, EPS = att.words, 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


@pytest.mark.parametrize("fmt", ["int8", "fp8", "fp4"])
@pytest.mark.parametrize("per,plen,lens", [(5, 0, [10, 68, 66, 69]), (4, 129, [69, 66, 67, 0]), (20, 70, [51, 69, 60])])
def test_tokens_that_fit_before_those_that_do_not(ctx, orc, fmt, per, plen, lens):
    """A step that passes a sequence's last row: its tokens before that see the rows up to their own, as any."""
    rng = np.random.default_rng(200 + per)
    L = bkv.Layers(ctx, orc, 5)
    D, HEADS, KV, HD, n, cap = bkv.D, bkv.HEADS, bkv.KV, bkv.HD, len(lens), 70
    block = DecoderBlock(ctx, L.all, np.ones(D), np.ones(D), HEADS, KV, HD, bkv.THETA, 1e-5, capacity=400)
    cache = bkv.make(ctx, fmt, n, cap)
    bkv.fill(cache, rng, lens)
    shared, p = None, (np.zeros((0, KV, HD)),) * 2
    if plen:
        shared = bkv.make(ctx, fmt, 1, plen)
        bkv.fill(shared, rng, [plen])
        p = bkv.held(shared, [plen])[0]
    h = rng.standard_normal((n, per, D)).astype(np.float32)
    hd = torch.from_numpy(h).cuda()
    need = block.decode_kv_workspace_size(cache, n, prefix_len=plen, n_tokens=per)
    block.decode_kv_dev(hd, words(lens), n, cache, torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda"), need,
                        prefix=shared, prefix_len=plen, n_tokens=per)
    torch.cuda.synchronize()
    now = bkv.held(cache, [min(x + per, cap) for x in lens])
    got = hd.cpu().numpy().astype(np.float64)
    for i in range(n):
        k, v = now[i]
        for t in range(min(per, cap - lens[i])):
            seen = lens[i] + t + 1
            a, tol = bkv.attention(bkv.rotated(L.q, HEADS, plen + lens[i] + t), np.concatenate([p[0], k[:seen]]),
                                   np.concatenate([p[1], v[:seen]]))
            want, bound = bkv.o_layer(L, a, tol)
            want = want + h[i, t]
            off = np.abs(got[i, t] - want) - bound - 2 * EPS * np.abs(want)
            assert (off <= 0).all(), f"sequence {i}, token {t}: past its bound by {off.max()}"
    block.close()
