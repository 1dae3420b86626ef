"""GPU: drafted tokens over vocabularies of more units than a wave has lanes, and
enough rows for 32 ids a thread, against the definition in 64 bits (as
test_gpu_verify): a wave looks through a row's units 64 at a time, 512 or 2048
ids each, so that 32768 and 131072 are where its second round begins."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import test_gpu_verify as ver
from quantibbler_amd import GpuContext
from test_gpu_verify import INF, tensor, words

BOTH = pytest.mark.parametrize("dtype", ["float32", "bfloat16"])


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


def number_of(row, v, t=1.0):
    """The f32 number that draws id v of a row of weights softmax(row / t): the middle of its part of the sum."""
    p = ver.chances(row, t)
    return np.float32((np.cumsum(p)[v] - 0.5 * p[v]) / p.sum())


@BOTH
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("n,k,vocab", [(1, 2, 32769), (2, 3, 50021), (1, 4, 128256), (2, 1, 131073), (1, 2, 200003)])
def test_against_the_definition(ctx, dtype, given, n, k, vocab):
    rng = np.random.default_rng(vocab)
    for case in range(3):
        temperature = None if case == 0 else (0.3 + 1.5 * rng.random(n)).astype(np.float32)
        if case == 2:
            temperature[0] = 0.0
        x, y, ids, u = ver.make(case, n, k, vocab, dtype, given, masked=case == 1, temperature=temperature)
        if case == 1:
            ids[:, 0] = vocab - 1  # refused or not: in the last unit
        got = ver.verify(ctx, x, y, ids, u, None, None if temperature is None else tensor(temperature), dtype)
        ver.check(*got, x, y, ids, u, None, temperature, f"case {case}")


@BOTH
@pytest.mark.parametrize("vocab", [32768, 32769, 66000, 128256, 200003])
def test_draws_from_every_round_of_units(ctx, dtype, vocab):
    """Numbers that draw the first and last id of the units on both sides of each border of 64 of them, of a flat row
    (one id a request), with nothing drafted and with a draft that is looked up and refused in the same, the first or
    the last unit."""
    unit, rng = 512, np.random.default_rng(vocab)
    borders = [b for b in range(0, vocab + 1, 64 * unit)] + [vocab]
    at = sorted({min(max(b + o, 0), vocab - 1) for b in borders for o in (-unit - 1, -unit, -1, 0, 1, unit - 1, unit)})
    n = 4  # few rows, so that units are of 512 ids
    row = torch.from_numpy(0.25 * rng.standard_normal(vocab)).to(getattr(torch, dtype)).cuda()
    host = row.double().cpu().numpy()
    for i in range(0, len(at), n):
        some = (at[i:i + n] * n)[:n]
        x = row.expand(n, 1, vocab).contiguous()
        u = np.array([[number_of(host, v)] for v in some], np.float32)
        none = torch.empty((n, 0), dtype=torch.int32, device="cuda")
        got = ver.verify(ctx, x, None, none, tensor(u), dtype=dtype)
        ver.check(*got, x, None, none, tensor(u), None, None, f"ids {some}")
        for passed in (0, some[0], vocab - 1):
            x2 = row.expand(n, 2, vocab).contiguous()
            u2 = tensor(np.concatenate([np.ones((n, 1), np.float32), u], 1))
            ids = words([[passed]] * n)
            got = ver.verify(ctx, x2, None, ids, u2, dtype=dtype)
            ver.check(*got, x2, None, ids, u2, None, None, f"ids {some} past {passed}")


@BOTH
@pytest.mark.parametrize("given", [False, True])
def test_weights_in_a_few_units(ctx, dtype, given):
    """All but some ids masked: nothing in the first 64 units, nothing behind them, one id in the last, the maximum past
    the first round; warm and greedy, and numbers past the last weight."""
    vocab, n, k = 128256, 4, 1
    alive = [[40000, 40001, 128255], [5, 32767], [128255], [32768, 100, 65536, 99999]]
    rng = np.random.default_rng(4)
    x = np.full((n, k + 1, vocab), -INF)
    for i, some in enumerate(alive):
        x[i][:, some] = rng.standard_normal((k + 1, len(some)))
    x[3, :, 65536] = 7.0
    y = tensor(x[:, :k] + 0.5 * rng.standard_normal((n, k, vocab)), getattr(torch, dtype)) if given else None
    x = tensor(x, getattr(torch, dtype))
    for ids in ([[a[0]] for a in alive], [[a[-1]] for a in alive], [[7]] * n):
        for number in (0.0, 0.3, 0.9999, 1.0, 5.0):
            u = tensor(np.full((n, k + 1), number, np.float32))
            for heat in (1.0, 0.0):
                heats = np.full(n, heat, np.float32)
                got = ver.verify(ctx, x, y, words(ids), u, temperature=tensor(heats), dtype=dtype)
                if number < 1.0:
                    ver.check(*got, x, y, words(ids), u, None, heats, f"{ids}, {number}, {heat}")
                else:  # an id that has a weight, always
                    tokens, counts = got[0].tolist(), got[1].tolist()
                    assert all(t in a for row, c, a in zip(tokens, counts, alive) for t in row[:c])
                    assert all(c >= 1 for c in counts)


@BOTH
@pytest.mark.parametrize("given,n,k,vocab", [(True, 64, 4, 32003), (False, 110, 4, 32003), (True, 10, 4, 200003),
                                             (False, 17, 4, 200003), (True, 40, 16, 12289)])
def test_32_ids_a_thread(ctx, dtype, given, n, k, vocab):
    """8192 units of 2048 ids and more; every third request by itself, at eight ids a thread, answers alike."""
    rows = n * (2 * k + 1 if given else k + 1)
    assert rows * (-(-vocab // 2048)) >= 8192
    rng = np.random.default_rng(vocab)
    counts = rng.integers(0, k + 1, n)
    counts[:2] = k
    heat = (0.4 + rng.random(n)).astype(np.float32)
    heat[1::5] = 0.0
    x, y, ids, u = ver.make(6, n, k, vocab, dtype, given, masked=True, temperature=np.where(heat > 0, heat, 1.0))
    u[: n // 2, :2] *= 0.01  # more of the drafts kept
    tokens, got = ver.verify(ctx, x, y, ids, u, words(counts), tensor(heat), dtype)
    few = slice(0, min(n, 24))
    ver.check(tokens[few], got[few], x[few], None if y is None else y[few], ids[few], u[few], counts, heat)
    for i in range(0, n, 3):
        one = ver.verify(ctx, x[i:i + 1], None if y is None else y[i:i + 1], ids[i:i + 1], u[i:i + 1],
                         words(counts[i:i + 1]), tensor(heat[i:i + 1]), dtype)
        assert torch.equal(one[0], tokens[i:i + 1]) and torch.equal(one[1], got[i:i + 1]), f"request {i}"


def test_greedy_rows_without_a_distribution(ctx):
    """At temperature 0 a row is what argmax makes of it, whatever it holds: no number is passed over, an infinity is the
    likeliest, and of nothing the first id is taken, which counts, and is kept where it was drafted."""
    from quantibbler_amd.gpu import argmax_dev

    n, k, vocab = 6, 2, 40001
    x = torch.randn((n, k + 1, vocab), device="cuda")
    x[1], x[2] = -INF, float("nan")
    x[3, :, 35000], x[4, :, ::2], x[5, :, :39999] = INF, float("nan"), -INF
    best = torch.empty((n, k + 1), dtype=torch.int32, device="cuda")
    argmax_dev(ctx, x, n * (k + 1), vocab, best)
    torch.cuda.synchronize()
    assert best[1:4].tolist() == [[0] * 3, [0] * 3, [35000] * 3]
    u, cold = torch.rand((n, k + 1), device="cuda"), torch.zeros(n, device="cuda")
    for y in (None, torch.randn((n, k, vocab), device="cuda")):
        tokens, counts = ver.verify(ctx, x, y, best[:, :k].contiguous(), u, temperature=cold)
        assert torch.equal(tokens, best) and counts.tolist() == [k + 1] * n
        tokens, counts = ver.verify(ctx, x, y, (best[:, :k] + 1).contiguous(), u, temperature=cold)
        assert torch.equal(tokens[:, 0], best[:, 0]) and counts.tolist() == [1] * n
