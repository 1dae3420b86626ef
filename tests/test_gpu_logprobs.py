"""GPU: log probabilities, entropy and likeliest tokens against float64.

With d = x - max, E over the softmax and eps = 2^-24 (half a step of f32): a
term exp(d) is off by (2 + 1.5 |d|) eps (d rounded, times log2 e, the
exponential's last place), a tree over 32 logits a thread, 64 lanes, 4 waves
and the chunks adds at most 60 eps, so log l is off by (62 + 1.5 E|d|) eps and
its own rounding; x - max and the last subtraction add a rounding each.  The
entropy's E d is off by E(|d| (64 + 1.5 |d|)) eps and l's share of it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from quantibbler_amd import GpuContext
from quantibbler_amd.gpu import argmax_dev, logprobs_dev, logprobs_workspace_size

EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


def call(ctx, x, targets, top, stride=None, rows=None, vocab=None, ws=None):
    rows, vocab = x.shape if rows is None else (rows, vocab)
    need = logprobs_workspace_size(rows, vocab, top)
    ws = torch.full((max(need, 16),), 0xFF, dtype=torch.uint8, device="cuda") if ws is None else ws
    lp, ent = torch.full((rows,), 9.0, device="cuda"), torch.full((rows,), 9.0, device="cuda")
    ids = torch.full((rows, max(top, 1)), -5, dtype=torch.int32, device="cuda")
    tops = torch.full((rows, max(top, 1)), 9.0, device="cuda")
    logprobs_dev(ctx, x, rows, vocab, targets, lp, ent, ws, need, top_k=top, top_ids=ids if top else None,
                 top_logprobs=tops if top else None, dtype=str(x.dtype).split(".")[1], row_stride=stride,
                 stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    return lp.cpu().numpy(), ent.cpu().numpy(), ids.cpu().numpy(), tops.cpu().numpy()


def close(got, want, tol, label):
    got = got.astype(np.float64)
    with np.errstate(invalid="ignore"):
        same = (np.abs(got - want) <= tol) | (got == want) | (np.isnan(got) & np.isnan(want))
    assert same.all(), f"{label}: {np.count_nonzero(~same)} off, {got[~same][:3]} for {want[~same][:3]}"


def reference(x, targets, top):
    """numpy float64 of one row."""
    x = x.astype(np.float64)
    order = np.argsort(-np.where(np.isnan(x), -np.inf, x), kind="stable")[:top]
    if np.isnan(x).any() or np.isposinf(x).any() or np.isneginf(x).all():
        return np.nan, np.nan, order, np.full(top, np.nan), 1.0, 1.0, np.full(top, 1.0)
    d = x - x.max()
    e = np.exp(d)
    p = e / e.sum()
    lse = np.log(e.sum())
    fin = np.where(np.isneginf(d), 0.0, d)
    m1, m2 = (p * np.abs(fin)).sum(), (p * fin * fin).sum()
    base = (64 + 1.5 * m1 + 2 * abs(lse)) * EPS
    lp = d[targets] - lse if 0 <= targets < x.size else np.nan
    mag = lambda a: np.where(np.isfinite(a), np.abs(a), 0.0)
    return (lp, lse - (p * fin).sum(), order, d[order] - lse, base + 2 * EPS * mag(lp),
            base + (64 * m1 + 1.5 * m2 + 64 * m1 + 1.5 * m1 * m1) * EPS, base + 2 * EPS * mag(d[order] - lse))


def against(ctx, x, targets, top, **kw):
    t = x if kw.get("stride") is None else x[:, :kw["vocab"]]
    lp, ent, ids, tops = call(ctx, x, targets, top, **kw)
    tn, xn = targets.cpu().numpy(), t.float().cpu().numpy()
    for r in range(len(lp)):
        w = reference(xn[r], tn[r], top)
        close(lp[r:r + 1], np.array([w[0]]), w[4], f"row {r} logprob")
        close(ent[r:r + 1], np.array([w[1]]), w[5], f"row {r} entropy")
        if top:
            assert ids[r].tolist() == w[2].tolist(), f"row {r} ids"
            close(tops[r], w[3], w[6], f"row {r} top")


def logits(seed, rows, vocab, dtype=torch.float32, scale=3.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (scale * torch.randn((rows, vocab), device="cuda", generator=g)).to(dtype)


def ids_of(seed, rows, vocab):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, vocab, rows).astype(np.int32)).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 0), (3, 5, 5), (2, 64, 64), (5, 255, 3), (2, 8191, 20),
                                            (2, 8192, 64), (2, 8193, 64), (3, 8200, 1), (4, 16385, 7), (2, 32003, 20),
                                            (1, 128256, 64), (9, 50001, 0), (1, 300001, 64)])
def test_against_float64(ctx, dtype, rows, vocab, top):
    against(ctx, logits(vocab + rows, rows, vocab, dtype), ids_of(vocab, rows, vocab), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lower_id(ctx, dtype):
    x = torch.zeros((4, 20000), device="cuda", dtype=dtype)
    x[1] = -torch.arange(20000, device="cuda").remainder(3).to(dtype)
    x[2, 11111:] = 5.0
    x[3, ::2] = -0.0
    against(ctx, x, ids_of(1, 4, 20000), 40)


def test_sorted_and_one_sided_rows(ctx):
    """Every likely token in one thread's, one wave's or one chunk's share of the row."""
    n = 30000
    x = torch.empty((5, n), device="cuda")
    x[0] = torch.arange(n, device="cuda") * 1e-3
    x[1] = -torch.arange(n, device="cuda") * 1e-3
    x[2:] = -50.0
    x[2, 4096:4160] = torch.arange(64, device="cuda").float()
    x[3, 3:n:1024] = 1.0
    x[4, n - 64:] = 2.0
    against(ctx, x, ids_of(2, 5, n), 64)


def test_masks_and_values_that_are_no_numbers(ctx):
    x = logits(4, 9, 9000)
    x[0, 5:8999] = float("-inf")
    x[1] = float("-inf")
    x[2, 7] = float("nan")
    x[3, 8999] = float("inf")
    x[4, 0:8192] = float("-inf")         # a whole chunk
    x[5, 8192:] = float("-inf")
    x[6] = -3.4028234663852886e38        # a type's lowest value as the mask
    x[6, 100] = 0.0
    x[7] = 3.0e38
    x[8] = float("nan")
    t = torch.tensor([6, 0, 1, 1, 3, 8500, 100, 4, 2], dtype=torch.int32, device="cuda")
    against(ctx, x, t, 12)
    like = torch.full((1, 9000), -3.3895313892515355e38, dtype=torch.bfloat16, device="cuda")
    like[0, 77] = 1.0
    against(ctx, like, torch.tensor([77], dtype=torch.int32, device="cuda"), 3)


def test_targets_outside_the_vocabulary(ctx):
    x = logits(6, 4, 100)
    t = torch.tensor([-1, 100, 2 ** 31 - 1, -100], dtype=torch.int32, device="cuda")
    lp, ent, ids, tops = call(ctx, x, t, 2)
    assert np.isnan(lp).all() and np.isfinite(ent).all() and np.isfinite(tops).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_strided_rows(ctx, dtype, shift):
    """A vocabulary padded to a wider row, at any alignment of the rows."""
    vocab, wide = 9001, 9011
    base = logits(7, 3, wide + 8, dtype)
    x = base.flatten()[shift:shift + 3 * wide].view(3, wide)
    x[:, vocab:] = 100.0
    against(ctx, x, ids_of(3, 3, vocab), 9, stride=wide, rows=3, vocab=vocab)


def test_outputs_left_out_and_first_is_argmax(ctx):
    x = logits(8, 6, 40000)
    need = logprobs_workspace_size(6, 40000, 1)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    ids, tops = torch.empty(6, dtype=torch.int32, device="cuda"), torch.empty(6, device="cuda")
    logprobs_dev(ctx, x, 6, 40000, None, None, None, ws, need, top_k=1, top_ids=ids, top_logprobs=tops)
    am = torch.empty(6, dtype=torch.int32, device="cuda")
    argmax_dev(ctx, x, 6, 40000, am)
    torch.cuda.synchronize()
    assert torch.equal(ids, am)


def test_graph_and_streams(ctx):
    """Captured and replayed with new logits, and on a stream of its own: each replay the eager result, bit for bit."""
    rows, vocab, top = 5, 20001, 8
    x, t = logits(9, rows, vocab), ids_of(9, rows, vocab)
    need = logprobs_workspace_size(rows, vocab, top)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = [torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"),
           torch.empty((rows, top), dtype=torch.int32, device="cuda"), torch.empty((rows, top), device="cuda")]

    def go():
        logprobs_dev(ctx, x, rows, vocab, t, out[0], out[1], ws, need, top_k=top, top_ids=out[2], top_logprobs=out[3],
                     stream=torch.cuda.current_stream())

    go()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for rep in range(3):
        x.copy_(logits(20 + rep, rows, vocab))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.cpu().numpy().copy() for o in out]
        want = call(ctx, x, t, top)
        for a, b in zip(got, want):
            assert a.tobytes() == b.tobytes()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go()
    s.synchronize()
    for a, b in zip(out, call(ctx, x, t, top)):
        assert a.cpu().numpy().tobytes() == b.tobytes()
    del graph
