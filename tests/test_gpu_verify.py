"""GPU: drafted tokens against the target's probabilities: the ids and counts of
the definition in 64 bits on the same logits and numbers, exactly.  (A draw
hangs on whether a running sum is above a number: sums that differ by 1e-13 of
the whole answer differently in one draw of 10^13 over the ids next to it, and
the cases that meet a border on purpose are made of numbers whose sums are
exact.)"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from quantibbler_amd import GpuContext, KernelError
from quantibbler_amd.gpu import verify_drafts_dev, verify_drafts_workspace_size

INF = float("inf")


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


def chances(row, t):
    """softmax(row / t), all on the first of the largest at t = 0; None for a row that has none."""
    row = np.asarray(row, np.float64)
    if not t > 0:
        row = np.where(np.isnan(row), -INF, row)
        p = np.zeros(len(row))
        p[int(np.argmax(row)) if row.max() > -INF else 0] = 1.0
        return p
    if np.isnan(row).any() or row.max() in (INF, -INF):
        return None
    e = np.exp((row - row.max()) / np.float64(t))
    return e / e.sum()


def expected(x, y, ids, m, u, t):
    """One request: its tokens."""
    out = []
    for j in range(m + 1):
        p, w = chances(x[j], t), None
        if p is None:
            return out, None
        if j < m:
            d = int(ids[j])
            q = chances(y[j], t) if y is not None else np.eye(1, len(p), d)[0] if 0 <= d < len(p) else np.zeros(len(p))
            if not t > 0:
                q = np.eye(1, len(p), d)[0] if 0 <= d < len(p) else np.zeros(len(p))
            if 0 <= d < len(p) and q is not None and np.float64(u[j]) * q[d] < p[d]:
                out.append(d)
                continue
            w = np.maximum(p - q, 0.0) if q is not None else None
        if w is None or not w.sum() > 0:
            w = p
        sums = np.cumsum(w)
        over = np.flatnonzero((sums > np.float64(u[m]) * sums[-1]) & (w > 0))
        return out, int(over[0]) if len(over) else int(np.flatnonzero(w > 0)[-1])


def tensor(x, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def words(v):
    return torch.tensor(np.asarray(v).tolist(), dtype=torch.int32, device="cuda")


def verify(ctx, x, y, ids, u, counts=None, temperature=None, dtype="float32", pos=None, stream=None, ws=None, **kw):
    """Device tensors x [n][k + 1][vocab], y [n][k][vocab] or None, ids [n][k], u [n][k + 1]."""
    n, k, vocab = ids.shape[0], ids.shape[1], x.shape[-1]
    need = verify_drafts_workspace_size(n, k, vocab, y is not None)
    if ws is None:
        ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    tokens = torch.full((n, k + 1), 77, dtype=torch.int32, device="cuda")
    got = torch.full((n,), 77, dtype=torch.int32, device="cuda")
    verify_drafts_dev(ctx, x, n, k, vocab, ids, u, tokens, got, ws, need, draft_logits=y, n_drafts=counts,
                      temperature=temperature, pos=pos, dtype=dtype, stream=stream, **kw)
    return tokens, got


def check(tokens, got, x, y, ids, u, counts, temperature, label=""):
    x, u, ids = x.double().cpu().numpy(), u.cpu().numpy(), ids.cpu().numpy()
    y = None if y is None else y.double().cpu().numpy()
    tokens, got = tokens.cpu().numpy(), got.cpu().numpy()
    for i in range(len(x)):
        m = ids.shape[1] if counts is None else min(int(counts[i]), ids.shape[1])
        kept, token = expected(x[i], None if y is None else y[i], ids[i], m, u[i],
                               1.0 if temperature is None else float(temperature[i]))
        want = kept + [-1 if token is None else token]
        want += [-1] * (tokens.shape[1] - len(want))
        assert tokens[i].tolist() == want, f"{label} request {i}: {tokens[i].tolist()}, not {want}"
        assert got[i] == len(kept) + (token is not None), f"{label} request {i}"


def make(seed, n, k, vocab, dtype, given, masked=False, near=0.5, temperature=None):
    rng = np.random.default_rng(seed)
    x = 2.5 * rng.standard_normal((n, k + 1, vocab))
    for i in range(n):
        for j in range(k + 1):
            x[i, j, rng.integers(0, vocab, 3)] = 8.0 + rng.standard_normal()
    if masked:
        hide = rng.random(vocab) < 0.4
        hide[rng.integers(0, vocab)] = False
        x[..., hide] = -INF
    t = getattr(torch, dtype)
    y = tensor(x[:, :k] + near * rng.standard_normal((n, k, vocab)), t)
    x = tensor(x, t)
    ids = np.zeros((n, k), np.int32)
    y64 = y.double().cpu().numpy()
    for i in range(n):
        for j in range(k):
            p = chances(y64[i, j], 1.0 if temperature is None else float(temperature[i]))
            ids[i, j] = rng.choice(vocab, p=p)
    return x, (y if given else None), tensor(ids, torch.int32), tensor(rng.random((n, k + 1)), torch.float32)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("n,k,vocab", [(1, 0, 1), (1, 1, 1), (3, 2, 2), (5, 1, 7), (4, 3, 255), (2, 4, 2048), (2, 4, 2049),
                                       (3, 5, 8191), (2, 3, 8193), (2, 2, 32003), (33, 4, 1000), (2, 64, 300), (9, 8, 20011)])
def test_against_the_definition(ctx, dtype, given, n, k, vocab):
    if given and k == 0:
        pytest.skip("no drafts")
    rng = np.random.default_rng(vocab + n)
    for case in range(3):
        temperature = None if case == 0 else (0.3 + 1.5 * rng.random(n)).astype(np.float32)
        counts = None if case == 0 else rng.integers(0, k + 2, n)  # one past k counts as k
        if case == 2:
            temperature[::2] = 0.0
        x, y, ids, u = make(case, n, k, vocab, dtype, given, masked=case == 2, temperature=temperature)
        got = verify(ctx, x, y, ids, u, None if counts is None else words(counts),
                     None if temperature is None else tensor(temperature), dtype)
        check(*got, x, y, ids, u, counts, temperature, f"case {case}")


@pytest.mark.parametrize("given", [False, True])
def test_a_card_full_of_rows(ctx, given):
    """Enough rows for chunks of 32 ids a thread; the same requests a few at a time take eight, and answer alike."""
    n, k, vocab = 40, 4, 32003
    x, y, ids, u = make(5, n, k, vocab, "bfloat16", given)
    tokens, got = verify(ctx, x, y, ids, u, dtype="bfloat16")
    check(tokens[:6], got[:6], x[:6], None if y is None else y[:6], ids[:6], u[:6], None, None)
    for i in range(0, n, 3):
        some = verify(ctx, x[i:i + 3], None if y is None else y[i:i + 3], ids[i:i + 3], u[i:i + 3], dtype="bfloat16")
        assert torch.equal(some[0], tokens[i:i + 3]) and torch.equal(some[1], got[i:i + 3])


def test_draws_on_the_borders(ctx):
    """Logits all alike over a power of two: running sums are exact, and the number j / V draws id j, the one below it
    id j - 1; a draft that was looked up is passed over."""
    for vocab in (1, 2, 64, 8192, 16384):
        n = min(vocab, 300)
        at = np.linspace(0, vocab - 1, n).round().astype(np.int64)
        x = torch.zeros((n, 1, vocab), device="cuda")
        for shift in (0.0, 2.0 ** -24):
            u = (at / vocab - shift * np.maximum(at / vocab, 2.0 ** -14)).astype(np.float32)
            u = np.maximum(u, 0)
            want = np.maximum(at - (shift > 0), 0)
            tokens, got = verify(ctx, x, None, torch.empty((n, 0), dtype=torch.int32, device="cuda"), tensor(u[:, None]))
            assert (tokens[:, 0].cpu().numpy() == want).all() and bool((got == 1).all())
    vocab, d = 8192, 4000  # V - 1 ids are left: those before d by j / (V - 1), the ones behind one later
    x = torch.zeros((2, 2, vocab), device="cuda")
    x[:, 0, vocab - 1] = -INF  # V - 2 of them: 8190
    u = tensor(np.array([[1.0, 3999.5 / 8190], [1.0, 4000.5 / 8190]], np.float32))
    tokens, _ = verify(ctx, x, None, words([[d], [d]]), u)
    assert tokens.tolist() == [[3999, -1], [4001, -1]]


def test_acceptance_on_the_border(ctx):
    """u q(d) < p(d) is strict: p = 1/2, q = 1 and u = 1/2 keeps nothing, the number below it does."""
    x = torch.zeros((2, 2, 2), device="cuda")
    below = float(np.nextafter(np.float32(0.5), np.float32(0)))
    u = tensor(np.array([[0.5, 0.9], [below, 0.9]], np.float32))
    tokens, counts = verify(ctx, x, None, words([[1], [1]]), u)
    assert tokens.tolist() == [[0, -1], [1, 1]] and counts.tolist() == [1, 2]


def test_equal_distributions_keep_every_draft(ctx):
    n, k, vocab = 6, 5, 3001
    x, _, _, _ = make(7, n, k, vocab, "float32", False)
    ids = torch.randint(0, vocab, (n, k), device="cuda", dtype=torch.int32)
    u = torch.rand((n, k + 1), device="cuda") * 0.999
    tokens, counts = verify(ctx, x, x[:, :k].contiguous(), ids, u)
    assert torch.equal(tokens[:, :k], ids) and bool((counts == k + 1).all())
    # and one that is not kept although they are (a number of 1) draws from p
    u[:, 0] = 1.0
    tokens, counts = verify(ctx, x, x[:, :k].contiguous(), ids, u)
    assert bool((counts == 1).all())
    check(tokens, counts, x, x[:, :k].contiguous(), ids, u, None, None)


def test_numbers_out_of_range(ctx):
    """Numbers of 1 and more, below 0 or NaN: an id that has a weight, always."""
    n, vocab = 5, 9001
    x = torch.full((n, 2, vocab), -INF, device="cuda")
    x[:, :, 100] = 1.0
    x[:, :, 8000] = 1.0
    u = tensor(np.array([[1.0, 1.0], [2.0, 1e30], [1.0, -3.0], [float("nan")] * 2, [1.0, float("-inf")]], np.float32))
    tokens, counts = verify(ctx, x, None, words([[5]] * n), u)
    assert tokens[:, 0].tolist() == [8000, 8000, 100, 8000, 100] and bool((counts == 1).all())


def test_rows_without_a_distribution(ctx):
    n, k, vocab = 8, 2, 5000
    x, y, ids, u = make(11, n, k, vocab, "float32", True)
    u[:] = 0.01
    ids[:] = x[:, :k].argmax(-1).int()  # kept, but for what follows
    x[1, 0, 7], x[2, 1, 4999], x[3, 2, 0], x[4, 0] = float("nan"), INF, float("nan"), -INF
    y[5, 1, 9], y[6, 0] = float("nan"), -INF
    ids[7, 0] = vocab
    for draft in (y, None):
        tokens, counts = verify(ctx, x, draft, ids, u)
        check(tokens, counts, x, draft, ids, u, None, None)
        assert counts[1:5].tolist() == [0, 1, 2, 0]
    ids[7, 0] = -1
    check(*verify(ctx, x, y, ids, u), x, y, ids, u, None, None)
    # the likeliest id is the one that the greedy sampler takes, whatever else the row holds
    cold = torch.zeros(n, device="cuda")
    check(*verify(ctx, x, y, ids, u, temperature=cold), x, y, ids, u, None, cold.cpu().numpy())


def test_greedy_is_argmax(ctx):
    """At temperature 0 what is emitted is argmax's ids, first ones at ties, one after the other."""
    from quantibbler_amd.gpu import argmax_dev

    n, k, vocab = 7, 6, 12345
    x = torch.randint(-3, 4, (n, k + 1, vocab), device="cuda").float()
    x[0, 0] = 0.0
    x[1, 1, 5:] = float("nan")
    best = torch.empty((n, k + 1), dtype=torch.int32, device="cuda")
    argmax_dev(ctx, x, n * (k + 1), vocab, best)
    torch.cuda.synchronize()
    for wrong in range(k + 1):
        ids = best[:, :k].clone()
        if wrong < k:
            ids[:, wrong] = (ids[:, wrong] + 1) % vocab
        u = torch.rand((n, k + 1), device="cuda")
        tokens, counts = verify(ctx, x, None, ids, u, temperature=torch.zeros(n, device="cuda"))
        assert torch.equal(tokens[:, :wrong + 1], best[:, :wrong + 1]) and bool((tokens[:, wrong + 1:] == -1).all())
        assert bool((counts == wrong + 1).all())


def test_emitted_tokens_have_the_targets_distribution(ctx):
    """40000 requests of one draft each over eight ids: the first emitted id's share is p within five deviations, with a
    draft model near, far and looked up."""
    n, vocab = 40000, 8
    rng = np.random.default_rng(3)
    p_logits = rng.standard_normal(vocab)
    x = tensor(np.broadcast_to(p_logits, (n, 2, vocab)), torch.float32)
    p = chances(p_logits.astype(np.float32), 1.0)
    for far in (0.0, 0.5, 3.0, None):
        q_logits = p_logits + (far or 0.0) * rng.standard_normal(vocab)
        q = chances(q_logits.astype(np.float32), 1.0)
        ids = rng.choice(vocab, n, p=q) if far is not None else np.full(n, 2)
        y = tensor(np.broadcast_to(q_logits, (n, 1, vocab)), torch.float32) if far is not None else None
        tokens, _ = verify(ctx, x, y, words(ids[:, None]), tensor(rng.random((n, 2)).astype(np.float32)))
        share = np.bincount(tokens[:, 0].cpu().numpy(), minlength=vocab) / n
        assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n)).all(), f"{far}: {share} for {p}"


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_apart_and_positions(ctx, dtype):
    """Rows inside wider ones, at any alignment; positions advance by what was emitted."""
    n, k, vocab = 4, 3, 4099
    x, y, ids, u = make(21, n, k, vocab, dtype, True)
    wide = torch.full((n, k + 1, vocab + 13), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, :, 3:3 + vocab] = x
    thin = torch.full((n, k, vocab + 6), float("nan"), dtype=x.dtype, device="cuda")
    thin[:, :, 5:5 + vocab] = y
    pos = words([5, 0, 1000, 7])
    tokens = torch.empty((n, k + 1), dtype=torch.int32, device="cuda")
    counts = torch.empty(n, dtype=torch.int32, device="cuda")
    need = verify_drafts_workspace_size(n, k, vocab, True)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    verify_drafts_dev(ctx, wide[:, :, 3:], n, k, vocab, ids, u, tokens, counts, ws, need, draft_logits=thin[:, :, 5:],
                      pos=pos, dtype=dtype, row_stride=vocab + 13, draft_row_stride=vocab + 6)
    check(tokens, counts, x, y, ids, u, None, None)
    assert pos.tolist() == [a + b for a, b in zip([5, 0, 1000, 7], counts.tolist())]


def test_large_and_small_logits(ctx):
    """Logits of 1e30 and a temperature of 1e-30, of 1e30 and infinite: a distribution still."""
    n, vocab = 6, 3000
    rng = np.random.default_rng(9)
    for size, t in ((1e30, 1.0), (1e-30, 1.0), (1.0, 1e-30), (1.0, 1e30), (1.0, INF), (1e30, 1e30)):
        x = tensor(size * rng.standard_normal((n, 2, vocab)), torch.float32)
        x[:, :, ::3] = -INF
        ids = tensor(rng.integers(0, vocab, (n, 1)), torch.int32)
        u = tensor(rng.random((n, 2)), torch.float32)
        temperature = np.full(n, t, np.float32)
        got = verify(ctx, x, x[:, :1].contiguous(), ids, u, temperature=tensor(temperature))
        check(*got, x, x[:, :1], ids, u, None, np.minimum(temperature, 3e38), f"{size}, {t}")


def test_replays_and_streams(ctx):
    """Captured once and replayed on new logits, numbers, counts and temperatures; two graphs with their own workspaces
    beside each other; other streams answer alike."""
    n, k, vocab = 5, 4, 20000
    graphs = []
    for g in range(2):
        x, y, ids, u = make(30 + g, n, k, vocab, "float32", g == 0)
        counts, heat, pos = words([k] * n), torch.ones(n, device="cuda"), words([0] * n)
        need = verify_drafts_workspace_size(n, k, vocab, g == 0)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        out = [torch.empty((n, k + 1), dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")]

        def step(x=x, y=y, ids=ids, u=u, counts=counts, heat=heat, pos=pos, ws=ws, need=need, out=out):
            verify_drafts_dev(ctx, x, n, k, vocab, ids, u, *out, ws, need, draft_logits=y, n_drafts=counts,
                              temperature=heat, pos=pos, stream=torch.cuda.current_stream())

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append((graph, x, y, ids, u, counts, heat, pos, out))
    for rep in range(4):
        for g, (graph, x, y, ids, u, counts, heat, pos, out) in enumerate(graphs):
            x2, y2, ids2, u2 = make(50 + 2 * rep + g, n, k, vocab, "float32", g == 0)
            for a, b in ((x, x2), (y, y2), (ids, ids2), (u, u2)):
                if a is not None:
                    a.copy_(b)
            counts.copy_(words([rep % (k + 1), k, 0, 2, 9]))
            heat.copy_(tensor(np.array([1, 0, 0.5, 2, 1], np.float32)))
            pos.fill_(10 * rep)
            graph.replay()
            torch.cuda.synchronize()
            check(*out, x, y, ids, u, counts.tolist(), heat.tolist(), f"replay {rep}")
            assert pos.tolist() == [10 * rep + c for c in out[1].tolist()]
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                again = verify(ctx, x, y, ids, u, counts, heat, stream=s)
            torch.cuda.synchronize()
            assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])
    del graphs
