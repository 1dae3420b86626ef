"""GPU: attention over the 8-bit KV cache against float64 on the values the
cache stands for (read back through read_dev).

Tolerance of an output channel, with w the softmax weights and eps = 2^-24:
scores are off by at most b = scale ((d + 8) eps max_j sum_c |q_c k_jc| + 2^-28
max|q| max_j sum_c |k_jc|) -- f32 sums of d exact products, f32 queries held in
22 bits (f32: 2^-23 more of the first sum), fp16's smallest step against the
largest channel -- which moves every weight by 2 b; a weight is rounded to fp16
(2^-11; f32 queries: two halves, 2^-22), the exponential and the scales add
4 eps, the sums n eps each; weights below 2^-26 of the reference are steps of
2^-36; the output is rounded once (bf16 2^-8, f32 eps)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from quantibbler_amd import GpuContext, KernelError, KvCache

EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


def words(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def normal(seed, shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g)


def make(ctx, fmt, n, cap, kv, d, poison=True):
    buf = torch.empty(KvCache.size(fmt, n, cap, kv, d), dtype=torch.uint8, device="cuda")
    if poison:
        buf.fill_(0xFF)  # NaN codes and scales where nothing is written
    return KvCache(ctx, fmt, n, cap, kv, d, buf)


def fill(cache, seed, rows, first=0, scale=1.0, poke=None):
    """rows[i] rows into sequence first + i; returns what they read back as, [i] -> (k, v) [rows][kv][d] float64."""
    kv, d, total = cache.n_kv_heads, cache.head_dim, sum(rows)
    k = scale * (normal(seed, (total, kv, d)) + 2.0 * normal(seed + 1, (1, kv, d)))
    v = scale * normal(seed + 2, (total, kv, d)) * torch.exp(normal(seed + 3, (total, kv, 1)))
    if poke:
        poke(k, v)
    starts, at, n = words(np.concatenate([[0], np.cumsum(rows)])), words([0] * len(rows)), len(rows)
    cache.write_dev(k, v, "float32", at, total, first_seq=first, n_seqs=n, row_start=starts)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    cache.read_dev(ko, vo, "float32", at, total, first_seq=first, n_seqs=n, row_start=starts)
    out, s = [], 0
    for r in rows:
        out.append((ko[s:s + r].double(), vo[s:s + r].double()))
        s += r
    return out


def attend(cache, q, lens, dtype, prefix=None, plen=0, pseq=0, first=0, max_len=None, ws=None, stream=None):
    n, sq, heads, d = q.shape
    need = cache.attention_workspace_size(heads, n, seq_q=sq, max_len=max_len, prefix_len=plen)
    if ws is None:
        ws = torch.full((max(need, 16),), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 77.0)
    cache.attention_dev(q, dtype, heads, lens, out, ws, need, first_seq=first, n_seqs=n, seq_q=sq, max_len=max_len,
                        prefix=prefix, prefix_seq=pseq, prefix_len=plen, stream=stream)
    return out


def reference(q, prefix, own, lens, max_len=None):
    """float64 outputs and their tolerances (without the output's rounding)."""
    n, sq, heads, d = q.shape
    f32 = q.dtype == torch.float32
    q64 = q.double()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    scale = d ** -0.5
    for b in range(n):
        ln = lens[b] if max_len is None else min(lens[b], max_len)
        k = torch.cat([prefix[0], own[b][0][:ln]])
        v = torch.cat([prefix[1], own[b][1][:ln]])
        p, kv = prefix[0].shape[0], k.shape[1]
        if k.shape[0] == 0:
            continue
        index = torch.arange(k.shape[0], device="cuda")
        for h in range(heads):
            j = h // (heads // kv)
            kk, vv = k[:, j], v[:, j]
            qq = q64[b, :, h]
            s = (qq @ kk.t().contiguous()) * scale
            seen = (index[None] < p) | (index[None] < p + ln - sq + 1 + torch.arange(sq, device="cuda")[:, None])
            any_ = seen.any(-1, keepdim=True)
            w = torch.where(seen, s, torch.full_like(s, float("-inf")))
            w = torch.where(any_, (w - w.amax(-1, keepdim=True)).exp(), torch.zeros_like(w))
            w = torch.where(any_, w / w.sum(-1, keepdim=True), w)
            ok = seen.any(0)  # rows no query sees may be NaN
            kk, vv, w = kk[ok], vv[ok], w[:, ok]
            out[b, :, h] = w @ vv
            mass = (qq.abs() @ kk.abs().t().contiguous()).amax(-1, keepdim=True)
            bound = scale * (((d + 8) * EPS + (2.0 ** -23 if f32 else 0)) * mass +
                             2.0 ** -28 * qq.abs().amax(-1, keepdim=True) * kk.abs().sum(-1).max())
            m = int(ok.sum())
            rel = 2 * bound + (2.0 ** -22 if f32 else 2.0 ** -11) + (2 * m + 70) * EPS
            tol[b, :, h] = rel * (w @ vv.abs()) + m * 2.0 ** -36 * vv.abs().max()
    return out, tol


def check(got, want, tol, label=""):
    step = EPS if got.dtype == torch.float32 else 2.0 ** -8
    bad = ~((got.double() - want).abs() <= tol + step * want.abs() + 1e-40)
    assert not bool(bad.any()), f"{label}: {int(bad.sum())} of {bad.numel()} off, worst " \
        f"{float((got.double() - want).abs()[bad].max()):.3g} at {bad.nonzero()[:2].tolist()}"


def empty_prefix(kv, d):
    z = torch.zeros((0, kv, d), dtype=torch.float64, device="cuda")
    return z, z


# n, heads, kv heads, d, queries, own rows, prefix
SHAPES = [(1, 1, 1, 16, 1, [1], 0), (1, 4, 2, 64, 1, [63], 0), (2, 4, 4, 80, 1, [64, 65], 1),
          (1, 8, 2, 128, 1, [700], 0), (3, 6, 3, 128, 1, [0, 1, 130], 0), (3, 8, 2, 128, 1, [5, 0, 300], 77),
          (5, 32, 8, 128, 1, [100, 3, 257, 64, 1], 1000), (17, 8, 8, 64, 1, [i for i in range(17)], 300),
          (4, 4, 1, 256, 1, [9, 80, 200, 0], 129), (2, 14, 2, 240, 1, [70, 5], 64),
          (2, 4, 2, 128, 5, [3, 90], 0), (2, 4, 2, 128, 5, [3, 90], 50), (3, 16, 2, 112, 4, [4, 65, 129], 190),
          (1, 2, 1, 96, 70, [70], 0), (2, 7, 1, 32, 33, [20, 400], 65), (1, 8, 1, 256, 20, [21], 500),
          (1, 8, 8, 48, 1, [0], 4097), (1, 4, 2, 128, 300, [1300], 0)]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,heads,kv,d,sq,rows,plen", SHAPES)
def test_against_float64(ctx, fmt, dtype, n, heads, kv, d, sq, rows, plen):
    q = (1.5 * normal(n + d, (n, sq, heads, d))).to(getattr(torch, dtype))
    cache = make(ctx, fmt, n, max(1, max(rows)), kv, d)
    own = fill(cache, 10, rows)
    shared, p = None, empty_prefix(kv, d)
    if plen:
        shared = make(ctx, fmt, 1, plen, kv, d)
        p = fill(shared, 30, [plen])[0]
    got = attend(cache, q, words(rows), dtype, shared, plen)
    want, tol = reference(q, p, own, rows)
    check(got, want, tol)
    # a query that sees nothing is zeros, and exactly the ones the reference leaves so
    none = (want == 0).all(-1)
    assert bool((got[none] == 0).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_prefix_in_the_same_buffer_and_later_sequences(ctx, dtype):
    """Sequence 2 of a cache is the prefix of sequences 3 .. 5; a length past max_len counts as max_len."""
    kv, d, heads = 2, 64, 6
    cache = make(ctx, "int8", 6, 260, kv, d)
    held = fill(cache, 50, [10, 10, 200, 40, 260, 129])
    q = normal(51, (3, 1, heads, d)).to(getattr(torch, dtype))
    for max_len in (None, 128, 1, 0):
        lens = [40, 260, 129]
        got = attend(cache, q, words(lens), dtype, cache, 200, pseq=2, first=3, max_len=max_len)
        want, tol = reference(q, held[2], held[3:], lens, max_len)
        check(got, want, tol, f"max_len {max_len}")
    far = attend(cache, q, words([40, -1, 2 ** 31 - 1]), dtype, cache, 200, pseq=2, first=3, max_len=100)
    want, tol = reference(q, held[2], held[3:], [40, 100, 100])
    check(far, want, tol, "lengths past the bound")


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_values_out_of_the_ordinary(ctx, fmt, dtype):
    """Rows, queries and scores of very unlike size."""
    kv, d, heads, rows = 2, 128, 4, [200, 333]
    for ks, qs in ((1e-12, 1e10), (1e8, 1e-9), (30.0, 3.0), (1e-30, 1.0), (0.0, 1.0), (1.0, 0.0)):
        cache = make(ctx, fmt, 2, 333, kv, d)

        def poke(k, v):
            k[5] *= 1e-3
            v[7] = 0.0
            v[8] *= 1e4
            v[300:310] *= 1e-20
        own = fill(cache, 60, rows, scale=ks, poke=poke)
        q = (qs * normal(61, (2, 1, heads, d))).to(getattr(torch, dtype))
        q[0, 0, 1] *= torch.exp(4 * normal(62, (d,))).to(q.dtype)
        want, tol = reference(q, empty_prefix(kv, d), own, rows)
        check(attend(cache, q, words(rows), dtype), want, tol, f"scale {ks}, {qs}")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores_that_climb(ctx, dtype):
    """Each tile's scores above the last's, far apart: the running reference moves in every tile."""
    kv, d, heads, n = 1, 64, 3, 1500
    cache = make(ctx, "int8", 1, n, kv, d)

    def poke(k, v):
        k[:] = 0.0
        k[:, 0, 0] = torch.arange(n, device="cuda") * 0.5
        k[:, 0, 1] = -torch.arange(n, device="cuda") * 0.5
    own = fill(cache, 70, [n], poke=poke)
    q = torch.zeros((1, 1, heads, d), device="cuda")
    q[0, 0, 0, 0], q[0, 0, 1, 1], q[0, 0, 2, 0] = 2.0, 2.0, 100.0
    q = q.to(getattr(torch, dtype))
    want, tol = reference(q, empty_prefix(kv, d), own, [n])
    check(attend(cache, q, words([n]), dtype), want, tol)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_rows_that_are_no_numbers(ctx, fmt):
    """A NaN row is NaN for the queries that see it, and nothing to the others; a NaN query is NaN alone."""
    kv, d, heads, sq = 2, 64, 4, 6
    for into in ("k", "v"):
        cache = make(ctx, fmt, 2, 100, kv, d)

        def poke(k, v):
            (k if into == "k" else v)[99 - 2, 1] = float("nan")  # sequence 0's row 97, kv head 1
        own = fill(cache, 80, [100, 90], poke=poke)
        q = normal(81, (2, sq, heads, d))
        q[1, 3, 2, 5] = float("inf")
        got = attend(cache, q, words([100, 90]), "float32")
        nan = torch.zeros((2, sq, heads), dtype=torch.bool, device="cuda")
        nan[0, 3:, 2:] = True  # query t sees rows 0 .. 94 + t
        nan[1, 3, 2] = True
        assert bool(got[nan].isnan().all()) and not bool(got[~nan].isnan().any())
        q[1, 3, 2, 5] = 0.0
        own = [tuple(x.nan_to_num(0.0) for x in pair) for pair in own]  # weight 0 for the rest: 0 in float64 too
        want, tol = reference(q, empty_prefix(kv, d), own, [100, 90])
        fine = ~nan[..., None].expand_as(got)
        check(got[fine], want[fine], tol[fine])


def test_graph_follows_the_device_words(ctx):
    """A step captured once -- rows written, lengths advanced, attention behind a prefix -- and replayed: every replay
    the eager call's result, bit for bit, with eager work between; two captured graphs keep their own workspaces."""
    from quantibbler_amd.gpu import advance_positions_dev

    n, kv, heads, d, cap, plen = 3, 2, 8, 64, 200, 333
    shared = make(ctx, "int8", 1, plen, kv, d)
    fill(shared, 90, [plen])
    lens = [60, 0, 127]
    rows = torch.empty((2, n, kv, d), device="cuda")
    graphs = []
    for g in range(2):
        cache = make(ctx, "int8", n, cap, kv, d)
        fill(cache, 91 + g, lens)
        q, out = torch.empty((n, 1, heads, d), device="cuda"), torch.empty((n, 1, heads, d), device="cuda")
        at = words(lens)
        need = cache.attention_workspace_size(heads, n, prefix_len=plen)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")

        def step(cache=cache, q=q, out=out, at=at, ws=ws, need=need):
            s = torch.cuda.current_stream()
            cache.write_dev(rows[0], rows[1], "float32", at, n, stream=s)
            advance_positions_dev(ctx, at, n, s)
            cache.attention_dev(q, "float32", heads, at, out, ws, need, prefix=shared, prefix_len=plen, stream=s)

        rows.copy_(normal(1, rows.shape))
        q.copy_(normal(2, q.shape))
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append((graph, cache, q, out, at))
    for rep in range(5):
        for g, (graph, cache, q, out, at) in enumerate(graphs):
            rows.copy_(normal(100 + rep, rows.shape))
            q.copy_(normal(200 + 10 * g + rep, q.shape))
            graph.replay()
            torch.cuda.synchronize()
            assert at.tolist() == [x + 2 + rep for x in lens]
            want = attend(cache, q, at, "float32", shared, plen)
            torch.cuda.synchronize()
            assert out.cpu().numpy().tobytes() == want.cpu().numpy().tobytes()
    del graphs


def test_same_answer_every_time_and_on_any_stream(ctx):
    n, kv, heads, d = 9, 2, 16, 128
    rows = [37 * i for i in range(n)]
    cache, shared = make(ctx, "fp8", n, 300, kv, d), make(ctx, "fp8", 1, 900, kv, d)
    fill(cache, 110, rows)
    fill(shared, 111, [900])
    q = normal(112, (n, 1, heads, d)).to(torch.bfloat16)
    lens = words(rows)
    first = attend(cache, q, lens, "bfloat16", shared, 900)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(attend(cache, q, lens, "bfloat16", shared, 900, stream=s))
    torch.cuda.synchronize()
    for o in outs + [attend(cache, q, lens, "bfloat16", shared, 900)]:
        assert torch.equal(o, first)


def test_a_sequence_alone_or_in_the_batch(ctx):
    """What other sequences hold does not enter a row: alone, the same sequence agrees to the tolerance of a sum in
    another order (both within it of float64)."""
    n, kv, heads, d = 4, 2, 8, 64
    rows = [300, 7, 150, 64]
    cache = make(ctx, "int8", n, 300, kv, d)
    own = fill(cache, 120, rows)
    q = normal(121, (n, 1, heads, d))
    want, tol = reference(q, empty_prefix(kv, d), own, rows)
    check(attend(cache, q, words(rows), "float32"), want, tol)
    for i in range(n):
        check(attend(cache, q[i:i + 1].contiguous(), words(rows[i:i + 1]), "float32", first=i), want[i:i + 1],
              tol[i:i + 1])


@pytest.mark.parametrize("n,heads,kv,d", [(1, 2, 2, 64), (9, 4, 1, 128)])
def test_a_long_prefix(ctx, n, heads, kv, d):
    """More key tiles than there are splits, by far: one row tile of 16 and one of 64."""
    plen = 100003
    shared, cache = make(ctx, "fp8", 1, plen, kv, d), make(ctx, "fp8", n, 70, kv, d)
    p = fill(shared, 150, [plen])[0]
    rows = [70 - i for i in range(n)]
    own = fill(cache, 151, rows)
    q = normal(152, (n, 1, heads, d))
    want, tol = reference(q, p, own, rows)
    check(attend(cache, q, words(rows), "float32", shared, plen), want, tol)


def test_offsets_past_32_bits(ctx):
    """The last sequence of a cache of eleven gigabytes."""
    n, cap, kv, d, heads, rows = 40, 131072, 8, 128, 16, 500
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    cache = make(ctx, "int8", n, cap, kv, d, poison=False)
    assert cache.buffer.numel() > 10 << 30
    own = fill(cache, 130, [rows], first=n - 1)
    q = normal(131, (1, 1, heads, d))
    got = attend(cache, q, words([rows]), "float32", first=n - 1)
    want, tol = reference(q, empty_prefix(kv, d), own, [rows])
    check(got, want, tol)
    # and its last rows
    k = normal(132, (3, kv, d))
    cache.write_dev(k, k, "float32", words([cap - 3]), 3, first_seq=n - 1, n_seqs=1)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    cache.read_dev(ko, vo, "float32", words([cap - 3]), 3, first_seq=n - 1, n_seqs=1)
    top = k.abs().amax(-1, keepdim=True)
    assert bool(((ko - k).abs() <= top / 127 * 0.5001).all()) and torch.equal(ko, vo)


def test_step_end_to_end(ctx):
    """A decode step as it is used: a fused projection's keys and values into the cache, attention behind the prefix,
    an lm_head, log probabilities -- against float64 on the read-back cache and the head's own logits."""
    from quantibbler_amd import LmHead
    from quantibbler_amd.gpu import logprobs_dev, logprobs_workspace_size

    n, kv, heads, d, plen, vocab = 5, 2, 4, 64, 100, 777
    shared, cache = make(ctx, "int8", 1, plen, kv, d), make(ctx, "int8", n, 50, kv, d)
    p = fill(shared, 140, [plen])[0]
    lens = [0, 3, 49, 20, 11]
    fill(cache, 141, lens)
    qkv = normal(142, (n, (heads + 2 * kv) * d))
    at = words(lens)
    width = qkv.stride(0)
    cache.write_dev(qkv[:, heads * d:], qkv[:, (heads + kv) * d:], "float32", at, n, row_stride=width)
    now = [x + 1 for x in lens]
    q = qkv[:, :heads * d].reshape(n, 1, heads, d).contiguous()
    out = attend(cache, q, words(now), "float32", shared, plen)
    total = sum(now)
    ko = torch.empty((total, kv, d), device="cuda")
    vo = torch.empty_like(ko)
    cache.read_dev(ko, vo, "float32", words([0] * n), total, row_start=words(np.concatenate([[0], np.cumsum(now)])))
    own, s = [], 0
    for r in now:
        own.append((ko[s:s + r].double(), vo[s:s + r].double()))
        s += r
    want, tol = reference(q, p, own, now)
    check(out, want, tol)
    rows = normal(143, (vocab, heads * d)).cpu().numpy() * 0.1
    head = LmHead.from_rows(ctx, rows)
    logits = torch.empty((n, vocab), device="cuda")
    head.logits_dev(out, n, logits)
    lp, ent = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    need = logprobs_workspace_size(n, vocab, 0)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    targets = words([3, 700, 776, 0, 50])
    logprobs_dev(ctx, logits, n, vocab, targets, lp, ent, ws, need)
    torch.cuda.synchronize()
    ref = torch.log_softmax(logits.double(), -1)
    # magnitudes of logits and their spread stay below 30: 64-fold roundings of them
    assert bool(((lp.double() - ref.gather(1, targets.long()[:, None])[:, 0]).abs() <= 64 * 30 * EPS).all())
    assert bool(((ent.double() + (ref.exp() * ref).sum(-1)).abs() <= 64 * 30 * EPS).all())
    head.close()
