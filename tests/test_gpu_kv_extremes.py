"""GPU: attention over the 8-bit KV cache where keys, values and queries are of
very unlike size, in every body (16 and 64 query rows, own rows and prefix),
against float64 on the values the cache stands for.

Tolerance as test_gpu_attention_kv's, with everything taken over the rows a
query sees alone: a weight below 2^-26 of the query's largest weight times
value scale is a step of fp16's subnormals, and is off by at most 2^-36 of it
(half a step, 2^-25, where that largest stands between 2^11 and 2^12, or
higher)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import test_gpu_attention_kv as att
from quantibbler_amd import GpuContext

EPS = att.EPS
words, normal = att.words, att.normal


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


def reference(q, prefix, own, lens):
    """float64 outputs and their tolerances (without the output's rounding)."""
    n, sq, heads, d = q.shape
    f32 = q.dtype == torch.float32
    q64, scale = q.double(), d ** -0.5
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for b in range(n):
        k = torch.cat([prefix[0], own[b][0][:lens[b]]])
        v = torch.cat([prefix[1], own[b][1][:lens[b]]])
        p, kv, m = prefix[0].shape[0], k.shape[1], k.shape[0]
        last = p + lens[b] - sq + 1 + torch.arange(sq, device="cuda")[:, None]
        index = torch.arange(m, device="cuda")[None]
        seen = (index < p) | (index < last)
        none = ~seen.any(-1)
        for h in range(heads):
            j = h // (heads // kv)
            kk, vv, qq = k[:, j], v[:, j], q64[b, :, h]
            s = torch.where(seen, (qq @ kk.t().contiguous()) * scale, torch.full_like(seen, -torch.inf, dtype=torch.float64))
            w = s.softmax(-1)
            w[none] = 0.0
            out[b, :, h] = w @ vv
            mass = torch.where(seen, qq.abs() @ kk.abs().t().contiguous(), 0.0).amax(-1, keepdim=True)
            low = torch.where(seen, kk.abs().sum(-1)[None], 0.0).amax(-1, keepdim=True)
            bound = scale * (((d + 8) * EPS + (2.0 ** -23 if f32 else 0)) * mass +
                             2.0 ** -28 * qq.abs().amax(-1, keepdim=True) * low)
            rel = 2 * bound + (2.0 ** -22 if f32 else 2.0 ** -11) + (2 * m + 70) * EPS
            most = (w * vv.abs().amax(-1)[None]).amax(-1, keepdim=True)
            tol[b, :, h] = rel * (w @ vv.abs()) + m * 2.0 ** -36 * most
    return out, tol


# n, heads, kv heads, d, queries, own rows, prefix: own rows by 16 and by 64, the prefix by 16 and by 64
SHAPES = [(1, 4, 2, 64, 5, [90], 0), (2, 4, 2, 128, 5, [90, 300], 150), (1, 4, 1, 256, 3, [70], 40),
          (1, 8, 2, 80, 1, [2000], 0), (1, 256, 256, 64, 70, [200], 0), (1, 128, 128, 128, 70, [90], 100),
          (1, 64, 64, 256, 70, [90], 30), (17, 64, 16, 128, 1, [9 + i for i in range(17)], 500)]


def both(ctx, fmt, shape, poke=None, poke_prefix=None):
    n, heads, kv, d, sq, rows, plen = shape
    cache = att.make(ctx, fmt, n, max(rows), kv, d)
    own = att.fill(cache, 10, rows, poke=poke)
    shared, p = None, att.empty_prefix(kv, d)
    if plen:
        shared = att.make(ctx, fmt, 1, plen, kv, d)
        p = att.fill(shared, 30, [plen], poke=poke_prefix or poke)[0]
    return cache, own, shared, p


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_queries_near_the_bottom_of_the_range(ctx, fmt, dtype, shape):
    """Queries of 1e-36 against keys of 2e34: the scores are ordinary numbers, and a query keeps its bits."""
    n, heads, kv, d, sq, rows, plen = shape

    def poke(k, v):
        k *= 2e34
    cache, own, shared, p = both(ctx, fmt, shape, poke)
    q = (1e-36 * normal(n + d, (n, sq, heads, d))).to(getattr(torch, dtype))
    want, tol = reference(q, p, own, rows)
    att.check(att.attend(cache, q, words(rows), dtype, shared, plen), want, tol)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_keys_near_the_top_of_the_range(ctx, fmt, dtype, shape):
    """Keys of 1e37 against queries of 1e-36: the scores are ordinary numbers, and so is the answer."""
    n, heads, kv, d, sq, rows, plen = shape

    def poke(k, v):
        k *= 1e37
    cache, own, shared, p = both(ctx, fmt, shape, poke)
    q = (1e-36 * normal(n + d, (n, sq, heads, d))).to(getattr(torch, dtype))
    want, tol = reference(q, p, own, rows)
    att.check(att.attend(cache, q, words(rows), dtype, shared, plen), want, tol)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,d,sq,rows", [(4, 2, 64, 3, 1), (128, 128, 128, 130, 64), (64, 64, 256, 70, 1)])
def test_a_nan_query_that_sees_nothing_is_zeros(ctx, dtype, heads, kv, d, sq, rows):
    """Query t sees own rows 0 .. rows - sq + t: the first ones none, whatever they hold."""
    cache = att.make(ctx, "int8", 1, rows, kv, d)
    own = att.fill(cache, 20, [rows])
    q = normal(21, (1, sq, heads, d)).to(getattr(torch, dtype))
    q[0, 0, 1, 3], q[0, 1, 0, 0] = float("nan"), float("inf")
    got = att.attend(cache, q, words([rows]), dtype)
    assert bool((got[0, :sq - rows] == 0).all())
    want, tol = reference(q.nan_to_num(0.0, 0.0, 0.0), att.empty_prefix(kv, d), own, [rows])
    att.check(got, want, tol)


@pytest.mark.parametrize("power", [20, 45, 100])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[4] > 1])
def test_a_value_that_only_the_last_query_sees(ctx, fmt, dtype, shape, power):
    """The last query's own row is 2^power times the others: the queries before it answer as if it were not there."""
    n, heads, kv, d, sq, rows, plen = shape

    def poke(k, v):
        if v.shape[0] == sum(rows):
            v[np.cumsum(rows) - 1] *= 2.0 ** power
    cache, own, shared, p = both(ctx, fmt, shape, poke)
    q = normal(n + d, (n, sq, heads, d)).to(getattr(torch, dtype))
    got = att.attend(cache, q, words(rows), dtype, shared, plen)
    want, tol = reference(q, p, own, rows)
    att.check(got, want, tol)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("where", [0, 7, -1])
def test_a_large_value_of_next_to_no_weight(ctx, fmt, dtype, shape, where):
    """A row of 1e15 whose weight is some e^-60 of the others': seen by every query, and still nothing to it."""
    n, heads, kv, d, sq, rows, plen = shape

    def poke(k, v):
        k *= 0.3
        at = where if plen or where >= 0 else 3
        if v.shape[0] != sum(rows) or not plen:
            k[at], v[at] = -60.0 * d ** -0.5, v[at] * 1e15
    cache, own, shared, p = both(ctx, fmt, shape, poke)
    q = (1.0 + 0.1 * normal(n + d, (n, sq, heads, d))).to(getattr(torch, dtype))
    want, tol = reference(q, p, own, rows)
    att.check(att.attend(cache, q, words(rows), dtype, shared, plen), want, tol)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES[:6])
def test_contributions_that_change_places(ctx, dtype, shape):
    """Scores that rise by 30 every 16 rows, twice in 48, while the values fall by 2^45 each time or rise by as much."""
    n, heads, kv, d, sq, rows, plen = shape
    for fall in (-45.0, 45.0):
        def poke(k, v):
            tile = (torch.arange(k.shape[0], device="cuda") // 16 % 3).float()[:, None, None]
            k.mul_(0.1).add_(tile * 30.0 * d ** -0.5)
            v.mul_(torch.exp2(tile * fall))
        cache, own, shared, p = both(ctx, "int8", shape, poke)
        q = (1.0 + 0.1 * normal(n + d, (n, sq, heads, d))).to(getattr(torch, dtype))
        want, tol = reference(q, p, own, rows)
        att.check(att.attend(cache, q, words(rows), dtype, shared, plen), want, tol, f"{fall}")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[4] > 1])
def test_what_a_query_does_not_see_has_no_part(ctx, dtype, shape):
    """The last query's own row, changed: the queries before it stay as they were, bit for bit."""
    n, heads, kv, d, sq, rows, plen = shape
    q = normal(n + d, (n, sq, heads, d)).to(getattr(torch, dtype))
    got = []
    for factor in (1.0, 40.0):
        def poke(k, v):
            if v.shape[0] == sum(rows):
                k[np.cumsum(rows) - 1] *= factor
                v[np.cumsum(rows) - 1] *= factor ** 8
        cache, own, shared, p = both(ctx, "int8", shape, poke)
        got.append(att.attend(cache, q, words(rows), dtype, shared, plen))
    assert torch.equal(got[0][:, :-1], got[1][:, :-1]) and not torch.equal(got[0][:, -1], got[1][:, -1])


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_near_the_top_of_the_range(ctx, fmt, dtype, shape):
    """Values of some 1e38, all of one sign, with weights all alike: their mean is a number, if their sum is not."""
    n, heads, kv, d, sq, rows, plen = shape

    def poke(k, v):
        v.uniform_(0.7e38, 1.3e38)
    cache, own, shared, p = both(ctx, fmt, shape, poke)
    q = (0.05 * normal(n + d, (n, sq, heads, d))).to(getattr(torch, dtype))
    want, tol = reference(q, p, own, rows)
    att.check(att.attend(cache, q, words(rows), dtype, shared, plen), want, tol)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [3e4, 1e7, 1e14])
def test_scores_past_the_exponents_range(ctx, fmt, dtype, shape, size):
    """Scores of 1e9, 1e14 and 1e28: the likeliest key has all the weight, and its value is the answer (where float64
    tells it from the next by more than the scores' own roundings)."""
    n, heads, kv, d, sq, rows, plen = shape

    def poke(k, v):
        k *= size
    cache, own, shared, p = both(ctx, fmt, shape, poke)
    q = (size * normal(n + d, (n, sq, heads, d))).to(getattr(torch, dtype))
    got = att.attend(cache, q, words(rows), dtype, shared, plen).double()
    assert bool(got.isfinite().all())
    told = 0
    for b in range(n):
        k, v = (torch.cat([x, y[:rows[b]]]) for x, y in zip(p, own[b]))
        index = torch.arange(len(k), device="cuda")[None]
        seen = index < plen + rows[b] - sq + 1 + torch.arange(sq, device="cuda")[:, None]
        for h in range(heads):
            kk, vv, qq = k[:, h // (heads // kv)], v[:, h // (heads // kv)], q[b, :, h].double()
            s = torch.where(seen, qq @ kk.t().contiguous(), torch.full_like(seen, -torch.inf, dtype=torch.float64))
            two, at = s.topk(2, -1)
            # a score is off by (d + 8) eps and, f32, 2^-23 of its terms; fp16's smallest step against the largest channel
            off = (((d + 8) * EPS + 2.0 ** -23) * (qq.abs() @ kk.abs().t().contiguous()).amax(-1) +
                   2.0 ** -28 * qq.abs().amax(-1) * kk.abs().sum(-1).max())
            clear = two[:, 0] - two[:, 1] > 2 * off + 60.0 * d ** 0.5
            told += int(clear.sum())
            want = vv[at[:, 0]]
            # the weight is 1 and rides with the value's scale: rounded as a weight is (fp16's half step 2^-11, in two
            # halves 2^-22), the exact product with the code by some f32 roundings on the way, and as an output
            step = 2.0 ** -8 + 2.0 ** -11 if dtype == "bfloat16" else EPS + 2.0 ** -22
            assert bool(((got[b, :, h] - want).abs() <= (step + 70 * EPS) * want.abs())[clear].all()), f"row {b} head {h}"
    assert told > n * sq * heads // 2
