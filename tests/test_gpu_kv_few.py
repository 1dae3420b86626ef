"""GPU: the 4-bit cache's attention by the body of four rows where a wave takes
more than one tile, at every width of it, and the bits that channels far below
their row's largest keep -- against float64 on the values the cache stands for.

Tolerances as test_gpu_attention_kv's and test_gpu_kv_extremes'."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import test_gpu_attention_kv as att
import test_gpu_kv_extremes as ext
from quantibbler_amd import GpuContext

BOTH = pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
words, normal, EPS = att.words, att.normal, att.EPS

# n, heads, kv heads, d, queries, own rows, prefix: up to four rows a kv head, one launch of several tiles a wave and splits
LOOPS = [(1, 4, 1, 64, 1, [1000], 0), (2, 3, 1, 48, 1, [1024, 1025], 0), (3, 4, 2, 16, 2, [257, 700, 1500], 70),
         (1, 1, 1, 64, 3, [2200], 0), (2, 2, 2, 32, 4, [1300, 4], 130), (1, 4, 1, 128, 1, [769], 0),
         (1, 4, 1, 112, 1, [1100], 33), (1, 4, 1, 256, 1, [512], 0), (2, 4, 1, 240, 1, [513, 900], 65),
         (3, 8, 2, 256, 1, [2300, 1, 600], 0), (1, 3, 3, 256, 3, [700], 300)]
FAR = [(1, 4, 1, 64, 1, [1000], 0), (2, 3, 1, 48, 1, [1024, 1025], 0), (1, 4, 1, 256, 1, [512], 0),
       (1, 4, 2, 240, 2, [900], 65), (1, 4, 1, 128, 1, [700], 0)]


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


@BOTH
@pytest.mark.parametrize("n,heads,kv,d,sq,rows,plen", LOOPS)
def test_more_than_one_tile_a_wave(ctx, dtype, n, heads, kv, d, sq, rows, plen):
    att.test_against_float64(ctx, "fp4", dtype, n, heads, kv, d, sq, rows, plen)


@BOTH
@pytest.mark.parametrize("n,heads,kv,d,sq,rows,plen", LOOPS)
def test_scores_that_climb(ctx, dtype, n, heads, kv, d, sq, rows, plen):
    """Each run of 16 rows above the last, so that references move in every tile, and values that fall or rise by as
    much: outputs are rescaled between tiles."""
    q = torch.ones((n, sq, heads, d), device="cuda").to(getattr(torch, dtype))
    for step, fall in ((0.05, 0.0), (3.0, -3.0), (3.0, 3.0)):
        def rise(k, v, step=step, fall=fall):
            first = 0
            for r in rows:
                at = torch.arange(r, device="cuda") // 16
                k[first:first + r] = (k[first:first + r] * 0.01) + (step * at / d ** 0.5).view(-1, 1, 1)
                v[first:first + r] *= torch.exp2((fall * at.double()).clamp(-60, 60)).float().view(-1, 1, 1)
                first += r
        cache = att.make(ctx, "fp4", n, max(rows), kv, d)
        own = att.fill(cache, 40, rows, poke=rise)
        shared, p = None, att.empty_prefix(kv, d)
        if plen:
            shared = att.make(ctx, "fp4", 1, plen, kv, d)
            p = att.fill(shared, 30, [plen])[0]
        want, tol = ext.reference(q, p, own, rows)
        att.check(att.attend(cache, q, words(rows), dtype, shared, plen), want, tol, f"{step}, {fall}")


@BOTH
@pytest.mark.parametrize("shape", FAR)
def test_sizes_near_the_ends_of_the_range(ctx, dtype, shape):
    ext.test_queries_near_the_bottom_of_the_range(ctx, "fp4", dtype, shape)
    ext.test_keys_near_the_top_of_the_range(ctx, "fp4", dtype, shape)
    ext.test_values_near_the_top_of_the_range(ctx, "fp4", dtype, shape)


@BOTH
@pytest.mark.parametrize("shape", FAR)
def test_contributions_of_unlike_size(ctx, dtype, shape):
    for where in (0, 7, 40 if shape[6] else 300, -1):
        ext.test_a_large_value_of_next_to_no_weight(ctx, "fp4", dtype, shape, where)
    if shape[4] > 1:
        for power in (20, 45, 100):
            ext.test_a_value_that_only_the_last_query_sees(ctx, "fp4", dtype, shape, power)


@pytest.mark.parametrize("n,heads,kv,d,sq,rows,plen", [
    (1, 4, 1, 128, 1, [1], 0), (1, 4, 1, 128, 1, [700], 0), (2, 4, 1, 64, 1, [300, 1000], 0), (1, 4, 1, 256, 1, [500], 0),
    (2, 4, 4, 96, 3, [40, 90], 0), (1, 16, 2, 128, 1, [700], 0), (2, 8, 2, 128, 5, [90, 300], 200),
    (1, 64, 64, 128, 70, [90], 100)])
def test_channels_far_below_their_rows_largest(ctx, n, heads, kv, d, sq, rows, plen):
    """f32 queries whose weight is one key's: its values come back with the bits that they have, in channels of 2^-17.5 of
    the row's largest (a multiplier of 2^-9, the smallest) as in the others; in the body of four rows with 18 bits there.

    The weight p of that key is the sum of weights too.  Its product with the scale and the multiplier, two halves
    (2^-22), products with the code in two sums, the sum's reciprocal and the join are some 15 roundings to f32, the value
    read back is one.  The body of four rows rounds 2^11 m / 2^9 and more, m the multiplier, to two fp16 halves, the
    second of which is off by half a step of 2^-24 at the least: 2^-25 / (2^2 m) of it.  A group's largest is at least a
    quarter of its row's but for `small`, so m is 112 small and more, or 2^-9."""
    small = torch.ones(d, device="cuda")
    for group, power in zip(range(0, -(-d // 32)), (0, -17.5, -6, -11, -17.5, -14, -8, -17.5)):
        small[32 * group:32 * group + 32] = 2.0 ** power
    lost = 2.0 ** -27 / (112 * small).clamp_min(2.0 ** -9) if sq * heads // kv <= 4 else torch.zeros(d, device="cuda")
    for where in (0, (plen or rows[0]) // 2, max(plen or min(rows) - sq, 0)):
        def one(k, v, where=where):
            v *= small
            k *= 0.01
            ends = [0]
            for r in rows:
                ends.append(ends[-1] + r)
            for e in ends[:-1] if len(v) == sum(rows) else [0]:
                if not plen:
                    k[e + min(where, min(rows) - sq)] = 60.0 * d ** -0.5

        def one_of_the_prefix(k, v, where=where):
            v *= small
            k *= 0.01
            k[min(where, plen - 1)] = 60.0 * d ** -0.5

        cache = att.make(ctx, "fp4", n, max(rows), kv, d)
        own = att.fill(cache, 60, rows, poke=one)
        shared, p = None, att.empty_prefix(kv, d)
        if plen:
            shared = att.make(ctx, "fp4", 1, plen, kv, d)
            p = att.fill(shared, 61, [plen], poke=one_of_the_prefix)[0]
        q = torch.full((n, sq, heads, d), 4.0, device="cuda")
        got = att.attend(cache, q, words(rows), "float32", shared, plen).double()
        for b in range(n):
            held = p[1][min(where, plen - 1)] if plen else own[b][1][min(where, min(rows) - sq)]
            want = held.repeat_interleave(heads // kv, 0).expand(sq, heads, d)
            off = (got[b] - want).abs()
            assert bool((off <= (2.0 ** -22 + lost.double() + 16 * EPS) * want.abs()).all()), \
                f"row {where} of sequence {b}: off by {float((off / want.abs().clamp_min(1e-30)).max()):.3g} of a value"


@BOTH
@pytest.mark.parametrize("fmt", ["int8", "fp8", "fp4"])
def test_calls_repeat_themselves(ctx, dtype, fmt):
    """The same call again, on a workspace that holds something else, behind other work and on another stream: the same
    bits, in every body and with splits."""
    for n, heads, kv, d, sq, rows, plen in [(32, 32, 8, 128, 1, [1076 + 32 * i for i in range(32)], 0),
                                            (16, 8, 8, 80, 5, [40 + 9 * i for i in range(16)], 4001),
                                            (64, 32, 8, 128, 1, [200 + 9 * i for i in range(64)], 3000),
                                            (1, 4, 1, 256, 1, [2000], 0), (2, 64, 64, 64, 70, [90, 200], 100)]:
        cache = att.make(ctx, fmt, n, max(rows), kv, d)
        att.fill(cache, 10, rows)
        shared = None
        if plen:
            shared = att.make(ctx, fmt, 1, plen, kv, d)
            att.fill(shared, 30, [plen])
        q = (1.5 * normal(n + d, (n, sq, heads, d))).to(getattr(torch, dtype))
        need = cache.attention_workspace_size(heads, n, seq_q=sq, prefix_len=plen)
        first, s = att.attend(cache, q, words(rows), dtype, shared, plen), torch.cuda.Stream()
        for rep in range(6):
            ws = torch.full((max(need, 16),), 17 * rep, dtype=torch.uint8, device="cuda")
            att.attend(cache, -q, words(rows), dtype, shared, plen)
            torch.cuda.synchronize()
            with torch.cuda.stream(s if rep % 2 else torch.cuda.current_stream()):
                again = att.attend(cache, q, words(rows), dtype, shared, plen, ws=ws, stream=torch.cuda.current_stream())
            torch.cuda.synchronize()
            assert torch.equal(again, first), f"{(n, heads, kv, d, sq, plen)}, {rep}"
