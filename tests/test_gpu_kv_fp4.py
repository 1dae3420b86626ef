"""GPU: the 4-bit KV cache -- rows in and out bit for bit against the
definition, and attention over it against float64 on the values it stands for,
with the cases and tolerances of the 8-bit formats (code times multiplier is
exact in fp16, so the cache's only rounding is the one at the write, and the
attention's are those that test_gpu_attention_kv counts).

A = max(max |x|, 2^-100), m = e4m3(largest |x| of 32 channels (448 (1 / A))),
code = e2m1((x (2688 (1 / A))) (1 / m)), scale = A (1 / 2688), value =
(code m) scale, every step rounded to f32."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import test_gpu_attention_kv as att
import test_gpu_kv_cache as kvc
import test_gpu_kv_extremes as ext
import test_gpu_kv_many as many
from quantibbler_amd import GpuContext, KvCache

words, normal = att.words, att.normal
F = np.float32
BOTH = pytest.mark.parametrize("dtype", ["float32", "bfloat16"])


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


def nearest(x, bits, least):
    """float64: the nearest number of that many bits behind the leading one, the even one at a tie, no finer below
    2^least."""
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** least))) - bits)
    return np.round(x / step) * step


def stored(x, fmt="fp4"):
    """numpy: the values rows [..][d] stand for, f32."""
    assert fmt == "fp4"
    x = np.asarray(x, F)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    x = np.where(bad, F(0), x).astype(F)
    A = np.maximum(np.abs(x).max(-1, keepdims=True), F(2.0 ** -100))
    per = F(1) / A
    out = np.empty_like(x)
    for c in range(0, x.shape[-1], 32):
        part = x[..., c:c + 32]
        m = nearest((np.abs(part).max(-1, keepdims=True) * (F(448) * per)).astype(np.float64), 3, -6).astype(F)
        with np.errstate(divide="ignore"):
            by = np.where(m > 0, F(1) / m, F(0)).astype(F)
        z = ((part * (F(2688) * per)) * by).astype(np.float64)
        code = np.clip(nearest(z, 1, 0), -6.0, 6.0)
        out[..., c:c + 32] = (code.astype(F) * m) * (A * (F(1) / F(2688)))
    return np.where(bad, F("nan"), out).astype(F)


@pytest.fixture(autouse=True)
def definition(monkeypatch):
    monkeypatch.setattr(kvc, "stored", stored)


# ---- rows ----------------------------------------------------------------------

@BOTH
@pytest.mark.parametrize("n,kv,d,rows,at,cap", kvc.CASES + [(3, 2, 48, [2, 3, 1], [1, 0, 5], 9),
                                                           (64, 8, 128, [1] * 64, list(range(64)), 70)])
def test_write_and_read(ctx, dtype, n, kv, d, rows, at, cap):
    kvc.test_write_and_read(ctx, "fp4", dtype, n, kv, d, rows, at, cap)


@BOTH
@pytest.mark.parametrize("n,kv,d,rows,at,cap", [c for c in kvc.CASES if many.by_tiles(sum(c[3]), 4097, c[0], c[2])] +
                         [(1, 1, 208, [64], [0], 64), (1, 1, 48, [65], [63], 128), (2, 1, 144, [4, 4], [62, 0], 66),
                          (3, 1, 96, [3, 70, 1], [1, 33, 64], 104), (2, 1, 16, [200, 333], [5, 31], 400)])
def test_rows_that_fill_the_card(ctx, dtype, n, kv, d, rows, at, cap):
    many.test_rows_by_tiles(ctx, "fp4", dtype, n, kv, d, rows, at, cap)


def test_every_code_and_tie(ctx):
    """Ties between codes and between multipliers, both sides of them, and every power of two below: A is a power of
    two, so that a group's multiplier and codes are the nearest to numbers that float32 holds."""
    edge = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], F)
    mults = np.array([m * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8, 16) if m * 2.0 ** (e - 3) <= 448], F)
    rows = []
    for m in np.concatenate([mults, np.arange(1, 8).astype(F) * F(2.0 ** -9)]):
        for top in (F(6) * m, np.nextafter(F(6) * m, F(1e9)), F(6.2) * m, F(6.4) * m, F(5.7) * m):
            group = np.zeros(32, F)
            group[:8], group[8:16], group[16] = edge * m, -edge * m, top
            rows.append(np.concatenate([np.full(1, 2688, F), np.zeros(31, F), group,
                                        np.nextafter(group, F(1e9)), np.nextafter(group, F(-1e9))]))
    x = np.ascontiguousarray(np.stack(rows)[:, None, :])
    for scale in (1.0, 2.0 ** -90, 2.0 ** 100, 1.37):
        t = torch.from_numpy((x * F(scale)).astype(F)).cuda()
        cache = kvc.make(ctx, "fp4", 1, len(x), 1, 128)
        cache.write_dev(t, t, "float32", words([0]), len(x))
        ko, vo = torch.empty_like(t), torch.empty_like(t)
        cache.read_dev(ko, vo, "float32", words([0]), len(x))
        want = stored(t.cpu().numpy())
        kvc.check(ko, want, f"key {scale}")
        kvc.check(vo, want, f"value {scale}")


def test_error_of_a_row(ctx):
    """What the format promises: half a step of the code (1/4, 1/2 or 1 of the multiplier by size) and, past 6, the 2^-4
    that a multiplier may be short of its group's largest."""
    x = normal(1, (500, 3, 128)) * torch.exp(normal(2, (500, 3, 1)))
    cache = kvc.make(ctx, "fp4", 1, 500, 3, 128)
    cache.write_dev(x, x, "float32", words([0]), 500)
    ko, vo = torch.empty_like(x), torch.empty_like(x)
    cache.read_dev(ko, vo, "float32", words([0]), 500)
    assert torch.equal(ko, vo)
    g, e = x.view(500, 3, 4, 32), (ko - x).abs().view(500, 3, 4, 32)
    top = g.abs().amax(-1, keepdim=True)
    assert bool((e <= top * (1 / 6 + 2.0 ** -4)).all())
    assert 0.05 < float((ko - x).norm() / x.norm()) < 0.15


def test_not_finite_rows(ctx):
    kvc.test_not_finite_rows(ctx, "fp4")


@BOTH
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_fused_rows(ctx, dtype, shift):
    kvc.test_fused_rows(ctx, "fp4", dtype, shift)
    many.test_fused_rows_by_tiles(ctx, "fp4", dtype, shift)


def test_rows_left_alone(ctx):
    kvc.test_rows_left_alone(ctx, "fp4")


@BOTH
def test_rows_left_alone_among_many(ctx, dtype):
    many.test_rows_left_alone_by_tiles(ctx, "fp4", dtype)


@pytest.mark.parametrize("kv", [3, 200])
def test_rows_written_a_few_at_a_time(ctx, kv):
    """One to five rows of each of eight sequences a call, beside each other in a byte, a tile and across tiles: what
    earlier calls wrote stays."""
    rng = np.random.default_rng(8)
    n, d, cap = 8, 48, 150
    cache = kvc.make(ctx, "fp4", n, cap, kv, d)
    x = torch.from_numpy(kvc.rows_of(rng, n * cap, kv, d)).cuda().view(n, cap, kv, d)
    at, call = [int(v) for v in rng.integers(0, 3, n)], 0
    first = list(at)
    while max(at) + 5 < cap:
        step = [1] * n if call % 3 == 0 else [int(v) for v in rng.integers(0, 6, n)]
        rows = torch.cat([x[i, at[i]:at[i] + step[i]] for i in range(n)])
        starts = None if call % 3 == 0 else words(np.concatenate([[0], np.cumsum(step)]))
        cache.write_dev(rows, rows, "float32", words(at), len(rows), row_start=starts)
        at, call = [a + s for a, s in zip(at, step)], call + 1
    for i in range(n):
        m = at[i] - first[i]
        ko, vo = torch.empty((m, kv, d), device="cuda"), torch.empty((m, kv, d), device="cuda")
        cache.read_dev(ko, vo, "float32", words([first[i]]), m, first_seq=i, n_seqs=1)
        want = stored(x[i, first[i]:at[i]].cpu().numpy())
        kvc.check(ko, want, f"key {i}")
        kvc.check(vo, want, f"value {i}")


@pytest.mark.parametrize("d", [48, 128])
def test_rows_written_by_parts_of_tiles(ctx, d):
    """Eight rows a sequence and more, as tiles go, from any row of a tile to any: what earlier calls wrote stays, in the
    other half of a byte too."""
    rng = np.random.default_rng(9)
    n, kv, cap = 3, 180, 210
    cache = kvc.make(ctx, "fp4", n, cap, kv, d)
    x = torch.from_numpy(kvc.rows_of(rng, n * cap, kv, d)).cuda().view(n, cap, kv, d)
    at = [0, 3, 62]
    first = list(at)
    while max(at) + 33 < cap:
        step = [0, 0, 0]
        while sum(step) < 24:
            step = [int(v) for v in rng.integers(0, 34, n)]
        rows = torch.cat([x[i, at[i]:at[i] + step[i]] for i in range(n)])
        cache.write_dev(rows, rows, "float32", words(at), len(rows), row_start=words(np.concatenate([[0], np.cumsum(step)])))
        at = [a + s for a, s in zip(at, step)]
    for i in range(n):
        m = at[i] - first[i]
        ko, vo = torch.empty((m, kv, d), device="cuda"), torch.empty((m, kv, d), device="cuda")
        cache.read_dev(ko, vo, "float32", words([first[i]]), m, first_seq=i, n_seqs=1)
        want = stored(x[i, first[i]:at[i]].cpu().numpy())
        kvc.check(ko, want, f"key {i}")
        kvc.check(vo, want, f"value {i}")


@pytest.mark.parametrize("kv", [1, 400])
def test_row_starts_that_say_nothing_sensible(ctx, kv):
    d, cap = 16, 40
    size = KvCache.size("fp4", 2, cap, kv, d)
    buf = torch.zeros(size + 4096, dtype=torch.uint8, device="cuda")
    cache = KvCache(ctx, "fp4", 2, cap, kv, d, buf)
    x = torch.ones((30, kv, d), device="cuda")
    for starts, at in (([20, 10, 0], [0, 0]), ([-1, -5, -9], [0, 0]), ([5, 40, 30], [-1, -2]), ([0, 15, 30], [39, 1000])):
        back = torch.full((2, 31, kv, d), 5.0, device="cuda")
        cache.write_dev(x, x, "float32", words(at), 30, row_start=words(starts))
        cache.read_dev(back[0], back[1], "float32", words(at), 30, row_start=words(starts))
        assert bool((back[:, 30] == 5.0).all())
    torch.cuda.synchronize()
    assert int(buf[size:].sum()) == 0


def test_offsets_past_32_bits(ctx):
    """The last sequence of a cache of six gigabytes: its rows, and attention over them."""
    n, cap, kv, d, heads, rows = 40, 131072, 8, 128, 16, 500
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB of device memory")
    cache = att.make(ctx, "fp4", n, cap, kv, d, poison=False)
    assert cache.buffer.numel() > 5 << 30
    own = att.fill(cache, 130, [rows], first=n - 1)
    q = normal(131, (1, 1, heads, d))
    want, tol = att.reference(q, att.empty_prefix(kv, d), own, [rows])
    att.check(att.attend(cache, q, words([rows]), "float32", first=n - 1), want, tol)
    k = normal(132, (3, kv, d))
    cache.write_dev(k, k, "float32", words([cap - 3]), 3, first_seq=n - 1, n_seqs=1)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    cache.read_dev(ko, vo, "float32", words([cap - 3]), 3, first_seq=n - 1, n_seqs=1)
    kvc.check(ko, stored(k.cpu().numpy()), "key")
    assert torch.equal(ko, vo)


# ---- attention -------------------------------------------------------------------

@BOTH
@pytest.mark.parametrize("n,heads,kv,d,sq,rows,plen", att.SHAPES)
def test_attention(ctx, dtype, n, heads, kv, d, sq, rows, plen):
    att.test_against_float64(ctx, "fp4", dtype, n, heads, kv, d, sq, rows, plen)


@BOTH
@pytest.mark.parametrize("n,heads,kv,d,sq,rows,plen", many.SHAPES)
def test_attention_that_fills_the_card(ctx, dtype, n, heads, kv, d, sq, rows, plen):
    many.test_attention_against_float64(ctx, "fp4", dtype, n, heads, kv, d, sq, rows, plen)


# bodies of 64 rows as this format takes them, and splits of a prefix by what they cost
WIDE = [(4, 64, 64, 256, 64, [64, 65, 130, 90], 64), (6, 64, 64, 240, 33, [33, 34, 200, 3, 0, 65], 0),
        (1, 256, 256, 256, 70, [90], 30), (2, 128, 128, 128, 80, [80, 900], 0), (1, 256, 256, 64, 70, [600], 100),
        (2, 96, 96, 112, 100, [513, 700], 65)]
LONG = [(16, 8, 8, 80, 5, [5 + 3 * i for i in range(16)], 4001), (33, 35, 5, 80, 2, [2 + i % 7 for i in range(33)], 8200),
        (20, 32, 8, 128, 4, [4 + 40 * i for i in range(20)], 5001), (2, 8, 2, 256, 9, [9, 300], 9000)]


@BOTH
@pytest.mark.parametrize("n,heads,kv,d,sq,rows,plen", WIDE + LONG)
def test_attention_by_64_rows_and_by_long_prefixes(ctx, dtype, n, heads, kv, d, sq, rows, plen):
    many.test_attention_against_float64(ctx, "fp4", dtype, n, heads, kv, d, sq, rows, plen)


@BOTH
def test_the_ends_of_the_range_by_64_rows_of_256_channels(ctx, dtype):
    shape = (1, 256, 256, 256, 70, [90], 30)
    ext.test_queries_near_the_bottom_of_the_range(ctx, "fp4", dtype, shape)
    ext.test_keys_near_the_top_of_the_range(ctx, "fp4", dtype, shape)
    ext.test_values_near_the_top_of_the_range(ctx, "fp4", dtype, shape)
    ext.test_a_large_value_of_next_to_no_weight(ctx, "fp4", dtype, shape, -1)
    ext.test_a_value_that_only_the_last_query_sees(ctx, "fp4", dtype, shape, 45)
    ext.test_scores_past_the_exponents_range(ctx, "fp4", dtype, shape, 1e7)


@BOTH
def test_values_out_of_the_ordinary(ctx, dtype):
    att.test_values_out_of_the_ordinary(ctx, "fp4", dtype)
    many.test_values_out_of_the_ordinary(ctx, "fp4", dtype)


def test_rows_that_are_no_numbers(ctx):
    att.test_rows_that_are_no_numbers(ctx, "fp4")
    for into in ("k", "v"):
        many.test_rows_that_are_no_numbers(ctx, "fp4", into)


@BOTH
@pytest.mark.parametrize("shape", ext.SHAPES)
def test_sizes_near_the_ends_of_the_range(ctx, dtype, shape):
    ext.test_queries_near_the_bottom_of_the_range(ctx, "fp4", dtype, shape)
    ext.test_keys_near_the_top_of_the_range(ctx, "fp4", dtype, shape)
    ext.test_values_near_the_top_of_the_range(ctx, "fp4", dtype, shape)


@BOTH
@pytest.mark.parametrize("shape", ext.SHAPES)
def test_contributions_of_unlike_size(ctx, dtype, shape):
    for where in (0, 7, -1):
        ext.test_a_large_value_of_next_to_no_weight(ctx, "fp4", dtype, shape, where)
    if shape[4] > 1:
        for power in (20, 45, 100):
            ext.test_a_value_that_only_the_last_query_sees(ctx, "fp4", dtype, shape, power)


@BOTH
@pytest.mark.parametrize("shape", ext.SHAPES)
@pytest.mark.parametrize("size", [3e4, 1e7, 1e14])
def test_scores_past_the_exponents_range(ctx, dtype, shape, size):
    ext.test_scores_past_the_exponents_range(ctx, "fp4", dtype, shape, size)


def test_replays_follow_the_device_words(ctx):
    """A step's rows and attention captured once and replayed at later positions: the eager calls' result, bit for bit."""
    n, kv, heads, d, cap, plen = 3, 2, 8, 80, 200, 333
    shared, cache = att.make(ctx, "fp4", 1, plen, kv, d), att.make(ctx, "fp4", n, cap, kv, d)
    att.fill(shared, 90, [plen])
    att.fill(cache, 91, [61, 0, 127])
    rows, q = torch.empty((2, n, kv, d), device="cuda"), torch.empty((n, 1, heads, d), device="cuda")
    at, lens, out = words([61, 0, 127]), words([62, 1, 128]), torch.empty_like(q)
    need = cache.attention_workspace_size(heads, n, prefix_len=plen)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream()
        cache.write_dev(rows[0], rows[1], "float32", at, n, stream=s)
        cache.attention_dev(q, "float32", heads, lens, out, ws, need, prefix=shared, prefix_len=plen, stream=s)

    rows.normal_()
    q.normal_()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rep in range(5):
        rows.copy_(normal(rep, rows.shape))
        q.copy_(normal(50 + rep, q.shape))
        at += 1
        lens += 1
        graph.replay()
        torch.cuda.synchronize()
        want = att.attend(cache, q, lens, "float32", shared, plen)
        ko, vo = torch.empty_like(rows[0]), torch.empty_like(rows[0])
        cache.read_dev(ko, vo, "float32", at, n)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        kvc.check(ko, stored(rows[0].cpu().numpy()), "key")
        kvc.check(vo, stored(rows[1].cpu().numpy()), "value")
    del graph
