"""GPU: the 8-bit KV cache and its attention at sizes that fill the card --
rows by 64-row tiles, bodies of 64 query rows -- by many kv heads, so that
lengths and masks stay those where a tile can go wrong.  Against the definition
bit for bit and against float64, with the tolerances of the smaller sizes."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import test_gpu_attention_kv as att
import test_gpu_kv_cache as kvc
from quantibbler_amd import GpuContext

words, normal = kvc.words, att.normal


def by_tiles(total, kv, n, d):
    """Past 4096 rows and heads, of 512 channels a sequence and head, rows go by tiles."""
    return total * kv > 4096 and total * d // 512 >= n


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,kv,d,rows,at,cap", [c for c in kvc.CASES if by_tiles(sum(c[3]), 4097, c[0], c[2])] +
                         [(1, 1, 208, [64], [0], 64), (1, 1, 48, [65], [63], 128), (2, 1, 144, [4, 4], [62, 0], 66)])
def test_rows_by_tiles(ctx, fmt, dtype, n, kv, d, rows, at, cap):
    rng = np.random.default_rng(d + cap)
    total = sum(rows)
    kv = max(kv, 4096 // total + 1)
    assert by_tiles(total, kv, n, d)
    k, v = kvc.rows_of(rng, total, kv, d), kvc.rows_of(rng, total, kv, d)
    k[rng.random(k.shape) < 0.05] = 0.0
    k[1, 0] = 0.0
    v[2, -1] = 2.0 ** -110 * v[2, -1]
    k[0, kv // 2, 3], v[total - 1, 0, d - 1] = np.nan, np.inf
    kt, vt = torch.from_numpy(k), torch.from_numpy(v)
    if dtype == "bfloat16":
        kt, vt = kvc.bf16(k), kvc.bf16(v)
        k, v = kt.float().numpy(), vt.float().numpy()
    starts = words(np.concatenate([[0], np.cumsum(rows)]))
    cache = kvc.make(ctx, fmt, n, cap, kv, d)
    cache.write_dev(kt.cuda(), vt.cuda(), dtype, words(at), total, row_start=starts)
    for out in ("float32", "bfloat16"):
        ko = torch.empty((total, kv, d), dtype=getattr(torch, out), device="cuda")
        vo = torch.empty_like(ko)
        cache.read_dev(ko, vo, out, words(at), total, row_start=starts)
        for got, x, name in ((ko, k, "key"), (vo, v, "value")):
            want = kvc.stored(x, fmt)
            kvc.check(got, kvc.bf16(want).float().numpy() if out == "bfloat16" else want, f"{name} {out}")


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_fused_rows_by_tiles(ctx, fmt, dtype, shift):
    """Out of wider rows at any alignment, and read back into wider rows that keep the rest."""
    rng = np.random.default_rng(shift)
    n, kv, d = 37, 120, 80
    wide = torch.from_numpy(rng.standard_normal((n, 2 * kv * d + 2 * shift + 7)).astype(np.float32)).cuda()
    wide = wide.to(getattr(torch, dtype))
    cut = slice(shift, shift + kv * d), slice(shift + kv * d + 1, shift + 1 + 2 * kv * d)
    cache = kvc.make(ctx, fmt, 1, 50, kv, d)
    cache.write_dev(wide[:, cut[0]], wide[:, cut[1]], dtype, words([13]), n, row_stride=wide.stride(0))
    back = torch.full_like(wide, 7.0)
    cache.read_dev(back[:, cut[0]], back[:, cut[1]], dtype, words([13]), n, row_stride=wide.stride(0))
    rest = torch.ones(wide.shape[1], dtype=torch.bool)
    for c in cut:
        rest[c] = False
        want = torch.from_numpy(kvc.stored(wide[:, c].float().cpu().numpy().reshape(n, kv, d), fmt).reshape(n, -1))
        kvc.check(back[:, c], want.to(back.dtype).float().numpy(), dtype)
    assert bool((back[:, rest.cuda()] == 7.0).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_rows_left_alone_by_tiles(ctx, fmt, dtype):
    """Rows past the capacity or of no sequence are left out, every other byte stays, and reading them gives NaN."""
    rng = np.random.default_rng(5)
    n, kv, d, cap = 3, 110, 32, 70
    full = torch.from_numpy(kvc.rows_of(rng, n * cap, kv, d)).cuda()
    cache = kvc.make(ctx, fmt, n, cap, kv, d, fill=0)
    cache.write_dev(full, full, "float32", words([0] * n), n * cap)
    new = torch.from_numpy(kvc.rows_of(rng, 40, kv, d)).cuda()
    starts = words([2, 32, 34])
    cache.write_dev(new, new, "float32", words([50, 3]), 40, first_seq=1, n_seqs=2, row_start=starts)
    want, w = kvc.stored(full.cpu().numpy().reshape(n, cap, kv, d), fmt), kvc.stored(new.cpu().numpy(), fmt)
    want[1, 50:70], want[2, 3:5] = w[2:22], w[32:34]
    cast = (lambda x: x) if dtype == "float32" else (lambda x: kvc.bf16(x).float().numpy())
    ko = torch.empty((n * cap, kv, d), dtype=getattr(torch, dtype), device="cuda")
    vo = torch.empty_like(ko)
    cache.read_dev(ko, vo, dtype, words([0] * n), n * cap)
    kvc.check(ko.view(n, cap, kv, d), cast(want), "key")
    kvc.check(vo.view(n, cap, kv, d), cast(want), "value")
    ko, vo = (torch.zeros((40, kv, d), dtype=ko.dtype, device="cuda") for _ in range(2))
    cache.read_dev(ko, vo, dtype, words([50, 3]), 40, first_seq=1, n_seqs=2, row_start=starts)
    out = np.full((40, kv, d), np.nan, np.float32)
    out[2:22], out[32:34] = w[2:22], w[32:34]
    kvc.check(ko, cast(out), "key")
    kvc.check(vo, cast(out), "value")


@pytest.mark.parametrize("n", [61, 62, 63, 126, 127, 5000])
@pytest.mark.parametrize("even", [False, True])
def test_many_sequences_by_tiles(ctx, n, even):
    """A tile finds its sequence among few and many, empty ones between them, rows of none before and behind."""
    rng = np.random.default_rng(n)
    kv, d, cap = 1 if n > 1000 else 64, 128, 90
    lens = np.full(n, 9) if even else np.where(rng.random(n) < 0.2, 0, rng.integers(1, 17, n))
    lens[n // 2] = 9 if even else 80
    pre, post = (0, 0) if even else (70, 3)
    total = int(lens.sum()) + pre + post
    assert by_tiles(total, kv, n, d)
    x = torch.from_numpy(kvc.rows_of(rng, total, kv, d)).cuda()
    at = rng.integers(0, cap, n)
    starts = None if even else words(pre + np.concatenate([[0], np.cumsum(lens)]))
    cache = kvc.make(ctx, "int8", n, cap, kv, d)
    cache.write_dev(x, x, "float32", words(at), total, row_start=starts)
    ko, vo = torch.zeros_like(x), torch.zeros_like(x)
    cache.read_dev(ko, vo, "float32", words(at), total, row_start=starts)
    want = kvc.stored(x.cpu().numpy(), "int8")
    where = np.concatenate([np.full(pre, cap)] + [a + np.arange(r) for a, r in zip(at, lens)] + [np.full(post, cap)])
    want[where >= cap] = np.nan
    kvc.check(ko, want, "key")
    kvc.check(vo, want, "value")


def test_row_starts_that_say_nothing_sensible_by_tiles(ctx):
    kv, d, cap = 150, 64, 40
    size = kvc.KvCache.size("int8", 2, cap, kv, d)
    buf = torch.zeros(size + 4096, dtype=torch.uint8, device="cuda")
    cache = kvc.KvCache(ctx, "int8", 2, cap, kv, d, buf)
    x = torch.ones((30, kv, d), device="cuda")
    for starts, at in (([20, 10, 0], [0, 0]), ([-1, -5, -9], [0, 0]), ([5, 40, 30], [-1, -2]), ([0, 15, 30], [39, 1000])):
        back = torch.full((2, 31, kv, d), 5.0, device="cuda")
        cache.write_dev(x, x, "float32", words(at), 30, row_start=words(starts))
        cache.read_dev(back[0], back[1], "float32", words(at), 30, row_start=words(starts))
        assert bool((back[:, 30] == 5.0).all())
    torch.cuda.synchronize()
    assert int(buf[size:].sum()) == 0


# n, heads, kv heads, d, queries, own rows, prefix: bodies of 64 rows on the prefix, on own rows, on both
SHAPES = [(1, 128, 128, 128, 1, [70], 130), (17, 128, 32, 128, 1, [9 * i for i in range(17)], 300),
          (1, 128, 128, 64, 64, [80], 65), (1, 256, 256, 64, 70, [70], 0), (1, 256, 256, 32, 70, [71], 100),
          (3, 64, 64, 256, 1, [0, 1, 130], 129), (3, 64, 64, 240, 20, [20, 21, 200], 64), (3, 64, 64, 256, 20, [3, 65, 0], 0),
          (3, 64, 64, 80, 33, [33, 34, 400], 0), (3, 64, 64, 96, 33, [64, 1, 65], 4097),
          (5, 448, 64, 112, 3, [3, 65, 0, 129, 64], 63), (1, 32, 16, 128, 300, [1300], 0),
          (256, 8, 1, 96, 1, [i % 70 for i in range(256)], 200), (2, 64, 64, 128, 80, [80, 900], 0)]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,heads,kv,d,sq,rows,plen", SHAPES)
def test_attention_against_float64(ctx, fmt, dtype, n, heads, kv, d, sq, rows, plen):
    q = (1.5 * normal(n + d, (n, sq, heads, d))).to(getattr(torch, dtype))
    cache = att.make(ctx, fmt, n, max(1, max(rows)), kv, d)
    own = att.fill(cache, 10, rows)
    shared, p = None, att.empty_prefix(kv, d)
    if plen:
        shared = att.make(ctx, fmt, 1, plen, kv, d)
        p = att.fill(shared, 30, [plen])[0]
    got = att.attend(cache, q, words(rows), dtype, shared, plen)
    want, tol = att.reference(q, p, own, rows)
    att.check(got, want, tol)
    assert bool((got[(want == 0).all(-1)] == 0).all())
    assert torch.equal(att.attend(cache, q, words(rows), dtype, shared, plen), got)  # in no other order


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_scores_that_climb(ctx, dtype, where, d):
    """Each tile's scores above the last's, far apart: the running reference moves in every tile."""
    kv, n, sq = (520 if d == 64 else 128, 500, 1) if where == "prefix" else (128, 500, 129)

    def poke(k, v):
        k[:] = 0.0
        k[:, :, 0] = torch.arange(n, device="cuda")[:, None] * 0.5
        k[:, 1::2, 0] *= -1.0
    cache = att.make(ctx, "int8", 1, n, kv, d)
    q = torch.zeros((1, sq, kv, d), device="cuda")
    q[..., 0] = torch.linspace(0.0, 40.0, sq * kv, device="cuda").view(1, sq, kv)
    q = q.to(getattr(torch, dtype))
    if where == "prefix":
        shared = att.make(ctx, "int8", 1, n, kv, d)
        p, own, rows = att.fill(shared, 70, [n], poke=poke)[0], att.fill(cache, 71, [3]), [3]
    else:
        shared, p, own, rows = None, att.empty_prefix(kv, d), att.fill(cache, 70, [n], poke=poke), [n]
    want, tol = att.reference(q, p, own, rows)
    att.check(att.attend(cache, q, words(rows), dtype, shared, n if shared else 0), want, tol)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_values_out_of_the_ordinary(ctx, fmt, dtype):
    kv, d, rows, sq = 64, 128, [200, 133], 80
    for ks, qs in ((1e-12, 1e10), (1e8, 1e-9), (1e-30, 1.0), (0.0, 1.0), (1.0, 0.0)):
        cache = att.make(ctx, fmt, 2, 200, kv, d)

        def poke(k, v):
            k[5] *= 1e-3
            v[7] = 0.0
            v[8] *= 1e4
            v[300:310] *= 1e-20
        own = att.fill(cache, 60, rows, scale=ks, poke=poke)
        q = (qs * normal(61, (2, sq, kv, d))).to(getattr(torch, dtype))
        want, tol = att.reference(q, att.empty_prefix(kv, d), own, rows)
        att.check(att.attend(cache, q, words(rows), dtype), want, tol, f"scale {ks}, {qs}")


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("into", ["k", "v"])
def test_rows_that_are_no_numbers(ctx, fmt, into):
    """A NaN row is NaN for the queries that see it, and nothing to the others; a NaN query is NaN alone."""
    kv, d, sq, n = 64, 128, 130, 200

    def poke(k, v):
        (k if into == "k" else v)[n - 20, 1] = float("nan")
    cache = att.make(ctx, fmt, 1, n, kv, d)
    own = att.fill(cache, 80, [n], poke=poke)
    q = normal(81, (1, sq, kv, d))
    q[0, 3, 2, 5] = float("inf")
    got = att.attend(cache, q, words([n]), "float32")
    nan = torch.zeros((1, sq, kv), dtype=torch.bool, device="cuda")
    nan[0, sq - 20:, 1] = True  # query t sees rows 0 .. n - sq + t
    nan[0, 3, 2] = True
    assert bool(got[nan].isnan().all()) and not bool(got[~nan].isnan().any())
    q[0, 3, 2, 5] = 0.0
    own = [tuple(x.nan_to_num(0.0) for x in pair) for pair in own]
    want, tol = att.reference(q, att.empty_prefix(kv, d), own, [n])
    fine = ~nan[..., None].expand_as(got)
    att.check(got[fine], want[fine], tol[fine])


def test_lengths_past_the_bound(ctx):
    kv, d, sq = 64, 128, 80
    cache = att.make(ctx, "int8", 2, 200, kv, d)
    own = att.fill(cache, 50, [200, 150])
    q = normal(51, (2, sq, kv, d))
    got = att.attend(cache, q, words([-1, 2 ** 31 - 1]), "float32", max_len=100)
    want, tol = att.reference(q, att.empty_prefix(kv, d), own, [100, 100])
    att.check(got, want, tol)


def test_graph_replays(ctx):
    """Rows by tiles and bodies of 64 rows captured once; every replay the eager calls' result, eager work between."""
    kv, d, sq, n, plen = 64, 128, 40, 3, 200
    shared, cache = att.make(ctx, "int8", 1, plen, kv, d), att.make(ctx, "int8", n, 200, kv, d)
    att.fill(shared, 90, [plen])
    rows, q = torch.empty((2, n * sq, kv, d), device="cuda"), torch.empty((n, sq, kv, d), device="cuda")
    at, lens, out = words([0] * n), words([sq] * n), torch.empty_like(q)
    need = cache.attention_workspace_size(kv, n, seq_q=sq, prefix_len=plen)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream()
        cache.write_dev(rows[0], rows[1], "float32", at, n * sq, stream=s)
        cache.attention_dev(q, "float32", kv, lens, out, ws, need, seq_q=sq, prefix=shared, prefix_len=plen, stream=s)

    rows.normal_()
    q.normal_()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rep in range(4):
        rows.copy_(normal(rep, rows.shape))
        q.copy_(normal(50 + rep, q.shape))
        at.fill_(30 * rep)
        lens.fill_(30 * rep + sq)
        graph.replay()
        torch.cuda.synchronize()
        want = att.attend(cache, q, lens, "float32", shared, plen)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
