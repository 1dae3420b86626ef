"""GPU: rows into and out of the 8-bit KV cache, bit for bit against the
definition: scale = A (1 / L) and code = nearest(x (L (1 / A))) in f32 steps,
the value code * scale."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from quantibbler_amd import GpuContext, KvCache

LEVELS = {"int8": 127.0, "fp8": 448.0}


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


def stored(x, fmt):
    """numpy: the values rows [..][d] stand for, f32."""
    x = np.asarray(x, np.float32)
    L = np.float32(LEVELS[fmt])
    with np.errstate(invalid="ignore"):
        top = np.abs(x).max(-1, keepdims=True)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    A = np.maximum(np.where(bad, np.float32(0), top).astype(np.float32), np.float32(2.0 ** -100))
    y = (np.where(bad, np.float32(0), x) * (L * (np.float32(1) / A))).astype(np.float32).astype(np.float64)
    step = 1.0
    if fmt == "fp8":
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
    code = np.round(y / step) * step
    return np.where(bad, np.float32("nan"), code.astype(np.float32) * (A * (np.float32(1) / L))).astype(np.float32)


def words(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def make(ctx, fmt, n, cap, kv, d, fill=None):
    buf = torch.empty(KvCache.size(fmt, n, cap, kv, d), dtype=torch.uint8, device="cuda")
    buf.fill_(0xFF if fill is None else fill)  # NaN codes and scales wherever nothing was written
    return KvCache(ctx, fmt, n, cap, kv, d, buf)


def rows_of(rng, n, kv, d):
    return (rng.standard_normal((n, kv, d)) * np.exp(2 * rng.standard_normal((n, kv, 1)))).astype(np.float32)


def bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16)


def check(got, want, label):
    got, want = got.float().cpu().numpy(), np.asarray(want, np.float32)
    same = (got.view(np.uint32) == want.view(np.uint32)) | (np.isnan(got) & np.isnan(want)) | ((got == 0) & (want == 0))
    assert same.all(), f"{label}: {np.count_nonzero(~same)} values differ, first at {np.argwhere(~same)[:3].tolist()}"


CASES = [(4, 2, 64, [15, 9, 0, 14], [0, 50, 3, 60], 80), (20, 3, 128, [i % 13 for i in range(20)], [5 * i for i in range(20)], 110),
         (300, 1, 32, [17 + i % 3 for i in range(300)], [i for i in range(300)], 330), (1, 1, 16, [1], [0], 1), (1, 1, 16, [3], [61], 64), (3, 2, 64, [5, 0, 70], [7, 3, 60], 131),
         (2, 5, 80, [130, 1], [1, 63], 140), (4, 8, 128, [1, 1, 1, 1], [0, 15, 64, 1000], 1025),
         (2, 1, 256, [65, 64], [15, 0], 128), (1, 3, 240, [17], [0], 17), (2, 8, 128, [300, 211], [0, 5], 320)]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,kv,d,rows,at,cap", CASES)
def test_write_and_read(ctx, fmt, dtype, n, kv, d, rows, at, cap):
    rng = np.random.default_rng(d + cap)
    total = sum(rows)
    k, v = rows_of(rng, total, kv, d), rows_of(rng, total, kv, d)
    k[rng.random(k.shape) < 0.05] = 0.0
    if total > 2:
        k[1, 0] = 0.0                       # a head's row of zeros
        v[2, -1] = 2.0 ** -110 * v[2, -1]   # below the floor
    kt, vt = torch.from_numpy(k), torch.from_numpy(v)
    if dtype == "bfloat16":
        kt, vt = bf16(k), bf16(v)
        k, v = kt.float().numpy(), vt.float().numpy()
    starts = words(np.concatenate([[0], np.cumsum(rows)]))
    cache = make(ctx, fmt, n, cap, kv, d)
    s = torch.cuda.current_stream()
    cache.write_dev(kt.cuda(), vt.cuda(), dtype, words(at), total, row_start=starts, stream=s)
    for out in ("float32", "bfloat16"):
        ko = torch.empty((total, kv, d), dtype=getattr(torch, out), device="cuda")
        vo = torch.empty_like(ko)
        cache.read_dev(ko, vo, out, words(at), total, row_start=starts, stream=s)
        for got, x, name in ((ko, k, "key"), (vo, v, "value")):
            want = stored(x, fmt)
            check(got, bf16(want).float().numpy() if out == "bfloat16" else want, f"{name} {out}")


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_every_code_and_tie(ctx, fmt):
    """A row's largest value is L, so codes are the nearest to x itself: ties between codes, both sides of them, and
    every power of two below."""
    L = LEVELS[fmt]
    if fmt == "int8":
        edge = np.arange(-127, 127) + 0.5
    else:
        m = [j * 2.0 ** (e - 3) for e in range(-6, 9) for j in np.arange(8, 16) + 0.5] + \
            [(j + 0.5) * 2.0 ** -9 for j in range(8)]
        edge = np.array([x for x in m if x < 448] + [-x for x in m if x < 448])
    x = np.concatenate([edge, np.nextafter(edge.astype(np.float32), np.float32(1e9)),
                        np.nextafter(edge.astype(np.float32), np.float32(-1e9)),
                        2.0 ** np.arange(-40, 7)]).astype(np.float32)
    d = 128
    x = np.concatenate([x, np.zeros(-len(x) % (d - 1), np.float32)]).reshape(-1, d - 1)
    x = np.concatenate([np.full((len(x), 1), L, np.float32), x], 1)[:, None, :]
    n = len(x)
    cache = make(ctx, fmt, 1, n, 1, d)
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    cache.write_dev(t, t, "float32", words([0]), n)
    ko, vo = torch.empty_like(t), torch.empty_like(t)
    cache.read_dev(ko, vo, "float32", words([0]), n)
    check(ko, stored(x, fmt), "key")
    check(vo, stored(x, fmt), "value")


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_not_finite_rows(ctx, fmt):
    """A NaN or an infinity makes its head's row NaN and no other."""
    rng = np.random.default_rng(3)
    x = rows_of(rng, 6, 2, 64)
    x[1, 0, 5], x[2, 1, 63], x[4, 0, 0] = np.nan, np.inf, -np.inf
    cache = make(ctx, fmt, 1, 6, 2, 64)
    t = torch.from_numpy(x).cuda()
    cache.write_dev(t, t, "float32", words([0]), 6)
    ko, vo = torch.empty_like(t), torch.empty_like(t)
    cache.read_dev(ko, vo, "float32", words([0]), 6)
    want = stored(x, fmt)
    assert np.isnan(want).all(-1).sum() == 3
    check(ko, want, "key")
    check(vo, want, "value")


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_fused_rows(ctx, fmt, dtype, shift):
    """Keys and values taken out of wider rows, at any alignment, and read back into wider rows."""
    rng = np.random.default_rng(shift)
    n, kv, d = 37, 3, 80
    wide = torch.from_numpy(rng.standard_normal((n, 2 * kv * d + 2 * shift + 7)).astype(np.float32)).cuda()
    wide = wide.to(getattr(torch, dtype))
    k, v = wide[:, shift:shift + kv * d], wide[:, shift + kv * d + 1:shift + 1 + 2 * kv * d]
    cache = make(ctx, fmt, 1, 50, kv, d)
    cache.write_dev(k, v, dtype, words([13]), n, row_stride=wide.stride(0))
    back = torch.full_like(wide, 7.0)
    ko, vo = back[:, shift:shift + kv * d], back[:, shift + kv * d + 1:shift + 1 + 2 * kv * d]
    cache.read_dev(ko, vo, dtype, words([13]), n, row_stride=wide.stride(0))
    for got, x in ((ko, k), (vo, v)):
        want = torch.from_numpy(stored(x.float().cpu().numpy().reshape(n, kv, d), fmt).reshape(n, -1))
        check(got, want.to(back.dtype).float().numpy(), dtype)
    rest = torch.ones(wide.shape[1], dtype=torch.bool)
    rest[shift:shift + kv * d] = False
    rest[shift + kv * d + 1:shift + 1 + 2 * kv * d] = False
    assert bool((back[:, rest.cuda()] == 7.0).all())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_rows_left_alone(ctx, fmt):
    """Rows past the capacity and rows no sequence claims are left out; nothing else of the buffer changes: writing one
    sequence's middle rows leaves every other byte but theirs."""
    rng = np.random.default_rng(5)
    n, kv, d, cap = 3, 2, 32, 70
    full = torch.from_numpy(rows_of(rng, n * cap, kv, d)).cuda()
    cache = make(ctx, fmt, n, cap, kv, d, fill=0)
    cache.write_dev(full, full, "float32", words([0] * n), n * cap)
    new = torch.from_numpy(rows_of(rng, 40, kv, d)).cuda()
    # sequence 1: rows 2 .. 31 at 50 .. 79 (ten past the capacity), sequence 2: rows 32 .. 33 at 3; 0, 1, 34 .. nobody's
    cache.write_dev(new, new, "float32", words([50, 3]), 40, first_seq=1, n_seqs=2, row_start=words([2, 32, 34]))
    want = stored(full.cpu().numpy().reshape(n, cap, kv, d), fmt)
    w = stored(new.cpu().numpy(), fmt)
    want[1, 50:70] = w[2:22]
    want[2, 3:5] = w[32:34]
    ko, vo = torch.empty((n * cap, kv, d), device="cuda"), torch.empty((n * cap, kv, d), device="cuda")
    cache.read_dev(ko, vo, "float32", words([0] * n), n * cap)
    check(ko.view(n, cap, kv, d), want, "key")
    check(vo.view(n, cap, kv, d), want, "value")
    # and reading such rows says so: NaN
    ko, vo = torch.zeros((40, kv, d), device="cuda"), torch.zeros((40, kv, d), device="cuda")
    cache.read_dev(ko, vo, "float32", words([50, 3]), 40, first_seq=1, n_seqs=2, row_start=words([2, 32, 34]))
    out = np.full((40, kv, d), np.nan, np.float32)
    out[2:22], out[32:34] = w[2:22], w[32:34]
    check(ko, out, "key")
    check(vo, out, "value")


def test_rows_written_one_step_at_a_time(ctx):
    """Decode steps beside each other in one 64-row tile, eight sequences a call: what earlier steps wrote stays."""
    rng = np.random.default_rng(8)
    n, kv, d, steps = 8, 3, 48, 70
    cache = make(ctx, "int8", n, steps, kv, d)
    x = torch.from_numpy(rows_of(rng, steps * n, kv, d)).cuda().view(steps, n, kv, d)
    at = words([0] * n)
    for t in range(steps):
        cache.write_dev(x[t], x[t], "float32", at, n)
        at += 1
    ko, vo = torch.empty((n * steps, kv, d), device="cuda"), torch.empty((n * steps, kv, d), device="cuda")
    cache.read_dev(ko, vo, "float32", words([0] * n), n * steps)
    want = stored(x.permute(1, 0, 2, 3).contiguous().cpu().numpy().reshape(n * steps, kv, d), "int8")
    check(ko, want, "key")
    check(vo, want, "value")


def test_row_starts_that_say_nothing_sensible(ctx):
    """Descending or far row starts and positions of 2^32 - 1 address nothing outside the buffer."""
    kv, d, cap = 1, 16, 40
    buf = torch.zeros(KvCache.size("int8", 2, cap, kv, d) + 4096, dtype=torch.uint8, device="cuda")
    size = KvCache.size("int8", 2, cap, kv, d)
    cache = KvCache(ctx, "int8", 2, cap, kv, d, buf)
    x = torch.ones((30, kv, d), device="cuda")
    for starts, at in (([20, 10, 0], [0, 0]), ([-1, -5, -9], [0, 0]), ([5, 40, 30], [-1, -2]), ([0, 15, 30], [39, 1000])):
        cache.write_dev(x, x, "float32", words(at), 30, row_start=words(starts))
        cache.read_dev(torch.empty_like(x), torch.empty_like(x), "float32", words(at), 30, row_start=words(starts))
    torch.cuda.synchronize()
    assert int(buf[size:].sum()) == 0
