"""GPU: heads normed and turned to their positions, against float64.

Tolerance, eps = 2^-24, of a turned pair (a, b) of normed values: a sum of d
squares in f32 is off by d eps at most, whatever its order, its mean's root's
reciprocal by half that and 4 eps; the products with it and the weight, cos and
sin (rounded once), the two products and their sum add a few more, 8 eps
together, of |a cos| + |b sin|; an angle is off by the position times 2^-64 of a
turn; the result is rounded once (bf16 2^-8)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from quantibbler_amd import GpuContext, KernelError
from quantibbler_amd.gpu import Rope, rotate_heads_dev

EPS = 2.0 ** -24
NORM_EPS = 1e-5
SCALINGS = [None, {"kind": "linear", "factor": 4.0}, {"kind": "base", "factor": 2.5},
            {"kind": "ramp", "factor": 8.0, "original_len": 8192, "low": 1.0, "high": 4.0},
            {"kind": "yarn", "factor": 16.0, "original_len": 4096}]


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


def words(v):
    return torch.tensor([x - (1 << 32) if x >= 1 << 31 else x for x in v], dtype=torch.int32, device="cuda")


def frequencies(theta, rotary, scaling):
    """Radians a position, long double, and the size of cos and sin."""
    L = np.longdouble
    i = np.arange(rotary // 2).astype(L)
    kind, factor = (scaling or {}).get("kind"), L((scaling or {}).get("factor", 1.0))
    base, size = L(theta), 1.0
    if kind == "base" and rotary > 2:
        base = base * factor ** (L(rotary) / L(rotary - 2))
    f, keep = base ** (-2 * i / L(rotary)), np.ones(rotary // 2)
    tau = 2 * L("3.14159265358979323846264338327950288")
    if kind == "linear":
        keep = np.zeros(rotary // 2)
    if kind == "ramp":
        keep = (scaling["original_len"] * f / tau - scaling["low"]) / (scaling["high"] - scaling["low"])
    if kind == "yarn":
        size = 0.1 * math.log(scaling["factor"]) + 1.0
        where = [rotary * math.log(scaling["original_len"] / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (32.0, 1.0)]
        first, last = max(math.floor(where[0]), 0), min(math.ceil(where[1]), rotary - 1)
        keep = 1.0 - (np.arange(rotary // 2) - first) / max(last - first, 0.001)
    keep = np.clip(np.asarray(keep, L), L(0), L(1))
    return f * keep + f / factor * (1 - keep), size


def reference(x, w, at, theta, rotary, inter, scaling):
    """float64 [rows][heads][d] and its tolerance (without the output's rounding)."""
    x = np.asarray(x, np.float64)
    d = x.shape[-1]
    rel = 8 * EPS
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + NORM_EPS) * np.asarray(w, np.float64)
        rel += (d / 2 + 4) * EPS
    f, size = frequencies(theta, rotary, scaling)
    tau = 2 * np.longdouble("3.14159265358979323846264338327950288")
    at = np.asarray(at, np.longdouble)[:, None, None]
    part = at * (f / tau)
    angle = ((part - np.floor(part)) * tau).astype(np.float64)
    c, s = np.cos(angle) * size, np.sin(angle) * size
    off = (at * np.longdouble(2.0) ** -60).astype(np.float64) * size
    one, two = (slice(0, rotary, 2), slice(1, rotary, 2)) if inter else (slice(0, rotary // 2), slice(rotary // 2, rotary))
    out, tol = x.copy(), rel * np.abs(x)
    a, b = x[..., one], x[..., two]
    out[..., one], out[..., two] = a * c - b * s, b * c + a * s
    both = off * (np.abs(a) + np.abs(b))
    tol[..., one] = rel * (np.abs(a * c) + np.abs(b * s)) + both
    tol[..., two] = rel * (np.abs(b * c) + np.abs(a * s)) + both
    return out, tol


def check(got, want, tol, label=""):
    step = EPS if got.dtype == torch.float32 else 2.0 ** -8
    g = got.double().cpu().numpy()
    bad = ~(np.abs(g - want) <= (tol + step * np.abs(want)) * (1 + 2.0 ** -20) + 1e-44)
    assert not bad.any(), f"{label}: {bad.sum()} of {bad.size} off, worst {np.abs(g - want)[bad].max():.3g}, first at " \
        f"{np.argwhere(bad)[:3].tolist()}"


def inputs(seed, n, heads, d, dtype):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((n, heads, d)) * np.exp(rng.standard_normal((n, heads, 1)))).astype(np.float32)
    t = torch.from_numpy(x).to(getattr(torch, dtype))
    return t.cuda(), t.double().numpy()


def places(rows, at, before):
    return [before + a + t for r, a in zip(rows, at) for t in range(r)]


# heads, kv heads, d, rotary, rows of each sequence, first positions
SHAPES = [(1, 1, 2, 2, [1], [0]), (4, 2, 16, 16, [1], [7]), (32, 8, 128, 128, [1], [2085]), (32, 8, 128, 32, [1] * 9, list(range(9))),
          (5, 1, 80, 20, [3, 0, 4], [0, 5, 100]), (7, 7, 96, 96, [2, 6], [9, 1]), (8, 2, 256, 256, [5], [70000]),
          (3, 1, 64, 62, [4], [3]), (6, 2, 24, 8, [10], [1]), (14, 2, 64, 64, [17, 1, 9], [0, 1000000, 77]),
          (2, 1, 254, 250, [3], [12]), (9, 3, 40, 40, [33], [0]), (40, 8, 128, 64, [70], [4000]), (1, 0, 128, 128, [3], [5]),
          (0, 2, 128, 128, [3], [5]), (3, 2, 240, 240, [6], [31]), (2, 2, 12, 4, [9], [2])]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("heads,kv,d,rotary,rows,at", SHAPES)
def test_against_float64(ctx, dtype, inter, normed, heads, kv, d, rotary, rows, at):
    n, before = sum(rows), 3
    scaling = SCALINGS[(d + rotary + heads) % len(SCALINGS)]
    rope = Rope(d, 10000.0, rotary_dim=rotary, interleaved=inter, scaling=scaling)
    rng = np.random.default_rng(d)
    w = [(1 + 0.3 * rng.standard_normal(d)).astype(np.float32) for _ in range(2)] if normed else [None, None]
    wd = [None if x is None else torch.from_numpy(x).cuda() for x in w]
    q, q64 = inputs(1, n, heads, d, dtype)
    k, k64 = inputs(2, n, kv, d, dtype)
    outs = [torch.full_like(x, 77.0) for x in (q, k)]
    starts = words(np.concatenate([[0], np.cumsum(rows)]).tolist())
    rotate_heads_dev(ctx, rope, q if heads else None, k if kv else None, dtype, n, heads, kv, words(at),
                     outs[0] if heads else None, outs[1] if kv else None, n_seqs=len(rows), row_start=starts,
                     before=before, q_norm=wd[0], k_norm=wd[1], eps=NORM_EPS, stream=torch.cuda.current_stream())
    for x64, x, weight, name in ((q64, outs[0], w[0], "q"), (k64, outs[1], w[1], "k")):
        if x.numel():
            check(x, *reference(x64, weight, places(rows, at, before), 10000.0, rotary, inter, scaling), name)


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("theta", [10000.0, 500000.0])
def test_far_positions(ctx, scaling, theta):
    """Positions up to 2^33: the angle is its fraction of a turn, whatever it has turned before."""
    d, heads = 128, 2
    at = [0, 1, 12345, 1 << 20, (1 << 24) + 1, (1 << 31) + 12347, (1 << 32) - 1]
    x, x64 = inputs(5, len(at), heads, d, "float32")
    rope = Rope(d, theta, scaling=scaling)
    for before in (0, 1000003, (1 << 32) - 1):
        out = torch.empty_like(x)
        rotate_heads_dev(ctx, rope, x, None, "float32", len(at), heads, 0, words(at), out, None, n_seqs=len(at),
                         before=before)
        check(out, *reference(x64, None, [a + before for a in at], theta, d, False, scaling), f"before {before}")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,rotary,inter", [(128, 128, False), (64, 16, True), (80, 20, False), (10, 6, True)])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_fused_rows_in_place(ctx, dtype, d, rotary, inter, shift):
    """q and k inside wider rows at any alignment, turned where they stand; nothing else of the rows changes, and rows
    that no sequence claims neither."""
    heads, kv, n = 5, 2, 21
    rng = np.random.default_rng(shift + d)
    width = (heads + 2 * kv) * d + 2 * shift + 5
    wide = torch.from_numpy(rng.standard_normal((n, width)).astype(np.float32)).to(getattr(torch, dtype)).cuda()
    was = wide.clone()
    w = torch.from_numpy((1 + 0.1 * rng.standard_normal(d)).astype(np.float32)).cuda()
    q, k = wide[:, shift:shift + heads * d], wide[:, shift + heads * d + 1:shift + 1 + (heads + kv) * d]
    rope = Rope(d, 10000.0, rotary_dim=rotary, interleaved=inter)
    rotate_heads_dev(ctx, rope, q, k, dtype, n, heads, kv, words([9, 50]), q, k, n_seqs=2, row_start=words([2, 6, 19]),
                     q_norm=w, eps=NORM_EPS, q_stride=width, k_stride=width, q_out_stride=width, k_out_stride=width)
    at = list(range(9, 13)) + list(range(50, 63))
    for x, old, m, weight in ((q, was[:, shift:shift + heads * d], heads, w.cpu().numpy()),
                              (k, was[:, shift + heads * d + 1:shift + 1 + (heads + kv) * d], kv, None)):
        want, tol = reference(old[2:19].double().cpu().numpy().reshape(17, m, d), weight, at, 10000.0, rotary, inter, None)
        check(x[2:19].reshape(17, m, d), want, tol)
    keep = torch.ones_like(wide, dtype=torch.bool)
    keep[2:19, shift:shift + heads * d] = False
    keep[2:19, shift + heads * d + 1:shift + 1 + (heads + kv) * d] = False
    assert torch.equal(wide[keep], was[keep])


@pytest.mark.parametrize("d", [128, 80])
def test_what_is_no_number_stays_in_its_head(ctx, d):
    heads, n = 4, 6
    x, _ = inputs(9, n, heads, d, "float32")
    w = torch.ones(d, device="cuda")
    rope = Rope(d, 10000.0)
    out, again = torch.empty_like(x), torch.empty_like(x)
    rotate_heads_dev(ctx, rope, x, None, "float32", n, heads, 0, words([5]), out, None, q_norm=w)
    x[1, 2, 3], x[4, 0, d - 1] = float("nan"), float("inf")
    rotate_heads_dev(ctx, rope, x, None, "float32", n, heads, 0, words([5]), again, None, q_norm=w)
    fine = torch.ones((n, heads), dtype=torch.bool, device="cuda")
    fine[1, 2] = fine[4, 0] = False
    assert torch.equal(out[fine], again[fine]) and bool(again[1, 2].isnan().all()) and not bool(again[4, 0].isfinite().all())
    # heads of zeros, and of numbers whose squares vanish, stay finite
    x = torch.zeros_like(x)
    x[0] = 1e-30
    rotate_heads_dev(ctx, rope, x, None, "float32", n, heads, 0, words([5]), again, None, q_norm=w)
    assert bool(again.isfinite().all()) and bool((again[1:] == 0).all())


def test_the_blocks_rotation_is_the_same_angle(ctx):
    """The half layout over the whole head, unscaled, is what a block turns by: cos and sin of the reference's f64
    angles, rounded to f32 (a last place apart where the f64 product of position and frequency is off)."""
    d, n = 64, 4096
    x = torch.zeros((n, 1, d), device="cuda")
    x[..., :d // 2] = 1.0
    out = torch.empty_like(x)
    rotate_heads_dev(ctx, Rope(d, 10000.0), x, None, "float32", n, 1, 0, words([0]), out, None)
    inv = np.array([10000.0 ** (-(2.0 * i) / d) for i in range(d // 2)])
    angle = np.arange(n)[:, None] * inv
    got = out.cpu().numpy()[:, 0]
    assert np.abs(got[:, :d // 2] - np.cos(angle).astype(np.float32)).max() <= 2.0 ** -24
    assert np.abs(got[:, d // 2:] - np.sin(angle).astype(np.float32)).max() <= 2.0 ** -24


def test_replays_follow_the_device_positions(ctx):
    d, heads, kv, n = 128, 8, 2, 5
    rope, at = Rope(d, 10000.0), words([3] * n)
    q, k = torch.empty((n, heads, d), device="cuda"), torch.empty((n, kv, d), device="cuda")
    qo, ko = torch.empty_like(q), torch.empty_like(k)

    def step(a, b):
        rotate_heads_dev(ctx, rope, q, k, "float32", n, heads, kv, at, a, b, n_seqs=n, stream=torch.cuda.current_stream())

    q.normal_(), k.normal_()
    step(qo, ko)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(qo, ko)
    for rep in range(4):
        q.normal_(), k.normal_()
        at += 1000
        graph.replay()
        a, b = torch.empty_like(q), torch.empty_like(k)
        step(a, b)
        torch.cuda.synchronize()
        assert torch.equal(a, qo) and torch.equal(b, ko)
    del graph


def test_rows_that_fill_the_card(ctx):
    """Many rows and few, the same rows: each its own result, bit for bit, on any stream."""
    d, heads, kv, n = 128, 32, 8, 3001
    q, q64 = inputs(11, n, heads, d, "bfloat16")
    k, k64 = inputs(12, n, kv, d, "bfloat16")
    w = torch.rand(d, device="cuda") + 0.5
    rope = Rope(d, 500000.0, scaling=SCALINGS[3])
    out, some = [torch.empty_like(x) for x in (q, k)], [torch.empty_like(x[:5]) for x in (q, k)]
    rotate_heads_dev(ctx, rope, q, k, "bfloat16", n, heads, kv, words([17]), *out, q_norm=w, k_norm=w,
                     eps=NORM_EPS)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    rotate_heads_dev(ctx, rope, q[-5:], k[-5:], "bfloat16", 5, heads, kv, words([17 + n - 5]), *some, q_norm=w, k_norm=w,
                     eps=NORM_EPS, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(out[0][-5:], some[0]) and torch.equal(out[1][-5:], some[1])
    pick = np.array([0, 1, 2, 63, 64, 1500, n - 1])
    for x, x64 in zip(out, (q64, k64)):
        want, tol = reference(x64[pick], w.cpu().numpy(), 17 + pick, 500000.0, d, False, SCALINGS[3])
        check(x[torch.from_numpy(pick).cuda()], want, tol)


def test_in_place_takes_one_stride(ctx):
    from quantibbler_amd import KernelError

    d, heads, kv, n = 64, 4, 2, 3
    wide = torch.randn((n, 500), device="cuda")
    kept = wide.clone()
    q, k = wide[:, :heads * d], wide[:, heads * d:(heads + kv) * d]
    out = torch.empty((n, 500), device="cuda")
    for strides in (dict(k_out_stride=500), dict(q_out_stride=500)):
        with pytest.raises(KernelError, match="in place needs one stride"):
            rotate_heads_dev(ctx, Rope(d, 10000.0), q.data_ptr(), k.data_ptr(), "float32", n, heads, kv, words([1]),
                             q.data_ptr(), k.data_ptr(), q_stride=500, k_stride=500, **strides)
    rotate_heads_dev(ctx, Rope(d, 10000.0), q, None, "float32", n, heads, 0, words([1]), out, None, q_stride=500,
                     q_out_stride=500)
    torch.cuda.synchronize()
    assert torch.equal(wide, kept)
