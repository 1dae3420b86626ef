"""GPU: a decoder block's step over an 8-bit cache behind a shared prefix.

The block's q, k and v layers have s1 = 0, so that every token's query, key
and value are the layers' biases, its down layer s1 = 0 and no bias, so that
the block's output is o(attention) + h: the step's rotation, its row in the
cache and its attention are then known in float64, and the output's distance
from it is bounded by the roundings of o's two stages (bf16 z, t and u, 2^-8
each; f32 sums; operands that keep 2^-17 of their block's largest)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from quantibbler_amd import DecoderBlock, FactorLayer, GpuContext, KernelError, KvCache

THETA, D, HEADS, KV, HD, FFN, R = 10000.0, 256, 4, 2, 64, 320, 48
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


def words(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


class Layers:
    """The seven layers; o's signs and scales kept."""

    def __init__(self, ctx, orc, seed):
        rng = np.random.default_rng(seed)
        self.all = []
        for name, dout, din in (("q", HEADS * HD, D), ("k", KV * HD, D), ("v", KV * HD, D), ("o", D, HEADS * HD),
                                ("gate", FFN, D), ("up", FFN, D), ("down", D, FFN)):
            ub = rng.choice([-1, 1], (dout, R)).astype(np.int8)
            vt = rng.choice([-1, 1], (R, din)).astype(np.int8)
            s1 = (np.exp(0.2 * rng.standard_normal(dout)) / math.sqrt(R * din)).astype(np.float16).astype(np.float32)
            s2 = np.exp(0.2 * rng.standard_normal(din)).astype(np.float16).astype(np.float32)
            bias = None
            if name in ("q", "k", "v"):
                s1[:] = 0.0
                bias = (1.5 * rng.standard_normal(dout)).astype(np.float16).astype(np.float32)
                setattr(self, name, bias.astype(np.float64))
            if name == "down":
                s1[:] = 0.0
            if name == "o":
                self.ub, self.vt, self.s1, self.s2 = (x.astype(np.float64) for x in (ub, vt, s1, s2))
            self.all.append(FactorLayer.from_rows(ctx, dout, din, R, orc.pack_bits(ub), orc.pack_bits(vt), s1, s2, bias))


def rotated(x, heads, p):
    """RoPE at position p in float64."""
    x = x.reshape(heads, HD)
    a = p * THETA ** (-2.0 * np.arange(HD // 2) / HD)
    c, s = np.cos(a), np.sin(a)
    lo, hi = x[:, :HD // 2], x[:, HD // 2:]
    return np.concatenate([lo * c - hi * s, hi * c + lo * s], 1)


def o_layer(L, at, tol):
    """float64 o(at) and its bound for an attention output known to tol."""
    z = L.s2 * at
    ez = L.s2 * tol + 2.0 ** -8 * (np.abs(z) + L.s2 * tol) + 2.0 ** -17 * np.abs(z).max()
    t = L.vt @ z
    et = ez.sum() + (len(z) + 2) * EPS * np.abs(z).sum()
    et = et + 2.0 ** -8 * (np.abs(t) + et) + 2.0 ** -17 * np.abs(t).max()
    u = L.ub @ t
    eu = et.sum() + (R + 2) * EPS * np.abs(t).sum()
    eu = eu + 2.0 ** -8 * (np.abs(u) + eu)
    return L.s1 * u, np.abs(L.s1) * eu * (1 + 4 * EPS) + 4 * EPS * np.abs(L.s1 * u)


def attention(q, k, v):
    """float64: q [heads][d], k and v [rows][kv][d]; the output and its bound for f32 queries (as in
    test_gpu_attention_kv; queries and keys are f32 roundings of rotated ones, 2^-22 of their size)."""
    out, tol = np.zeros((HEADS, HD)), np.zeros((HEADS, HD))
    for h in range(HEADS):
        kk, vv = k[:, h // (HEADS // KV)], v[:, h // (HEADS // KV)]
        s = kk @ q[h] / math.sqrt(HD)
        w = np.exp(s - s.max())
        w /= w.sum()
        out[h] = w @ vv
        b = (((HD + 8) * EPS + 2.0 ** -23 + 2.0 ** -21) * (np.abs(kk) @ np.abs(q[h])).max() +
             2.0 ** -28 * np.abs(q[h]).max() * np.abs(kk).sum(1).max()) / math.sqrt(HD)
        tol[h] = (2 * b + 2.0 ** -22 + (2 * len(s) + 70) * EPS) * (w @ np.abs(vv)) + len(s) * 2.0 ** -36 * np.abs(vv).max()
    return out.reshape(-1), tol.reshape(-1)


def make(ctx, fmt, n, cap):
    buf = torch.empty(KvCache.size(fmt, n, cap, KV, HD), dtype=torch.uint8, device="cuda")
    buf.fill_(0xFF)
    return KvCache(ctx, fmt, n, cap, KV, HD, buf)


def fill(cache, rng, rows, first=0):
    total = sum(rows)
    k, v = (torch.from_numpy(rng.standard_normal((total, KV, HD)).astype(np.float32)).cuda() for _ in range(2))
    starts = words(np.concatenate([[0], np.cumsum(rows)]))
    cache.write_dev(k, v, "float32", words([0] * len(rows)), total, first_seq=first, n_seqs=len(rows), row_start=starts)


def held(cache, rows, first=0):
    """What rows[i] rows of sequence first + i stand for, float64."""
    total = sum(rows)
    k, v = (torch.empty((total, KV, HD), device="cuda") for _ in range(2))
    starts = words(np.concatenate([[0], np.cumsum(rows)]))
    cache.read_dev(k, v, "float32", words([0] * len(rows)), total, first_seq=first, n_seqs=len(rows), row_start=starts)
    k, v, out, s = k.cpu().numpy().astype(np.float64), v.cpu().numpy().astype(np.float64), [], 0
    for r in rows:
        out.append((k[s:s + r], v[s:s + r]))
        s += r
    return out


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("n,plen", [(1, 0), (1, 70), (3, 129), (8, 1), (20, 0), (40, 200)])
def test_step_against_float64(ctx, orc, fmt, n, plen):
    rng = np.random.default_rng(100 + n + plen)
    L = Layers(ctx, orc, 5)
    block = DecoderBlock(ctx, L.all, np.ones(D), np.ones(D), HEADS, KV, HD, THETA, 1e-5, capacity=400)
    cap, first = 90, 2
    lens = [int(x) for x in rng.integers(0, cap - 1, n)]
    lens[0] = 0
    if n > 1:
        lens[-1] = cap - 1
    cache = make(ctx, fmt, n + first, cap)
    fill(cache, rng, lens, first)
    shared, p = None, (np.zeros((0, KV, HD)),) * 2
    if plen:
        shared = make(ctx, fmt, 2, plen + 5)
        fill(shared, rng, [plen], 1)
        p = held(shared, [plen], 1)[0]
    h = rng.standard_normal((n, D)).astype(np.float32)
    hd_ = torch.from_numpy(h).cuda()
    need = block.decode_kv_workspace_size(cache, n, prefix_len=plen)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    pos = words(lens)
    block.decode_kv_dev(hd_, pos, n, cache, ws, need, first_seq=first, prefix=shared, prefix_seq=1 if plen else 0,
                        prefix_len=plen)
    torch.cuda.synchronize()
    assert pos.tolist() == lens
    now = held(cache, [x + 1 for x in lens], first)
    got = hd_.cpu().numpy().astype(np.float64)
    top = 127.0 if fmt == "int8" else 448.0
    for i in range(n):
        at = plen + lens[i]
        k, v = now[i]
        for row, want in ((k[-1], rotated(L.k, KV, at)), (v[-1], L.v.reshape(KV, HD))):
            big = np.abs(want).max(1, keepdims=True)
            # half a step: of an integer code 0.5 / 127 of the largest; of e4m3 2^-4 of the value, 2^-10 / 448 below
            half = 0.5 / top * big if fmt == "int8" else np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 / top * big)
            assert (np.abs(row - want) <= half * (1 + 2.0 ** -10) + 2.0 ** -20 * big).all(), f"row of sequence {i}"
        a, tol = attention(rotated(L.q, HEADS, at), np.concatenate([p[0], k]), np.concatenate([p[1], v]))
        want, bound = o_layer(L, a, tol)
        want = want + h[i]
        off = np.abs(got[i] - want) - bound - 2 * EPS * np.abs(want)
        assert (off <= 0).all(), f"sequence {i}: past its bound by {off.max()}"
        # the bound says something: the prefix, the own rows and the new row each move the output by more
        assert bound.max() < np.abs(want - h[i]).max()
    block.close()


def test_captured_step_follows_its_positions(ctx, orc):
    """One captured step replayed at the positions after it: each replay the eager step's result, bit for bit."""
    from quantibbler_amd.gpu import advance_positions_dev

    rng = np.random.default_rng(9)
    n, plen, cap = 5, 100, 60
    L = Layers(ctx, orc, 6)
    block = DecoderBlock(ctx, L.all, np.ones(D), np.ones(D), HEADS, KV, HD, THETA, 1e-5, capacity=400)
    shared = make(ctx, "int8", 1, plen)
    fill(shared, rng, [plen])
    lens = [0, 7, 20, 50, 33]
    caches = [make(ctx, "int8", n, cap) for _ in range(2)]
    rows = rng.integers(0, 1 << 30)
    for c in caches:
        fill(c, np.random.default_rng(rows), lens)
    need = block.decode_kv_workspace_size(caches[0], n, prefix_len=plen)
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    pos = [words(lens) for _ in range(2)]
    h = [torch.zeros((n, D), device="cuda") for _ in range(2)]

    def step(i):
        s = torch.cuda.current_stream()
        block.decode_kv_dev(h[i], pos[i], n, caches[i], ws[i], need, prefix=shared, prefix_len=plen, stream=s)
        advance_positions_dev(ctx, pos[i], n, s)

    x = torch.from_numpy(rng.standard_normal((n, D)).astype(np.float32)).cuda()
    for i in range(2):
        h[i].copy_(x)
        step(i)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(0)
    for rep in range(4):
        x = torch.from_numpy(rng.standard_normal((n, D)).astype(np.float32)).cuda()
        h[0].copy_(x)
        h[1].copy_(x)
        graph.replay()
        step(1)
        torch.cuda.synchronize()
        assert torch.equal(h[0], h[1]) and pos[0].tolist() == [v + 2 + rep for v in lens]
    del graph
    block.close()


def test_step_refusals(ctx, orc):
    L = Layers(ctx, orc, 7)
    block = DecoderBlock(ctx, L.all, np.ones(D), np.ones(D), HEADS, KV, HD, THETA, 1e-5, capacity=100)
    cache, shared = make(ctx, "int8", 4, 60), make(ctx, "int8", 1, 50)
    h, pos = torch.zeros((4, D), device="cuda"), words([0] * 4)
    need = block.decode_kv_workspace_size(cache, 4, prefix_len=40)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def refused(words_, **kw):
        a = dict(h=h, pos=pos, n=4, cache=cache, workspace=ws, workspace_size=need, prefix=shared, prefix_len=40)
        a.update(kw)
        with pytest.raises(KernelError, match=words_):
            block.decode_kv_dev(**a)

    refused("prefix of 41 rows and 60 own positions exceed the block's capacity of 100", prefix_len=41)
    refused("does not fit its cache", prefix_len=51, max_len=20)
    refused("does not fit its cache", prefix_seq=1)
    refused("does not fit its cache", prefix=make(ctx, "fp8", 1, 50))
    refused("max_len 61 is not within", max_len=61)
    refused("max_len 0 is not within", max_len=0)
    refused("sequences 1 .. 5 of a kv cache holding 4", first_seq=1)
    refused("workspace of .* is smaller than the", workspace_size=need - 1)
    refused("needs the cache that holds the prefix", prefix=None)
    refused("positions must be", pos=pos[:3])
    refused("batched decode input must be", h=h[:3])
    other = KvCache(ctx, "int8", 4, 60, KV, 32, torch.empty(KvCache.size("int8", 4, 60, KV, 32), dtype=torch.uint8,
                                                           device="cuda"))
    refused("a kv cache of 2 heads of 32 for a block of 2 heads of 64", cache=other)
    block.set_serving("fp32")
    refused("fp32 serving")
    block.close()


def test_model_behind_a_shared_prefix(ctx, orc):
    """share_prefix and step_shared are the blocks' steps between the embedding and the head: bit for bit the calls made
    one by one, on either kind of token ids, up to the requests' capacity."""
    from test_gpu_trunk import synthetic_model

    from quantibbler_amd.gpu import embed, rms_norm_dev
    from quantibbler_amd.model import DeviceModel

    md = synthetic_model(orc, 808)
    rng = np.random.default_rng(12)
    prompt, n, cap = rng.integers(0, md.vocab_size, 65).tolist(), 3, 4
    m = DeviceModel(ctx, md, capacity=70)
    want = m.prefill(prompt).clone()
    assert torch.equal(m.share_prefix(prompt, n, cap), want)
    kd = md.n_kv_heads * md.head_dim
    own, shared = [], []
    for b in m.blocks:
        k, v = b.cache_ptrs()
        for seqs, rows, keep in ((1, 65, shared), (n, cap, own)):
            size = KvCache.size("int8", seqs, rows, md.n_kv_heads, md.head_dim)
            keep.append(KvCache(ctx, "int8", seqs, rows, md.n_kv_heads, md.head_dim,
                                torch.empty(size, dtype=torch.uint8, device="cuda")))
        shared[-1].write_dev(k, v, "float32", words([0]), 65, row_stride=kd)
    h = torch.empty((n, md.d_model), device="cuda")
    need = m.blocks[0].decode_kv_workspace_size(own[0], n, prefix_len=65)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    logits = torch.empty((n, md.vocab_size), device="cuda")
    for step in range(cap):
        ids = rng.integers(0, md.vocab_size, n).tolist()
        got = m.step_shared(words(ids) if step % 2 else ids).clone()
        embed(ctx, m.embedding, md.vocab_size, md.d_model, ids, h)
        for b, o, s in zip(m.blocks, own, shared):
            b.decode_kv_dev(h, words([step] * n), n, o, ws, need, prefix=s, prefix_len=65)
        hn = torch.empty_like(h)
        rms_norm_dev(ctx, h, n, md.d_model, m.final_norm, md.rms_norm_eps, hn)
        m.head.logits_dev(hn, n, logits)
        torch.cuda.synchronize()
        assert torch.equal(got, logits) and bool(logits.isfinite().all())
    with pytest.raises(ValueError, match="hold their 4 rows already"):
        m.step_shared([1, 2, 3])
    with pytest.raises(ValueError, match="2 tokens for 3 requests"):
        m.step_shared([1, 2])
    with pytest.raises(ValueError, match="3 requests of 6 rows behind 65 on a model of 70"):
        m.share_prefix(prompt, 3, 6)
    m.reset()
    with pytest.raises(ValueError, match="needs share_prefix"):
        m.step_shared([1, 2, 3])
    m.close()


def test_a_refused_prefix_leaves_the_model_as_it_was(ctx, orc):
    from test_gpu_trunk import synthetic_model

    from quantibbler_amd.model import DeviceModel

    m = DeviceModel(ctx, synthetic_model(orc, 808), capacity=70)
    m.prefill([5, 6, 7])
    want = m.step(9).clone()
    m.reset()
    m.prefill([5, 6, 7])
    for args, kw in ((([1, 2], 3, 6), {"fmt": "int4"}), (([1, 2], 3, 0), {}), (([1, 2], 0, 6), {}), (([], 3, 6), {})):
        with pytest.raises((ValueError, KernelError)):
            m.share_prefix(*args, **kw)
        assert m.pos == 3 and m._shared is None
    assert torch.equal(m.step(9), want)
    m.close()
