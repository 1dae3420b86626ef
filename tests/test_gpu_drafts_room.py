"""GPU: drafted tokens where a request's rows end: a step that passes the capacity,
verification within a limit, replays that reach it, captures after rejected
drafts, numbers of drafts of a request's own."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import test_gpu_attention_kv as att
import test_gpu_block_kv as bkv
import test_gpu_verify as ver
from quantibbler_amd import DecoderBlock, GpuContext

words, EPS = att.words, 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


@pytest.mark.parametrize("fmt", ["int8", "fp8", "fp4"])
@pytest.mark.parametrize("per,plen,lens", [(5, 0, [10, 68, 66, 69]), (4, 129, [69, 66, 67, 0]), (20, 70, [51, 69, 60])])
def test_tokens_that_fit_before_those_that_do_not(ctx, orc, fmt, per, plen, lens):
    """A step that passes a sequence's last row: its tokens before that see the rows up to their own, as any."""
    rng = np.random.default_rng(200 + per)
    L = bkv.Layers(ctx, orc, 5)
    D, HEADS, KV, HD, n, cap = bkv.D, bkv.HEADS, bkv.KV, bkv.HD, len(lens), 70
    block = DecoderBlock(ctx, L.all, np.ones(D), np.ones(D), HEADS, KV, HD, bkv.THETA, 1e-5, capacity=400)
    cache = bkv.make(ctx, fmt, n, cap)
    bkv.fill(cache, rng, lens)
    shared, p = None, (np.zeros((0, KV, HD)),) * 2
    if plen:
        shared = bkv.make(ctx, fmt, 1, plen)
        bkv.fill(shared, rng, [plen])
        p = bkv.held(shared, [plen])[0]
    h = rng.standard_normal((n, per, D)).astype(np.float32)
    hd = torch.from_numpy(h).cuda()
    need = block.decode_kv_workspace_size(cache, n, prefix_len=plen, n_tokens=per)
    block.decode_kv_dev(hd, words(lens), n, cache, torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda"), need,
                        prefix=shared, prefix_len=plen, n_tokens=per)
    torch.cuda.synchronize()
    now = bkv.held(cache, [min(x + per, cap) for x in lens])
    got = hd.cpu().numpy().astype(np.float64)
    for i in range(n):
        k, v = now[i]
        for t in range(min(per, cap - lens[i])):
            seen = lens[i] + t + 1
            a, tol = bkv.attention(bkv.rotated(L.q, HEADS, plen + lens[i] + t), np.concatenate([p[0], k[:seen]]),
                                   np.concatenate([p[1], v[:seen]]))
            want, bound = bkv.o_layer(L, a, tol)
            want = want + h[i, t]
            off = np.abs(got[i, t] - want) - bound - 2 * EPS * np.abs(want)
            assert (off <= 0).all(), f"sequence {i}, token {t}: past its bound by {off.max()}"
    block.close()


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("n_drafts", [False, True])
def test_verification_within_a_limit(ctx, given, n_drafts):
    """A request's drafts end where its rows do, whichever end comes first; without a row it emits nothing and stays."""
    n, k, vocab, limit = 12, 6, 5003, 100
    at = [0, 93, 94, 95, 97, 98, 99, 100, 101, 2 ** 31 - 1, -1, 50]  # -1: 2^32 - 1
    have = [6, 5, 6, 9, 1, 6, 0, 6, 2, 6, 6, 3] if n_drafts else [k] * n
    x, y, ids, u = ver.make(3, n, k, vocab, "float32", given)
    u[::2] *= 0.05
    heat = np.where(np.arange(n) % 3 == 1, 0.0, 0.8).astype(np.float32)
    pos = words(at)
    tokens, counts = ver.verify(ctx, x, y, ids, u, words(have) if n_drafts else None, ver.tensor(heat), pos=pos,
                                pos_limit=limit)
    live = [i for i in range(n) if 0 <= at[i] < limit]
    some = [min(have[i], limit - 1 - at[i]) for i in live]
    ver.check(tokens[live], counts[live], x[live], None if y is None else y[live], ids[live], u[live], some, heat[live])
    for i in set(range(n)) - set(live):
        assert tokens[i].tolist() == [-1] * (k + 1) and int(counts[i]) == 0
    assert pos.tolist() == [a + c for a, c in zip(at, counts.tolist())]
    # from 2^32 on, no limit
    pos = words(at)
    free = ver.verify(ctx, x, y, ids, u, words(have) if n_drafts else None, ver.tensor(heat), pos=pos, pos_limit=1 << 32)
    ver.check(*free, x, y, ids, u, have, heat)


def model(ctx, orc, capacity):
    from test_gpu_trunk import synthetic_model

    from quantibbler_amd.model import DeviceModel

    return DeviceModel(ctx, synthetic_model(orc, 808), capacity=capacity)


@pytest.mark.parametrize("fmt", ["int8", "fp4"])
def test_replays_up_to_the_capacity(ctx, orc, fmt):
    """A captured verification replayed until its requests are full: drafts are taken as far as there is room, the drawn
    token follows the last row, and a request without room emits nothing and stays where it is; an eager call is then
    refused with the rows that are held."""
    m = model(ctx, orc, 60)
    vocab, n, k, cap = m.md.vocab_size, 4, 3, 17
    rng = np.random.default_rng(3)
    m.share_prefix(rng.integers(0, vocab, 33).tolist(), n, cap, fmt=fmt)
    tokens, u = torch.zeros((n, k + 1), dtype=torch.int32, device="cuda"), torch.zeros((n, k + 1), device="cuda")
    heat = torch.tensor([0.8, 0.0, 1.5, 1.0], device="cuda")
    counts_in = words([k, 1, 2, k])
    m.verify_shared(tokens, u, n_drafts=counts_in, temperature=heat)
    torch.cuda.synchronize()
    m._shared["pos"].copy_(words([0, 3, 1, 2]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, counts = m.verify_shared(tokens, u, n_drafts=counts_in, temperature=heat, stream=torch.cuda.current_stream())
    logits = m._shared["drafts"][k + 1]["logits"].view(n, k + 1, vocab)
    full = 0
    for rep in range(24):
        before = m._shared["pos"].tolist()
        tokens.copy_(words(rng.integers(0, vocab, n * (k + 1))).view(n, k + 1))
        u.copy_(torch.from_numpy((0.02 * rng.random((n, k + 1))).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        room = [cap - b for b in before]
        most = [max(0, min(c, r - 1)) for c, r in zip([k, 1, 2, k], room)]
        live = [i for i in range(n) if room[i] > 0]
        ver.check(out[live], counts[live], logits[live], None, tokens[live, 1:], u[live], [most[i] for i in live],
                  heat[live], f"replay {rep}")
        for i in range(n):
            if room[i] <= 0:
                full += 1
                assert out[i].tolist() == [-1] * (k + 1) and int(counts[i]) == 0
        after = m._shared["pos"].tolist()
        assert after == [b + c for b, c in zip(before, counts.tolist())] and max(after) <= cap
    assert full and max(after) == cap
    for call in (lambda: m.verify_shared(tokens, u), lambda: m.step_shared([1] * n)):
        with pytest.raises(ValueError, match="no room for 4 rows behind 17 of|hold their 17 rows already"):
            call()
    del graph
    m.close()


def test_captures_after_drafts_that_were_not_kept(ctx, orc):
    """What eager calls did not keep is no reason to refuse a capture, which fetches nothing; one whose requests are
    known to be full is refused."""
    m = model(ctx, orc, 40)
    n, k, cap = 2, 3, 12
    m.share_prefix([1, 2, 3, 4, 5], n, cap, fmt="fp4")
    u, cold = torch.full((n, k + 1), 0.5, device="cuda"), torch.zeros(n, device="cuda")
    wrong = words([3, -1, -1, -1, 4, -1, -1, -1]).view(n, k + 1)
    for _ in range(3):
        _, counts = m.verify_shared(wrong, u, temperature=cold)  # an id of -1 is never kept: one row a call
    assert m._shared["pos"].tolist() == [3, 3]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, counts = m.verify_shared(wrong, u, temperature=cold, stream=torch.cuda.current_stream())
    for at in range(4, 15):
        graph.replay()
        torch.cuda.synchronize()
        assert m._shared["pos"].tolist() == [min(at, cap)] * n and counts.tolist() == [int(at <= cap)] * n
    with pytest.raises(ValueError, match="hold their 12 rows already"):
        m.step_shared([1, 2])
    m.share_prefix([1, 2, 3, 4, 5], n, 6, fmt="fp4")  # steps count what they hold exactly
    for _ in range(5):
        m.step_shared([1, 2])
    with pytest.raises(ValueError, match="no room for 4 rows behind 5 of a capacity of 6"):
        m.verify_shared(wrong, u, temperature=cold)
    del graph
    m.close()


@pytest.mark.parametrize("fmt", ["int8", "fp8", "fp4"])
def test_numbers_of_drafts_of_a_requests_own(ctx, orc, fmt):
    """Rows padded with -1, as the call's own output is: the same tokens, counts, logits and, in the steps after, rows as
    with other ids there, which no request looks at; sampled and greedy, against the definition on the logits."""
    rng = np.random.default_rng(9)
    n, k, cap = 4, 3, 40
    models = [model(ctx, orc, 80) for _ in range(2)]
    vocab = models[0].md.vocab_size
    prompt = rng.integers(0, vocab, 33).tolist()
    for m in models:
        m.share_prefix(prompt, n, cap, fmt=fmt)
    heat = torch.tensor([0.9, 0.0, 1.3, 0.7], device="cuda")
    for rep in range(5):
        have = [[3, 0, 1, 2], [0, 0, 0, 0], [2, 3, 0, 1], [1, 1, 3, 3], [3, 2, 2, 0]][rep]
        ids = rng.integers(0, vocab, (n, k + 1))
        padded = ids.copy()
        for i in range(n):
            padded[i, 1 + have[i]:] = -1
        u = torch.from_numpy(rng.random((n, k + 1)).astype(np.float32) * (0.05 if rep % 2 else 1.0)).cuda()
        y = torch.randn((n, k, vocab), device="cuda") if rep in (2, 4) else None
        got = []
        for m, rows in zip(models, (ids, padded)):
            tokens = words(rows.reshape(-1).tolist()).view(n, k + 1)
            out = m.verify_shared(tokens, u, draft_logits=y, n_drafts=words(have), temperature=heat)
            torch.cuda.synchronize()
            logits = m._shared["drafts"][k + 1]["logits"].view(n, k + 1, vocab).clone()
            got.append((out[0].clone(), out[1].clone(), logits, m._shared["pos"].clone()))
        for a, b in zip(got[0], got[1]):
            if a is got[0][2]:
                assert all(torch.equal(a[i, :have[i] + 1], b[i, :have[i] + 1]) for i in range(n)), f"call {rep}"
                assert all(bool(torch.isfinite(b[i, :have[i] + 1]).all()) for i in range(n))
            else:
                assert torch.equal(a, b), f"call {rep}"
        out, counts, logits, _ = got[1]
        ver.check(out, counts, logits, y, torch.from_numpy(ids[:, 1:].copy()), u, have, heat, f"call {rep}")
        step = rng.integers(0, vocab, n).tolist()
        assert torch.equal(models[0].step_shared(step), models[1].step_shared(step))
    for m in models:
        m.close()


def test_what_is_refused_runs_nothing(ctx, orc):
    """Tensors that do not fit are refused before a block has written a row."""
    m = model(ctx, orc, 40)
    n, k, vocab = 2, 2, m.md.vocab_size
    m.share_prefix([1, 2, 3], n, 20, fmt="fp4")
    rows, u = [[1, 2, 3], [4, 5, 6]], torch.zeros((n, k + 1), device="cuda")
    m.verify_shared(rows, u)
    torch.cuda.synchronize()
    before, steps = [c.buffer.clone() for c in m._shared["own"]], m._shared["steps"]
    for kw in (dict(uniforms=u[:1]), dict(uniforms=u.double()), dict(uniforms=u.cpu()),
               dict(draft_logits=torch.zeros((n, k, vocab - 1), device="cuda")),
               dict(draft_logits=torch.zeros((n, k, vocab), dtype=torch.bfloat16, device="cuda")),
               dict(n_drafts=torch.zeros(n, dtype=torch.int64, device="cuda")), dict(n_drafts=words([1])),
               dict(temperature=torch.zeros(1, device="cuda")), dict(temperature=[1.0, 1.0]),
               dict(tokens=torch.zeros((n, k + 1), dtype=torch.int64, device="cuda")),
               dict(tokens=words(range(12)).view(n, 6)[:, ::2]), dict(uniforms=None),
               dict(tokens=[[1], [2]], draft_logits=torch.zeros((n, 1, vocab), device="cuda"))):
        with pytest.raises(ValueError):
            m.verify_shared(**{"tokens": rows, "uniforms": u, **kw})
        torch.cuda.synchronize()
        assert all(torch.equal(a, c.buffer) for a, c in zip(before, m._shared["own"])), f"{sorted(kw)}"
        assert m._shared["steps"] == steps
    m.close()


@pytest.mark.parametrize("n", [1, 3])
def test_the_returned_tokens_as_the_next_input(ctx, orc, n):
    """The tensor that a call returned, filled with the next step's rows and handed back: as a tensor of its own."""
    models = [model(ctx, orc, 80) for _ in range(2)]
    k, vocab = 4, models[0].md.vocab_size
    rng = np.random.default_rng(17)
    for m in models:
        m.share_prefix([5, 6, 7], n, 60, fmt="fp4")
    held = [None, None]
    for rep in range(6):
        rows = words(rng.integers(0, vocab, n * (k + 1)).tolist()).view(n, k + 1)
        u = torch.from_numpy((0.02 * rng.random((n, k + 1))).astype(np.float32)).cuda()
        got = []
        for i, m in enumerate(models):
            tokens = rows.clone()
            if i and held[1] is not None:
                tokens = held[1].copy_(rows)
            out, counts = m.verify_shared(tokens, u)
            torch.cuda.synchronize()
            held[i] = out
            got.append((out.clone(), counts.clone()))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]), f"call {rep}"
    for m in models:
        m.close()
