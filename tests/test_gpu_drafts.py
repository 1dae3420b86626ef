"""GPU: drafted tokens through the serving path -- a block's step of several
tokens a sequence, a model's drafts behind a shared prompt, and the operators one
after the other as a program uses them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import test_gpu_attention_kv as att
import test_gpu_block_kv as bkv
import test_gpu_rotate as rot
import test_gpu_verify as ver
from quantibbler_amd import DecoderBlock, GpuContext, KernelError, LmHead
from quantibbler_amd.gpu import Rope, rotate_heads_dev, verify_drafts_dev, verify_drafts_workspace_size

words, EPS = att.words, 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    return GpuContext(0)


# ---- a block's step of several tokens -------------------------------------------

@pytest.mark.parametrize("fmt", ["int8", "fp8", "fp4"])
@pytest.mark.parametrize("n,per,plen", [(1, 1, 0), (1, 7, 70), (3, 2, 0), (3, 5, 129), (8, 8, 1), (2, 32, 200), (64, 1, 5)])
def test_tokens_against_float64(ctx, orc, fmt, n, per, plen):
    """As test_gpu_block_kv's step, with `per` tokens a sequence: each at its own position and over the rows up to its
    own."""
    rng = np.random.default_rng(100 + n + per + plen)
    L = bkv.Layers(ctx, orc, 5)
    D, HEADS, KV, HD = bkv.D, bkv.HEADS, bkv.KV, bkv.HD
    block = DecoderBlock(ctx, L.all, np.ones(D), np.ones(D), HEADS, KV, HD, bkv.THETA, 1e-5, capacity=400)
    cap, first = 90, 2
    lens = [int(x) for x in rng.integers(0, cap - per, n)]
    lens[0] = 0
    lens[-1] = cap - per
    cache = bkv.make(ctx, fmt, n + first, cap)
    bkv.fill(cache, rng, lens, first)
    shared, p = None, (np.zeros((0, KV, HD)),) * 2
    if plen:
        shared = bkv.make(ctx, fmt, 2, plen + 5)
        bkv.fill(shared, rng, [plen], 1)
        p = bkv.held(shared, [plen], 1)[0]
    h = rng.standard_normal((n, per, D)).astype(np.float32)
    hd = torch.from_numpy(h).cuda()
    need = block.decode_kv_workspace_size(cache, n, prefix_len=plen, n_tokens=per)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    pos = words(lens)
    block.decode_kv_dev(hd, pos, n, cache, ws, need, first_seq=first, prefix=shared, prefix_seq=1 if plen else 0,
                        prefix_len=plen, n_tokens=per)
    torch.cuda.synchronize()
    assert pos.tolist() == lens
    now = bkv.held(cache, [x + per for x in lens], first)
    got = hd.cpu().numpy().astype(np.float64)
    for i in range(0, n, max(1, n // 8)):
        k, v = now[i]
        for t in range(per):
            at, seen = plen + lens[i] + t, lens[i] + t + 1
            for row, want in ((k[seen - 1], bkv.rotated(L.k, KV, at)), (v[seen - 1], L.v.reshape(KV, HD))):
                big = np.abs(want).max(1, keepdims=True)
                if fmt == "fp4":  # half a step of the code, or what its multiplier is short of its group's largest
                    assert (np.abs(row - want) <= (1 / 6 + 2.0 ** -4) * big).all()
                else:
                    half = 0.5 / 127.0 * big if fmt == "int8" else np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 / 448 * big)
                    assert (np.abs(row - want) <= half * (1 + 2.0 ** -10) + 2.0 ** -20 * big).all()
            a, tol = bkv.attention(bkv.rotated(L.q, HEADS, at), np.concatenate([p[0], k[:seen]]),
                                   np.concatenate([p[1], v[:seen]]))
            want, bound = bkv.o_layer(L, a, tol)
            want = want + h[i, t]
            off = np.abs(got[i, t] - want) - bound - 2 * EPS * np.abs(want)
            assert (off <= 0).all(), f"sequence {i}, token {t}: past its bound by {off.max()}"
    block.close()


def test_a_step_past_the_capacity_stays_within_it(ctx, orc):
    """Tokens behind the last row are not written, and nothing outside the buffer is; the other sequences' results are
    those of a step without it."""
    L = bkv.Layers(ctx, orc, 6)
    D, KV, HD = bkv.D, bkv.KV, bkv.HD
    block = DecoderBlock(ctx, L.all, np.ones(D), np.ones(D), bkv.HEADS, KV, HD, bkv.THETA, 1e-5, capacity=400)
    n, per, cap = 3, 4, 70
    outs, rows = [], []
    for lens in ([10, 5, 60], [10, 68, 60], [10, 2 ** 31 - 1, 60]):
        size = att.KvCache.size("fp4", n, cap, KV, HD)
        buf = torch.zeros(size + 4096, dtype=torch.uint8, device="cuda")
        cache = att.KvCache(ctx, "fp4", n, cap, KV, HD, buf)
        bkv.fill(cache, np.random.default_rng(3), [cap] * n)
        h = torch.from_numpy(np.random.default_rng(4).standard_normal((n, per, D)).astype(np.float32)).cuda()
        need = block.decode_kv_workspace_size(cache, n, n_tokens=per)
        block.decode_kv_dev(h, words(lens), n, cache, torch.empty(need, dtype=torch.uint8, device="cuda"), need,
                            n_tokens=per)
        torch.cuda.synchronize()
        assert int(buf[size:].sum()) == 0
        outs.append(h[[0, 2]].clone())
        rows.append(bkv.held(cache, [cap] * n)[1])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert all(np.array_equal(rows[1][x][:68], rows[2][x][:68]) for x in range(2))


def test_refusals(ctx, orc):
    L = bkv.Layers(ctx, orc, 7)
    block = DecoderBlock(ctx, L.all, np.ones(bkv.D), np.ones(bkv.D), bkv.HEADS, bkv.KV, bkv.HD, bkv.THETA, 1e-5, capacity=100)
    cache = bkv.make(ctx, "fp4", 40, 60)
    need = block.decode_kv_workspace_size(cache, 4, n_tokens=3)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert block.decode_kv_workspace_size(cache, 33, n_tokens=2) == 0 and block.decode_kv_workspace_size(cache, 4, n_tokens=0) == 0

    def refused(says, h=12, **kw):
        a = dict(pos=words([0] * 40), n=4, cache=cache, workspace=ws, workspace_size=need, n_tokens=3)
        a.update(kw)
        with pytest.raises(KernelError, match=says):
            block.decode_kv_dev(torch.zeros((h, bkv.D), device="cuda"), **a)

    refused("batched decode input must be", h=11)
    refused("workspace of .* is smaller than the", workspace_size=need - 1)
    refused("takes 1 .. 64 rows, got 66 of 2 tokens", h=66, n=33, n_tokens=2)
    refused("takes 1 .. 64 tokens a sequence, got 65", h=65, n=1, n_tokens=65)
    refused("takes 1 .. 64 tokens a sequence, got 0", h=0, n_tokens=0)
    refused("negative", h=12, n=-4, n_tokens=-3)
    refused("positions must be", pos=words([0] * 3))
    block.close()


# ---- a model's drafts ------------------------------------------------------------

def near(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("fmt", ["int8", "fp4"])
def test_drafts_behind_a_shared_prompt(ctx, orc, fmt):
    """Greedy requests by drafts, right, wrong and partly right, against the same requests a token at a time: the logits
    behind every kept token are those of the step there (the projections of many rows are another kernel's: within 2 %, the
    gate of the steps themselves), what is emitted is the logits' own argmax, and what was not kept leaves no trace."""
    from test_gpu_trunk import synthetic_model

    from quantibbler_amd.model import DeviceModel

    md = synthetic_model(orc, 808)
    rng = np.random.default_rng(12)
    prompt, n, cap, steps = rng.integers(0, md.vocab_size, 65).tolist(), 3, 24, 12
    m = DeviceModel(ctx, md, capacity=65 + cap)
    m.share_prefix(prompt, n, cap, fmt=fmt)
    ids = [rng.integers(0, md.vocab_size, n).tolist()]
    logits = []
    for _ in range(steps):
        logits.append(m.step_shared(ids[-1]).clone())
        ids.append(logits[-1].argmax(-1).tolist())
    ids = np.array(ids)            # [steps + 1][n]: ids[t] is fed at row t, logits[t] behind it
    m.share_prefix(prompt, n, cap, fmt=fmt)
    cold = torch.zeros(n, device="cuda")
    at = np.zeros(n, int)          # rows that each request holds
    last = ids[0].copy()
    for call, k in enumerate((0, 3, 2, 4, 1)):
        rows = np.zeros((n, k + 1), np.int64)
        for i in range(n):
            rows[i, 0] = last[i]
            for j in range(k):
                t = at[i] + 1 + j
                right = t < len(ids) and not (call == 2 and j == i)
                rows[i, 1 + j] = ids[t, i] if right else (ids[min(t, steps), i] + 1) % md.vocab_size
        tokens = words(rows.reshape(-1)).view(n, k + 1)
        u = torch.rand((n, k + 1), device="cuda")
        drafts = None
        if call % 2 and k:         # a draft model that is sure of its drafts: greedy all the same
            drafts = torch.zeros((n, k, md.vocab_size), device="cuda").scatter_(2, tokens[:, 1:, None].long(), 30.0)
        out, counts = m.verify_shared(tokens if call != 1 else rows.tolist(), u, draft_logits=drafts, temperature=cold)
        torch.cuda.synchronize()
        mine = m._shared["drafts"][k + 1]["logits"].view(n, k + 1, -1)
        best = mine.argmax(-1).cpu().numpy()
        out, counts = out.cpu().numpy(), counts.cpu().numpy()
        assert m._shared["pos"].tolist() == (at + counts).tolist()
        for i in range(n):
            kept = 0
            while kept < k and rows[i, 1 + kept] == best[i, kept]:
                kept += 1
            assert counts[i] == kept + 1 and out[i].tolist() == rows[i, 1:1 + kept].tolist() + [best[i, kept]] + [-1] * (k - kept)
            for j in range(kept + 1):
                # while its history is the stepped one's
                if at[i] + j < steps and rows[i, j] == ids[at[i] + j, i]:
                    assert near(mine[i, j], logits[at[i] + j][i]) <= 0.02, f"call {call}, request {i}, token {j}"
            last[i] = out[i, kept]
            at[i] += counts[i]
            if at[i] < len(ids) and last[i] != ids[at[i], i]:
                pytest.skip("two ids within a rounding of each other")  # another history from here on
    assert m._shared["steps"] == 1 + 4 + 3 + 5 + 2  # a bound: what was not kept counts too
    # one step goes on from there, behind rows that were taken back
    t = int(at.min())
    if (at == t).all() and t < steps:
        got = m.step_shared(last.tolist())
        assert all(near(got[i], logits[t][i]) <= 0.02 for i in range(n))
    m.close()


def test_the_room_that_is_left(ctx, orc):
    """The bound on a request's rows is looked up when it does not do; what has no room is refused before anything runs."""
    from test_gpu_trunk import synthetic_model

    from quantibbler_amd.model import DeviceModel

    m = DeviceModel(ctx, synthetic_model(orc, 808), capacity=40)
    with pytest.raises(ValueError, match="needs share_prefix first"):
        m.verify_shared([[1]], torch.zeros((1, 1), device="cuda"))
    m.share_prefix([1, 2, 3, 4, 5], 2, 8, fmt="fp4")
    u = torch.full((2, 4), 0.5, device="cuda")
    cold = torch.zeros(2, device="cuda")
    wrong = [[3, 0, 0, 0], [4, 0, 0, 0]]
    held = 0
    for _ in range(10):
        before = m._shared["pos"].tolist()
        if max(before) + 4 > 8:
            break
        _, counts = m.verify_shared(wrong, u, temperature=cold)
        held = max(b + c for b, c in zip(before, counts.tolist()))
    assert held + 4 > 8 and m._shared["pos"].max().item() == held
    with pytest.raises(ValueError, match=f"no room for 4 rows behind {held} of a capacity of 8"):
        m.verify_shared(wrong, u, temperature=cold)
    for _ in range(8 - held):
        m.step_shared([1, 2])
    with pytest.raises(ValueError, match="the requests hold their 8 rows already"):
        m.step_shared([1, 2])
    for bad in ([[1, 2]], [1, 2], torch.zeros((2, 33), dtype=torch.int32, device="cuda")):
        with pytest.raises((ValueError, TypeError)):
            m.verify_shared(bad, u)
    m.close()


def test_a_captured_call_and_another_stream(ctx, orc):
    """A captured verification replayed at the positions after it: the eager calls' results, bit for bit; the eager ones
    on a stream of their own."""
    from test_gpu_trunk import synthetic_model

    from quantibbler_amd.model import DeviceModel

    md = synthetic_model(orc, 808)
    rng = np.random.default_rng(5)
    n, k, cap = 3, 2, 24
    prompt = rng.integers(0, md.vocab_size, 33).tolist()
    models = [DeviceModel(ctx, md, capacity=33 + cap) for _ in range(2)]
    for m in models:
        m.share_prefix(prompt, n, cap, fmt="fp4")
    torch.cuda.synchronize()
    tokens = torch.zeros((n, k + 1), dtype=torch.int32, device="cuda")
    u, drafts = torch.zeros((n, k + 1), device="cuda"), torch.zeros((n, k, md.vocab_size), device="cuda")
    heat = torch.full((n,), 0.7, device="cuda")
    s = torch.cuda.Stream()
    graph = None
    for rep in range(5):
        tokens.copy_(words(rng.integers(0, md.vocab_size, n * (k + 1))).view(n, k + 1))
        u.copy_(torch.from_numpy(rng.random((n, k + 1)).astype(np.float32)))
        drafts.normal_()
        torch.cuda.synchronize()
        want = models[1].verify_shared(tokens, u, draft_logits=drafts, temperature=heat, stream=s)
        s.synchronize()
        if rep == 0:
            got = models[0].verify_shared(tokens, u, draft_logits=drafts, temperature=heat)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = models[0].verify_shared(tokens, u, draft_logits=drafts, temperature=heat,
                                              stream=torch.cuda.current_stream())
        else:
            graph.replay()
            got = out
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(models[0]._shared["pos"], models[1]._shared["pos"])
        assert torch.equal(models[0]._shared["drafts"][k + 1]["logits"], models[1]._shared["drafts"][k + 1]["logits"])
    del graph
    for m in models:
        m.close()


# ---- the operators one after the other ----------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_program_of_its_own(ctx, dtype):
    """A fused projection's rows of drafted tokens: heads normed and rotated in place, keys and values into the 4-bit
    cache, attention behind a shared prompt, a head, verification -- each against its own definition on what the one
    before gave it, eager and replayed."""
    n, per, heads, kv, d, plen, vocab, cap = 5, 4, 8, 2, 128, 300, 1501, 64
    k, rows, width = per - 1, n * per, (heads + 2 * kv) * d
    t = getattr(torch, dtype)
    shared, cache = att.make(ctx, "fp4", 1, plen, kv, d), att.make(ctx, "fp4", n, cap, kv, d)
    p = att.fill(shared, 140, [plen])[0]
    lens = [0, 3, 49, 20, 60]
    att.fill(cache, 141, lens)
    rope = Rope(d, 10000.0, rotary_dim=64, scaling={"kind": "linear", "factor": 2.0})
    wq, wk = torch.rand(d, device="cuda") + 0.5, torch.rand(d, device="cuda") + 0.5
    qkv, pos = torch.empty((rows, width), dtype=t, device="cuda"), words(lens)
    out = torch.empty((n, per, heads, d), dtype=t, device="cuda")
    q, kk, vv = qkv[:, :heads * d], qkv[:, heads * d:(heads + kv) * d], qkv[:, (heads + kv) * d:]
    head = LmHead.from_rows(ctx, np.random.default_rng(3).standard_normal((vocab, heads * d)).astype(np.float32) * 0.1)
    logits, wide = torch.empty((rows, vocab), device="cuda"), torch.empty((rows, heads * d), device="cuda")
    ids, u = torch.zeros((n, k), dtype=torch.int32, device="cuda"), torch.empty((n, per), device="cuda")
    tokens, counts = torch.empty((n, per), dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    now = torch.empty_like(pos)
    need = cache.attention_workspace_size(heads, n, seq_q=per, prefix_len=plen)
    vneed = verify_drafts_workspace_size(n, k, vocab)
    ws, vws = (torch.empty(x, dtype=torch.uint8, device="cuda") for x in (need, vneed))
    queries = torch.empty((rows, heads, d), dtype=t, device="cuda")

    def step():
        s = torch.cuda.current_stream()
        rotate_heads_dev(ctx, rope, q, kk, dtype, rows, heads, kv, pos, queries, kk, n_seqs=n, before=plen, q_norm=wq,
                         k_norm=wk, eps=1e-5, q_stride=width, k_stride=width, k_out_stride=width, stream=s)
        cache.write_dev(kk, vv, dtype, pos, rows, row_stride=width, stream=s)
        torch.add(pos, per, out=now)
        cache.attention_dev(queries, dtype, heads, now, out, ws, need, seq_q=per, prefix=shared, prefix_len=plen, stream=s)
        wide.copy_(out.view(rows, heads * d))
        head.logits_dev(wide, rows, logits, stream=s)
        verify_drafts_dev(ctx, logits, n, k, vocab, ids, u, tokens, counts, vws, vneed, pos=pos, stream=s)

    def fresh(seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=g).to(t))
        ids.random_(0, vocab, generator=g)
        u.copy_(torch.rand(u.shape, device="cuda", generator=g) * (0.999 if seed % 2 else 0.001))
        pos.copy_(words(lens))

    def check(label):
        old = raw.double().cpu().numpy()
        at = [plen + x + j for x in lens for j in range(per)]
        rot_q = rot.reference(old[:, :heads * d].reshape(rows, heads, d), wq.cpu().numpy(), at, 10000.0, 64, False,
                              {"kind": "linear", "factor": 2.0})
        rot.check(queries, *rot_q, f"{label}: queries")
        rot_k = rot.reference(old[:, heads * d:(heads + kv) * d].reshape(rows, kv, d), wk.cpu().numpy(), at, 10000.0, 64,
                              False, {"kind": "linear", "factor": 2.0})
        rot.check(kk.reshape(rows, kv, d), *rot_k, f"{label}: keys")
        held = [min(x + per, cap) for x in lens]
        ko = torch.empty((sum(held), kv, d), device="cuda")
        vo = torch.empty_like(ko)
        cache.read_dev(ko, vo, "float32", words([0] * n), sum(held), row_start=words(np.concatenate([[0], np.cumsum(held)])))
        own, a = [], 0
        for r in held:
            own.append((ko[a:a + r].double(), vo[a:a + r].double()))
            a += r
        att.check(out, *att.reference(queries.view(n, per, heads, d), p, own, held), f"{label}: attention")
        ver.check(tokens, counts, logits.view(n, per, vocab), None, ids, u, None, None, label)
        assert pos.tolist() == [x + c for x, c in zip(lens, counts.tolist())]

    fresh(1)
    raw = qkv.clone()
    step()
    torch.cuda.synchronize()
    check("eager")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rep in range(2, 5):
        fresh(rep)
        raw = qkv.clone()
        graph.replay()
        torch.cuda.synchronize()
        check(f"replay {rep}")
    del graph
    head.close()


def test_two_captured_calls_that_share_a_workspace(ctx):
    """Verification and attention of two sizes captured apart on one workspace, replayed in turn and in any order: the
    eager calls' results; the same calls on two streams at once, each with a workspace of its own, too."""
    vocab, kv, heads, d = 5003, 2, 8, 128
    cache, held = att.make(ctx, "fp4", 6, 700, kv, d), [700, 64, 5, 333, 650, 5]
    att.fill(cache, 150, held)
    jobs = []
    for n, k in ((6, 3), (2, 1)):
        per = k + 1
        x, y = torch.randn((n * per, vocab), device="cuda") * 3, torch.randn((n * k, vocab), device="cuda") * 3
        ids = torch.randint(0, vocab, (n, k), dtype=torch.int32, device="cuda")
        u = torch.rand((n, per), device="cuda")
        tok, cnt = torch.empty((n, per), dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
        q = torch.randn((n, per, heads, d), device="cuda")
        lens, out = words(held[:n]), torch.empty_like(q)
        need = max(verify_drafts_workspace_size(n, k, vocab), cache.attention_workspace_size(heads, n, seq_q=per))

        def run(ws, s, n=n, k=k, per=per, x=x, y=y, ids=ids, u=u, tok=tok, cnt=cnt, q=q, lens=lens, out=out, need=need):
            verify_drafts_dev(ctx, x, n, k, vocab, ids, u, tok, cnt, ws, need, draft_logits=y, stream=s)
            cache.attention_dev(q, "float32", heads, lens, out, ws, need, n_seqs=n, seq_q=per, stream=s)
        jobs.append((run, need, (tok, cnt, out), (x, u, q)))
    shared = torch.full((max(j[1] for j in jobs),), 0xFF, dtype=torch.uint8, device="cuda")
    apart = [torch.full((j[1],), 0xFF, dtype=torch.uint8, device="cuda") for j in jobs]
    streams, graphs = [torch.cuda.Stream() for _ in jobs], []
    for run, _, _, _ in jobs:
        run(shared, torch.cuda.current_stream())
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run(shared, torch.cuda.current_stream())
    for order in ((0, 1), (1, 0), (0, 0, 1, 1, 0)):
        for _, _, _, inputs in jobs:
            inputs[0].normal_(), inputs[1].uniform_(0.0, 0.999), inputs[2].normal_()
        torch.cuda.synchronize()
        want = []
        for (run, _, outs, _), ws in zip(jobs, apart):
            run(ws, torch.cuda.current_stream())
            torch.cuda.synchronize()
            want.append([t.clone() for t in outs])
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for (_, _, outs, _), w in zip(jobs, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, w))
            for t in outs:
                t.zero_()
        torch.cuda.synchronize()
        for (run, _, _, _), ws, st in zip(jobs, apart, streams):
            run(ws, st)
        torch.cuda.synchronize()
        for (_, _, outs, _), w in zip(jobs, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, w))
    del graphs
