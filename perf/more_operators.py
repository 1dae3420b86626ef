"""Serving with drafted tokens over a 4-bit KV cache, as timed cases: heads
normed and rotated, rows in and out of the cache, the attention that reads it
and the verification of the drafts.

``own`` false computes each operator in its plain form, elementary torch
operations in 32 bits (angles and probabilities in 64); ``own`` true makes the
calls of a program built on this library: ``rotate_heads_dev``, ``KvCache`` of
the format "fp4" (``write_dev``, ``read_dev``, ``attention_dev``) and
``verify_drafts_dev``.  Heads and widths are those of the repository's
4096-wide block (32 query heads, 8 kv heads of 128 channels, a 128256-row
vocabulary) or generic; inputs are made from the seed alone.
"""
import math
import random

import torch

own = False

DEV = "cuda"
FLOOR = 2.0 ** -100
GROUP = 32       # channels that share a multiplier
TOP = 448.0      # the largest multiplier, 6 the largest code
EPS = 1e-6


def listed():
    return [
        # a batched decode step's rows, out of the fused q/k/v rows of 32 sequences: the call's latency counts
        {"name": "cache4-step", "kind": "cache", "dtype": "bfloat16", "kv_heads": 8, "d": 128, "seqs": 32,
         "longest": 1, "mix": 0, "at": 2085, "fused": True},
        # prompts of unlike length written in one call and read back, some of them chunks that continue one
        {"name": "cache4-prompts", "kind": "cache", "dtype": "float32", "kv_heads": 8, "d": 128, "seqs": 6,
         "longest": 4001, "mix": 5, "at": 450, "fused": False},
        # one sequence's decode step without a prefix: latency
        {"name": "attend4-token", "kind": "attend", "dtype": "float32", "heads": 32, "kv_heads": 8, "d": 128,
         "seqs": 1, "longest": 700, "mix": 0, "queries": 1, "prefix": 0},
        # a batched decode step of 32 sequences of unlike length
        {"name": "attend4-step", "kind": "attend", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "d": 128,
         "seqs": 32, "longest": 2085, "mix": 0, "queries": 1, "prefix": 0},
        # five tokens of each of 16 requests, four of them drafted, behind one prompt; one query head a kv head
        {"name": "attend4-draft", "kind": "attend", "dtype": "float32", "heads": 8, "kv_heads": 8, "d": 80,
         "seqs": 16, "longest": 290, "mix": 5, "queries": 5, "prefix": 4001},
        # 64 requests behind a long document, the largest attention
        {"name": "attend4-wide", "kind": "attend", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "d": 128,
         "seqs": 64, "longest": 2048, "mix": 0, "queries": 1, "prefix": 16384},
        # one request's drafts looked up in its own text, which have no distribution: latency
        {"name": "verify-token", "kind": "verify", "dtype": "float32", "seqs": 1, "drafts": 3, "vocab": 32003,
         "given": False, "ragged": 0, "greedy": False, "masked": False},
        # unlike numbers of drafts over a vocabulary of odd size in bf16, some of it forbidden, some requests greedy
        {"name": "verify-mixed", "kind": "verify", "dtype": "bfloat16", "seqs": 12, "drafts": 7, "vocab": 50021,
         "given": True, "ragged": 3, "greedy": True, "masked": True},
        # 32 requests' four drafted tokens each against a draft model's distributions (the largest)
        {"name": "verify-step", "kind": "verify", "dtype": "float32", "seqs": 32, "drafts": 4, "vocab": 128256,
         "given": True, "ragged": 0, "greedy": False, "masked": False},
        # one token's heads, normed and rotated: latency
        {"name": "rotate-token", "kind": "rotate", "dtype": "float32", "heads": 32, "kv_heads": 8, "d": 128,
         "rotary": 128, "interleaved": False, "scaling": "none", "normed": True, "seqs": 1, "longest": 1, "mix": 0,
         "at": 2085, "before": 0, "fused": True},
        # a batched step's, a quarter of the head in neighbouring pairs, out of the fused rows
        {"name": "rotate-step", "kind": "rotate", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "d": 128,
         "rotary": 32, "interleaved": True, "scaling": "linear", "normed": False, "seqs": 64, "longest": 1, "mix": 0,
         "at": 2085, "before": 8192, "fused": True},
        # a long prompt's, far positions of a stretched context
        {"name": "rotate-prompt", "kind": "rotate", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "d": 128,
         "rotary": 128, "interleaved": False, "scaling": "ramp", "normed": True, "seqs": 1, "longest": 8192, "mix": 0,
         "at": 100003, "before": 0, "fused": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "cache", "attend", "attend", "attend", "verify", "verify", "rotate", "rotate"])
    dtype = rng.choice(["float32", "bfloat16"])
    kv, d = rng.choice([1, 2, 5, 8]), rng.choice([16, 64, 80, 128, 128, 256])
    n, mix = _log(rng, 1, 64), rng.choice([0, rng.randint(1, 1 << 20), rng.randint(1, 1 << 20)])
    if kind == "cache":
        return {"kind": kind, "dtype": dtype, "kv_heads": kv, "d": d, "seqs": n,
                "longest": _log(rng, 1, max(1, 8192 // n)), "mix": mix, "at": rng.randint(0, 1000),
                "fused": rng.random() < 0.4}
    if kind == "attend":
        group, queries = rng.choice([1, 2, 4, 7]), rng.choice([1, 1, 1, 2, 5, 16])
        prefix = rng.choice([0, _log(rng, 1, 16384), _log(rng, 64, 16384)])
        keys = int(1.8e10 / (4 * d * kv * group * queries * n))  # no more products than the largest listed case has
        prefix = min(prefix, keys)
        return {"kind": kind, "dtype": dtype, "heads": kv * group, "kv_heads": kv, "d": d, "seqs": n,
                "longest": _log(rng, 1, max(1, min(2048, keys - prefix))), "mix": mix, "queries": queries,
                "prefix": prefix}
    if kind == "verify":
        drafts, vocab = rng.choice([0, 1, 2, 3, 4, 5, 8, 16]), _log(rng, 2, 200000)
        n = min(n, max(1, 32 * 9 * 128256 // (vocab * (2 * drafts + 1))))
        return {"kind": kind, "dtype": dtype, "seqs": n, "drafts": drafts, "vocab": vocab,
                "given": drafts > 0 and rng.random() < 0.7, "ragged": rng.choice([0, rng.randint(1, 1 << 20)]),
                "greedy": rng.random() < 0.4, "masked": rng.random() < 0.4}
    rotary = rng.choice([d, d, d // 2, max(2, d // 4)])
    group = rng.choice([1, 2, 4, 7])
    return {"kind": kind, "dtype": dtype, "heads": kv * group, "kv_heads": kv, "d": d, "rotary": rotary,
            "interleaved": rng.random() < 0.4, "scaling": rng.choice(["none", "linear", "base", "ramp", "yarn"]),
            "normed": rng.random() < 0.5, "seqs": n, "longest": _log(rng, 1, max(1, 8192 // n)), "mix": mix,
            "at": _log(rng, 1, 200000), "before": rng.choice([0, rng.randint(1, 20000)]),
            "fused": rng.random() < 0.5}


# ---- inputs ------------------------------------------------------------------

def _lengths(case):
    """Rows of each sequence, the longest among them: evenly down to half of it, or (mix) spread over the logarithm,
    some with none."""
    n, longest = case["seqs"], case["longest"]
    if not case["mix"]:
        return [longest - (i * (longest // 2)) // n for i in range(n)]
    rng = random.Random(case["mix"])
    out = [_log(rng, 1, longest) if rng.random() < 0.9 else 0 for _ in range(n)]
    out[rng.randrange(n)] = longest
    return out


def _first_rows(case):
    """The position of each sequence's first row."""
    n, at = case["seqs"], case["at"]
    return [at - (i * at) // n for i in range(n)]


def _generator(seed, tag):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + int(tag))
    return g


def _normal(seed, tag, shape):
    return torch.randn(shape, device=DEV, generator=_generator(seed, tag))


def _uint32(values):
    return torch.tensor([int(v) for v in values], dtype=torch.int32, device=DEV)


def _starts(rows):
    out = [0]
    for r in rows:
        out.append(out[-1] + r)
    return out


def _kv_rows(seed, tag, n, kv, d, dtype):
    """Keys with a channel mean, as trained models have, and values of unlike size by token."""
    k = _normal(seed, tag, (n, kv, d)) + 2.0 * _normal(seed, 90, (1, kv, d))
    v = _normal(seed, tag + 1, (n, kv, d)) * torch.exp(0.5 * _normal(seed, tag + 2, (n, kv, 1)))
    return k.to(dtype), v.to(dtype)


def _cache_inputs(case, seed):
    kv, d, n = case["kv_heads"], case["d"], sum(_lengths(case))
    dtype = getattr(torch, case["dtype"])
    k, v = _kv_rows(seed, 10, n, kv, d, dtype)
    if not case["fused"]:
        return k, v
    rows = torch.zeros((n, 6 * kv * d), dtype=dtype, device=DEV)  # q | k | v of a projection's rows
    rows[:, 4 * kv * d:5 * kv * d] = k.view(n, kv * d)
    rows[:, 5 * kv * d:] = v.view(n, kv * d)
    return rows[:, 4 * kv * d:5 * kv * d].view(n, kv, d), rows[:, 5 * kv * d:].view(n, kv, d)


def _attend_inputs(case, seed):
    """q [n][queries][heads][d]; the prefix's and every sequence's key and value rows [.][kv_heads][d], f32."""
    n, dtype = case["seqs"], getattr(torch, case["dtype"])
    q = (1.5 * _normal(seed, 1, (n, case["queries"], case["heads"], case["d"]))).to(dtype)
    own_rows = _kv_rows(seed, 10, sum(_lengths(case)), case["kv_heads"], case["d"], torch.float32)
    return q, _kv_rows(seed, 20, case["prefix"], case["kv_heads"], case["d"], torch.float32), own_rows


def _counts(case):
    """How many drafts each request has."""
    n, k = case["seqs"], case["drafts"]
    if not case["ragged"]:
        return [k] * n
    rng = random.Random(case["ragged"])
    out = [rng.randint(0, k) for _ in range(n)]
    out[rng.randrange(n)] = k
    return out


def _verify_inputs(case, seed):
    """Target logits [n][k + 1][vocab], the draft model's [n][k][vocab] near them (None where the drafts come from a
    text), drafted ids [n][k], uniform numbers [n][k + 1] and a temperature a request."""
    n, k, vocab, dtype = case["seqs"], case["drafts"], case["vocab"], getattr(torch, case["dtype"])
    x = _normal(seed, 1, (n, k + 1, vocab)).mul_(2.5)
    likely = torch.randint(0, vocab, (n, k + 1, 6), device=DEV, generator=_generator(seed, 2))
    x.scatter_(2, likely, (9.0 + 2.0 * _normal(seed, 3, (n, k + 1, 1))).expand(n, k + 1, 6))  # alike: an id may come twice
    if case["masked"]:  # a grammar's or a sampler's forbidden tokens
        forbidden = _normal(seed, 4, (1, 1, vocab)) > 1.0
        forbidden[0, 0, 0] = False
        x.masked_fill_(forbidden, float("-inf"))
    temperature = torch.rand(n, device=DEV, generator=_generator(seed, 5)) + 0.5
    if case["greedy"]:
        temperature[::3] = 0.0
    y = (x[:, :k] + 0.5 * _normal(seed, 6, (n, k, vocab))).to(dtype)
    warm = torch.where(temperature > 0, temperature, torch.full_like(temperature, 0.05)).view(n, 1, 1)
    noise = -torch.log(-torch.log(torch.rand((n, k, vocab), device=DEV, generator=_generator(seed, 7)) * 0.999998 + 1e-6))
    ids = (y.float() / warm + noise).argmax(dim=-1).to(torch.int32) if k else torch.zeros((n, 0), dtype=torch.int32,
                                                                                          device=DEV)
    u = torch.rand((n, k + 1), device=DEV, generator=_generator(seed, 8))
    return x.to(dtype), y if case["given"] else None, ids, u, temperature


SCALINGS = {  # a context stretched in each of the usual ways
    "none": None,
    "linear": {"kind": "linear", "factor": 4.0},
    "base": {"kind": "base", "factor": 4.0},
    "ramp": {"kind": "ramp", "factor": 8.0, "original_len": 8192, "low": 1.0, "high": 4.0},
    "yarn": {"kind": "yarn", "factor": 16.0, "original_len": 4096, "low": 1.0, "high": 32.0},
}
THETA = 500000.0


def _rotate_inputs(case, seed):
    """q [rows][heads][d] and k [rows][kv_heads][d], in the fused rows of a projection or apart, and norm weights."""
    n, heads, kv, d = sum(_lengths(case)), case["heads"], case["kv_heads"], case["d"]
    dtype = getattr(torch, case["dtype"])
    q, k = (2.0 * _normal(seed, 1, (n, heads, d))).to(dtype), (2.0 * _normal(seed, 2, (n, kv, d))).to(dtype)
    if case["fused"]:
        rows = torch.zeros((n, (heads + 2 * kv) * d), dtype=dtype, device=DEV)
        rows[:, :heads * d] = q.view(n, heads * d)
        rows[:, heads * d:(heads + kv) * d] = k.view(n, kv * d)
        q, k = rows[:, :heads * d].view(n, heads, d), rows[:, heads * d:(heads + kv) * d].view(n, kv, d)
    weights = (None, None)
    if case["normed"]:
        weights = 1.0 + 0.2 * _normal(seed, 3, (d,)), 1.0 + 0.2 * _normal(seed, 4, (d,))
    return q, k, weights


# ---- the plain forms -----------------------------------------------------------

def _grouped(x, d):
    """[.][d] -> [.][groups][32], the last group filled up with zeros."""
    groups = -(-d // GROUP)
    wide = torch.zeros(x.shape[:-1] + (groups * GROUP,), dtype=x.dtype, device=x.device)
    wide[..., :d] = x
    return wide.view(x.shape[:-1] + (groups, GROUP))


def _quantise(x):
    """Rows [.][kv_heads][d] -> codes times multipliers, and one f32 scale a row and head."""
    x = x.float()
    d = x.shape[-1]
    top = x.abs().amax(dim=-1, keepdim=True)
    whole = torch.isfinite(top)
    top = torch.where(whole, top, torch.ones_like(top)).clamp_min(FLOOR)
    x = torch.where(whole, x, torch.zeros_like(x))
    per = 1.0 / top
    g = _grouped(x, d)
    mult = (g.abs().amax(dim=-1, keepdim=True) * (TOP * per).unsqueeze(-1)).to(torch.float8_e4m3fn).float()
    by = torch.where(mult > 0, 1.0 / mult, torch.zeros_like(mult))
    z = (g * (6.0 * TOP * per).unsqueeze(-1)) * by
    a = z.abs()
    code = 0.5 * ((a > 0.25).float() + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) + (a > 2.5).float() + (a >= 3.5) \
        + 2.0 * (a > 5.0)
    held = (torch.where(z < 0, -code, code) * mult).flatten(-2)[..., :d]
    return held, torch.where(whole, top * (1.0 / (6.0 * TOP)), torch.full_like(top, float("nan")))


def _plain_attend(s):
    n, sq, heads, kv, d = s["seqs"], s["queries"], s["heads"], s["kv_heads"], s["d"]
    group, dtype = heads // kv, s["q"].dtype
    q = s["q"].float().view(n, sq, kv, group, d).permute(2, 0, 1, 3, 4).contiguous()  # [kv][n][sq][group][d]
    pk, pv = ((codes * scales).permute(1, 0, 2).contiguous() for codes, scales in s["prefix_rows"])  # [kv][prefix][d]
    ok, ov = ((codes * scales).permute(2, 0, 1, 3).contiguous() for codes, scales in s["own_rows"])  # [kv][n][longest][d]
    longest, prefix = ok.shape[2], pk.shape[1]
    rows = sq * group
    scale = 1.0 / math.sqrt(d)
    sp = torch.matmul(q.view(kv, n * rows, d), pk.transpose(1, 2).contiguous()).view(kv, n, rows, prefix)
    so = torch.matmul(q.view(kv, n, rows, d), ok.transpose(2, 3).contiguous())        # [kv][n][rows][longest]
    limit = (s["lens_dev"].view(n, 1) - sq + 1 + torch.arange(sq, device=DEV).view(1, sq))  # own rows a query sees
    seen = torch.arange(longest, device=DEV).view(1, 1, longest) < limit.view(n, sq, 1)
    seen = seen.view(n, sq, 1, longest).expand(n, sq, group, longest).reshape(n, rows, longest)
    scores = torch.cat([sp, so.masked_fill(~seen, float("-inf"))], dim=-1) * scale
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p[..., :prefix].reshape(kv, n * rows, prefix), pv).view(kv, n, rows, d)
    out = out + torch.matmul(p[..., prefix:].contiguous(), ov)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.view(kv, n, sq, group, d).permute(1, 2, 0, 3, 4).reshape(n, sq, heads, d).to(dtype)


def _probabilities(x, temperature):
    """softmax(x / temperature) in 64 bits; at temperature 0 all of it on the largest, the lowest id first."""
    x = x.double()
    hot = torch.where(temperature > 0, temperature, torch.ones_like(temperature)).double().view(-1, 1)
    e = torch.exp((x - x.amax(dim=-1, keepdim=True)) / hot)
    best = torch.zeros_like(e).scatter_(1, x.argmax(dim=-1, keepdim=True), 1.0)
    return torch.where((temperature > 0).view(-1, 1), e / e.sum(dim=-1, keepdim=True), best)


def _plain_verify(s):
    n, k = s["seqs"], s["drafts"]
    counts, ids, t = s["counts"], s["ids"].long(), s["temperature"]
    tokens = torch.full((n, k + 1), -1, dtype=torch.int32, device=DEV)
    going = torch.ones(n, dtype=torch.bool, device=DEV)
    accepted = torch.zeros(n, dtype=torch.int32, device=DEV)
    for j in range(k + 1):
        p = _probabilities(s["logits"][:, j], t)
        rest = p
        take = torch.zeros(n, dtype=torch.bool, device=DEV)
        if j < k:
            drafted = j < counts
            at = ids[:, j:j + 1]
            if s["draft_logits"] is None:
                q = torch.zeros_like(p).scatter_(1, at, 1.0)
            else:
                q = _probabilities(s["draft_logits"][:, j], t)
            take = going & drafted & ((s["uniforms"][:, j].double() * q.gather(1, at)[:, 0]) < p.gather(1, at)[:, 0])
            less = (p - q).clamp_min(0.0)
            less = torch.where(less.sum(dim=-1, keepdim=True) > 0, less, p)
            rest = torch.where(drafted.view(n, 1), less, p)
        ends = going & ~take
        sums = rest.cumsum(dim=-1)
        u = s["uniforms"].gather(1, counts.view(n, 1).long()).double() * sums[:, -1:]
        token = ((sums > u) & (rest > 0)).to(torch.uint8).argmax(dim=-1)
        tokens[:, j] = torch.where(ends, token, torch.where(take, ids[:, min(j, k - 1)] if k else token,
                                                            torch.full_like(token, -1))).to(torch.int32)
        accepted += take.to(torch.int32)
        going = take
    return {"tokens": tokens, "counts": accepted + 1}


def _frequencies(rotary, scaling):
    """Radians a position of each pair, and the factor on cos and sin."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device=DEV)
    kind = scaling["kind"] if scaling else "none"
    theta = THETA
    if kind == "base" and rotary > 2:
        theta = THETA * scaling["factor"] ** (rotary / (rotary - 2))
    f = theta ** (-2.0 * i / rotary)
    if kind == "linear":
        return f / scaling["factor"], 1.0
    if kind == "ramp":  # by the turns that a pair makes within the original context
        turns = scaling["original_len"] * f / (2.0 * math.pi)
        keep = ((turns - scaling["low"]) / (scaling["high"] - scaling["low"])).clamp(0.0, 1.0)
        return f * keep + f / scaling["factor"] * (1.0 - keep), 1.0
    if kind == "yarn":  # by the pair's number, between those that make `high` and `low` turns there
        def pair(turns):
            return rotary * math.log(scaling["original_len"] / (turns * 2.0 * math.pi)) / (2.0 * math.log(THETA))

        first = max(math.floor(pair(scaling["high"])), 0)
        last = min(math.ceil(pair(scaling["low"])), rotary - 1)
        keep = 1.0 - ((i - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        return f * keep + f / scaling["factor"] * (1.0 - keep), 0.1 * math.log(scaling["factor"]) + 1.0
    return f, 1.0


def _plain_rotate(s):
    d, rotary = s["d"], s["rotary"]
    f, size = _frequencies(rotary, SCALINGS[s["scaling"]])
    angle = (s["positions"].double() + s["before"]).view(-1, 1) * f.view(1, -1)
    c, sn = ((torch.cos(angle) * size).float().unsqueeze(1), (torch.sin(angle) * size).float().unsqueeze(1))
    out = []
    for x, w in ((s["q"], s["weights"][0]), (s["k"], s["weights"][1])):
        dtype = x.dtype
        x = x.float()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w
        r = x[..., :rotary]
        a, b = (r[..., 0::2], r[..., 1::2]) if s["interleaved"] else (r[..., :rotary // 2], r[..., rotary // 2:])
        a, b = a * c - b * sn, b * c + a * sn
        r = torch.stack([a, b], dim=-1).flatten(-2) if s["interleaved"] else torch.cat([a, b], dim=-1)
        out.append(torch.cat([r, x[..., rotary:]], dim=-1).to(dtype))
    return out


# ---- the cases -------------------------------------------------------------------

def _bytes(n):
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device=DEV)


def _cache(ctx, n, capacity, kv, d):
    import quantibbler_amd as qa

    return qa.KvCache(ctx, "fp4", n, capacity, kv, d, _bytes(qa.KvCache.size("fp4", n, capacity, kv, d)))


def _prepare_verify(s, case, seed):
    s["logits"], s["draft_logits"], s["ids"], s["uniforms"], s["temperature"] = _verify_inputs(case, seed)
    s["counts"] = _uint32(_counts(case))
    if own:
        from quantibbler_amd.gpu import verify_drafts_workspace_size

        n, k = case["seqs"], case["drafts"]
        s["tokens"] = torch.empty((n, k + 1), dtype=torch.int32, device=DEV)
        s["emitted"] = torch.empty(n, dtype=torch.int32, device=DEV)
        s["need"] = verify_drafts_workspace_size(n, k, case["vocab"], case["given"])
        s["ws"] = _bytes(s["need"])
    return s


def _prepare_rotate(s, case, seed):
    rows, at = _lengths(case), _first_rows(case)
    s["q"], s["k"], s["weights"] = _rotate_inputs(case, seed)
    s["n_rows"] = sum(rows)
    if own:
        from quantibbler_amd.gpu import Rope

        s["rope"] = Rope(case["d"], THETA, rotary_dim=case["rotary"], interleaved=case["interleaved"],
                         scaling=SCALINGS[case["scaling"]])
        s["at_dev"], s["row_start"] = _uint32(at), _uint32(_starts(rows))
        s["out"] = [torch.empty(x.shape, dtype=x.dtype, device=DEV) for x in (s["q"], s["k"])]
    else:
        s["positions"] = torch.cat([torch.arange(a, a + r, device=DEV) for a, r in zip(at, rows)])
    return s


def prepare(case, seed):
    s = dict(case, stream=torch.cuda.current_stream())
    ctx = None
    if own:
        import quantibbler_amd as qa

        ctx = s["ctx"] = qa.GpuContext(0)
    if case["kind"] == "verify":
        return _prepare_verify(s, case, seed)
    if case["kind"] == "rotate":
        return _prepare_rotate(s, case, seed)
    kv, d, n, lens = case["kv_heads"], case["d"], case["seqs"], _lengths(case)
    starts = _starts(lens)
    if case["kind"] == "cache":
        at = _first_rows(case)
        s["k"], s["v"] = _cache_inputs(case, seed)
        s["n_rows"] = starts[-1]
        if own:
            s["at_dev"], s["row_start"] = _uint32(at), _uint32(starts)
            s["cache"] = _cache(ctx, n, max(r + a for r, a in zip(lens, at)) + 1, kv, d)
            s["out"] = [torch.empty((s["n_rows"], kv, d), dtype=s["k"].dtype, device=DEV) for _ in range(2)]
        return s
    longest = case["longest"]
    s["q"], prefix, own_rows = _attend_inputs(case, seed)
    s["lens_dev"] = _uint32(lens)
    if own:
        s["cache"] = _cache(ctx, n, longest, kv, d)
        s["cache"].write_dev(*own_rows, "float32", _uint32([0] * n), starts[-1], row_start=_uint32(starts),
                             stream=s["stream"])
        s["shared"] = None
        if case["prefix"]:
            s["shared"] = _cache(ctx, 1, case["prefix"], kv, d)
            s["shared"].write_dev(*prefix, "float32", _uint32([0]), case["prefix"], stream=s["stream"])
        s["out"] = torch.empty_like(s["q"])
        s["need"] = s["cache"].attention_workspace_size(case["heads"], n, seq_q=case["queries"], max_len=longest,
                                                        prefix_len=case["prefix"])
        s["ws"] = _bytes(s["need"])
        return s
    s["prefix_rows"] = [_quantise(x) for x in prefix]
    s["own_rows"] = []
    for x in own_rows:
        codes, scales = _quantise(x)
        wide, wide_scales = torch.zeros((n, longest, kv, d), device=DEV), torch.zeros((n, longest, kv, 1), device=DEV)
        for i in range(n):
            wide[i, :lens[i]] = codes[starts[i]:starts[i + 1]]
            wide_scales[i, :lens[i]] = scales[starts[i]:starts[i + 1]]
        s["own_rows"].append((wide, wide_scales))
    return s


def run(s):
    kind = s["kind"]
    if kind == "verify":
        if not own:
            return _plain_verify(s)
        from quantibbler_amd.gpu import verify_drafts_dev

        verify_drafts_dev(s["ctx"], s["logits"], s["seqs"], s["drafts"], s["vocab"], s["ids"], s["uniforms"],
                          s["tokens"], s["emitted"], s["ws"], s["need"], draft_logits=s["draft_logits"],
                          n_drafts=s["counts"], temperature=s["temperature"], dtype=s["dtype"], stream=s["stream"])
        return {"tokens": s["tokens"], "counts": s["emitted"]}
    if kind == "rotate":
        if not own:
            return _plain_rotate(s)
        from quantibbler_amd.gpu import rotate_heads_dev

        rotate_heads_dev(s["ctx"], s["rope"], s["q"], s["k"], s["dtype"], s["n_rows"], s["heads"], s["kv_heads"],
                         s["at_dev"], *s["out"], n_seqs=s["seqs"], row_start=s["row_start"], before=s["before"],
                         q_norm=s["weights"][0], k_norm=s["weights"][1], eps=EPS, q_stride=s["q"].stride(0),
                         k_stride=s["k"].stride(0), stream=s["stream"])
        return s["out"]
    if kind == "attend":
        if not own:
            return _plain_attend(s)
        s["cache"].attention_dev(s["q"], s["dtype"], s["heads"], s["lens_dev"], s["out"], s["ws"], s["need"],
                                 seq_q=s["queries"], prefix=s["shared"], prefix_len=s["prefix"], stream=s["stream"])
        return s["out"]
    if not own:
        dtype = getattr(torch, s["dtype"])
        return [(codes * scales).to(dtype) for codes, scales in (_quantise(s["k"]), _quantise(s["v"]))]
    s["cache"].write_dev(s["k"], s["v"], s["dtype"], s["at_dev"], s["n_rows"], row_start=s["row_start"],
                         row_stride=s["k"].stride(0), stream=s["stream"])
    s["cache"].read_dev(*s["out"], s["dtype"], s["at_dev"], s["n_rows"], row_start=s["row_start"], stream=s["stream"])
    return s["out"]


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "verify":
        n, rows = case["seqs"], sum(c + 1 for c in _counts(case))
        if case["given"]:
            rows += rows - n
        return {"bytes": rows * case["vocab"] * e + n * (case["drafts"] + 1) * 12, "flops": 4 * rows * case["vocab"]}
    kv, d = case["kv_heads"], case["d"]
    if case["kind"] == "rotate":
        n = sum(_lengths(case)) * (case["heads"] + kv) * d
        return {"bytes": 2 * n * e, "flops": (4 if case["normed"] else 0) * n + 3 * n * case["rotary"] // d}
    held = d / 2 + -(-d // GROUP) + 4  # bytes of a row's head in the cache
    if case["kind"] == "cache":
        n = 2 * sum(_lengths(case)) * kv
        return {"bytes": int(2 * n * (d * e + held)), "flops": 4 * n * d}
    n, sq = case["seqs"], case["queries"]
    seen = sum(max(0, x - sq + t + 1) for x in _lengths(case) for t in range(sq)) + n * sq * case["prefix"]
    return {"bytes": int(2 * (sum(_lengths(case)) + case["prefix"]) * kv * held + 2 * n * sq * case["heads"] * d * e),
            "flops": 4 * d * case["heads"] * seen}


# ---- 64 bits ------------------------------------------------------------------------

def _nearest(x, steps):
    """The nearest of a format's values below the next power of two, the even one at a tie: steps a binade, and the
    exponent from which on they are finer no more."""
    bits, least = steps
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** least))) - bits)
    return torch.round(x / step) * step


def _stored(x):
    """The values a cache stands for, from the definition: scale, reciprocals and scaled inputs are f32 numbers, the
    multiplier the nearest e4m3, the code the nearest e2m1."""
    x = x.to(torch.float32)
    d = x.shape[-1]
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    top = x.abs().max(dim=-1, keepdim=True).values.clamp(min=FLOOR)
    per = torch.reciprocal(top)
    for c in range(0, d, GROUP):
        part = x[..., c:c + GROUP]
        mult = _nearest((part.abs().max(dim=-1, keepdim=True).values * (per * TOP)).double(), (3, -6)).clamp(max=TOP)
        by = torch.reciprocal(mult.clamp(min=2.0 ** -9).to(torch.float32))
        code = _nearest(((part * (per * (6.0 * TOP))) * by).double(), (1, 0)).clamp(-6.0, 6.0)
        out[..., c:c + GROUP] = code * mult
    return out * (top * (1.0 / (6.0 * TOP))).double()


def _exact_attend(case, seed):
    q, prefix, own_rows = _attend_inputs(case, seed)
    pk, pv = (_stored(x) for x in prefix)
    k, v = (_stored(x) for x in own_rows)
    n, sq, group, lens = case["seqs"], case["queries"], case["heads"] // case["kv_heads"], _lengths(case)
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    start = _starts(lens)
    for h in range(case["heads"]):
        j = h // group
        for b in range(n):
            keys = torch.cat([pk[:, j], k[start[b]:start[b + 1], j]])
            vals = torch.cat([pv[:, j], v[start[b]:start[b + 1], j]])
            if keys.shape[0] == 0:
                continue
            scores = torch.matmul(q[b, :, h].double(), keys.t().contiguous()) / math.sqrt(case["d"])
            last = case["prefix"] + lens[b] - sq + 1 + torch.arange(sq, device=DEV)[:, None]
            index = torch.arange(keys.shape[0], device=DEV)[None]
            seen = (index < case["prefix"]) | (index < last)
            w = torch.where(seen, scores, torch.full_like(scores, float("-inf"))).softmax(dim=-1)
            out[b, :, h] = torch.where(seen.any(dim=-1, keepdim=True), torch.matmul(w, vals), torch.zeros_like(vals[:1]))
    return out


def _exact_verify(case, seed):
    x, y, ids, u, temperature = _verify_inputs(case, seed)
    n, k, vocab = case["seqs"], case["drafts"], case["vocab"]
    tokens = torch.full((n, k + 1), -1, dtype=torch.int32, device=DEV)
    counts = torch.zeros(n, dtype=torch.int32, device=DEV)

    def chances(row, t):
        if t > 0:
            return (row.double() / t).softmax(dim=0)
        out = torch.zeros(vocab, dtype=torch.float64, device=DEV)
        out[int((row == row.max()).nonzero()[0, 0])] = 1.0
        return out

    for i, c in enumerate(_counts(case)):
        t = float(temperature[i])
        for j in range(c + 1):
            weights = p = chances(x[i, j], t)
            if j < c:
                d = int(ids[i, j])
                q = chances(y[i, j], t) if y is not None else torch.zeros_like(p)
                if y is None:
                    q[d] = 1.0
                if float(u[i, j]) * float(q[d]) < float(p[d]):
                    tokens[i, j] = d
                    continue
                weights = (p - q).clamp(min=0.0)
                weights = weights if float(weights.sum()) > 0 else p
            support = weights.nonzero()[:, 0]
            sums = torch.cumsum(weights[support], dim=0)
            at = int(torch.searchsorted(sums, float(u[i, c]) * sums[-1:], right=True)[0])
            tokens[i, j] = int(support[min(at, support.numel() - 1)])
            counts[i] = j + 1
            break
    return {"tokens": tokens, "counts": counts}


def _radians(rotary, scaling):
    """A position's angle for each pair, pair by pair, and the factor on cos and sin."""
    kind, by, size, theta, out = (scaling or {}).get("kind"), (scaling or {}).get("factor", 1.0), 1.0, THETA, []
    if kind == "base" and rotary > 2:
        theta *= by ** (rotary / (rotary - 2.0))
    if kind == "yarn":
        size += math.log(by) / 10.0
    for i in range(rotary // 2):
        w = 1.0 / theta ** (2.0 * i / rotary)
        slow = 0.0  # how much of the pair is slowed down by the factor
        if kind == "linear":
            slow = 1.0
        elif kind == "ramp":
            wavelength = 2.0 * math.pi / w
            slow = 1.0 - (scaling["original_len"] / wavelength - scaling["low"]) / (scaling["high"] - scaling["low"])
        elif kind == "yarn":  # a pair makes `turns` turns in the original context where theta^(2 i / rotary) is that
            edge = [math.log(scaling["original_len"] / (2.0 * math.pi * turns), theta) * rotary / 2.0
                    for turns in (scaling["high"], scaling["low"])]
            first, last = max(0, math.floor(edge[0])), min(rotary - 1, math.ceil(edge[1]))
            slow = (i - first) / max(last - first, 0.001)
        slow = min(1.0, max(0.0, slow))
        out.append(w * (1.0 - slow) + w * slow / by)
    return torch.tensor(out, dtype=torch.float64, device=DEV), size


def _exact_rotate(case, seed):
    q, k, weights = _rotate_inputs(case, seed)
    rotary, rows, at = case["rotary"], _lengths(case), _first_rows(case)
    f, size = _radians(rotary, SCALINGS[case["scaling"]])
    place = torch.cat([torch.arange(r, device=DEV) + a for r, a in zip(rows, at)]) + case["before"]
    turn = torch.polar(torch.full((), size, dtype=torch.float64, device=DEV), torch.outer(place.double(), f))[:, None]
    out = []
    for x, w in zip((q, k), weights):
        x = x.double()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * w.double()
        first = slice(0, rotary, 2) if case["interleaved"] else slice(0, rotary // 2)
        second = slice(1, rotary, 2) if case["interleaved"] else slice(rotary // 2, rotary)
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return out


def exact(case, seed):
    if case["kind"] == "verify":
        return _exact_verify(case, seed)
    if case["kind"] == "rotate":
        return _exact_rotate(case, seed)
    if case["kind"] == "cache":
        return [_stored(x) for x in _cache_inputs(case, seed)]
    return _exact_attend(case, seed)
