"""The 8-bit KV cache, the attention that reads it and the log probabilities of
a serving step, as timed cases.

``own`` false computes each operator in its plain form, elementary torch
operations in 32 bits; ``own`` true makes the calls of a program built on this
library: ``KvCache.write_dev``, ``read_dev`` and ``attention_dev`` and
``logprobs_dev``.  Heads and widths are those of the repository's 4096-wide
block (32 query heads, 8 kv heads of 128 channels, a 128256-row vocabulary) or
generic; inputs are made from the seed alone.
"""
import math
import random

import torch

own = False

DEV = "cuda"
LEVELS = {"int8": 127.0, "fp8": 448.0}
FLOOR = 2.0 ** -100


def listed():
    return [
        # one token of one sequence written into its cache and read back: the smallest call, its latency counts
        {"name": "cache-token", "kind": "cache", "format": "int8", "dtype": "float32", "kv_heads": 8, "d": 128,
         "seqs": 1, "longest": 1, "mix": 0, "at": 2085, "fused": False},
        # a batched decode step's rows, taken out of the fused q/k/v rows of 32 sequences
        {"name": "cache-step", "kind": "cache", "format": "fp8", "dtype": "bfloat16", "kv_heads": 8, "d": 128,
         "seqs": 32, "longest": 1, "mix": 0, "at": 2085, "fused": True},
        # prompts of unlike length written in one call, some of them chunks that continue one; a ragged head dim
        {"name": "cache-prompts", "kind": "cache", "format": "int8", "dtype": "float32", "kv_heads": 5, "d": 80,
         "seqs": 6, "longest": 1201, "mix": 3, "at": 450, "fused": False},
        # four long sequences read back whole (moved to another program, or checked)
        {"name": "cache-read", "kind": "read", "format": "int8", "dtype": "bfloat16", "kv_heads": 8, "d": 128,
         "seqs": 4, "longest": 4096, "mix": 0, "at": 0},
        # one sequence's decode step without a prefix: latency
        {"name": "attend-token", "kind": "attend", "format": "int8", "dtype": "float32", "heads": 32, "kv_heads": 8,
         "d": 128, "seqs": 1, "longest": 700, "mix": 0, "queries": 1, "prefix": 0},
        # a batched decode step of 32 sequences of unlike length, no prefix
        {"name": "attend-step", "kind": "attend", "format": "int8", "dtype": "bfloat16", "heads": 32, "kv_heads": 8,
         "d": 128, "seqs": 32, "longest": 2085, "mix": 0, "queries": 1, "prefix": 0},
        # 32 requests behind one system prompt of 8192 tokens
        {"name": "prefix-step", "kind": "attend", "format": "int8", "dtype": "bfloat16", "heads": 32, "kv_heads": 8,
         "d": 128, "seqs": 32, "longest": 512, "mix": 0, "queries": 1, "prefix": 8192},
        # five drafted tokens of each of 16 requests checked at once, f32 queries, one query head a kv head
        {"name": "prefix-draft", "kind": "attend", "format": "fp8", "dtype": "float32", "heads": 8, "kv_heads": 8,
         "d": 80, "seqs": 16, "longest": 290, "mix": 5, "queries": 5, "prefix": 4001},
        # 64 requests behind a long document, the largest attention
        {"name": "prefix-wide", "kind": "attend", "format": "int8", "dtype": "bfloat16", "heads": 32, "kv_heads": 8,
         "d": 128, "seqs": 64, "longest": 2048, "mix": 0, "queries": 1, "prefix": 16384},
        # one decoded token's log probability, with the twenty likeliest beside it
        {"name": "score-token", "kind": "score", "dtype": "float32", "rows": 1, "vocab": 128256, "top": 20,
         "masked": False},
        # a batched step's, over a vocabulary of odd size in bf16, some of it forbidden
        {"name": "score-step", "kind": "score", "dtype": "bfloat16", "rows": 32, "vocab": 32003, "top": 5,
         "masked": True},
        # every token of a 2048-token prompt scored (the largest: 1 GB of logits)
        {"name": "score-prompt", "kind": "score", "dtype": "float32", "rows": 2048, "vocab": 128256, "top": 1,
         "masked": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "cache", "read", "attend", "attend", "attend", "attend", "score", "score"])
    fmt, dtype = rng.choice(["int8", "fp8"]), rng.choice(["float32", "bfloat16"])
    kv = rng.choice([1, 2, 5, 8])
    d = rng.choice([16, 64, 80, 128, 128, 256])
    n, mix = _log(rng, 1, 64), rng.choice([0, rng.randint(1, 1 << 20), rng.randint(1, 1 << 20)])
    if kind in ("cache", "read"):
        case = {"kind": kind, "format": fmt, "dtype": dtype, "kv_heads": kv, "d": d, "seqs": n,
                "longest": _log(rng, 1, max(1, 8192 // n)), "mix": mix,
                "at": 0 if kind == "read" else rng.randint(0, 1000)}
        if kind == "cache":
            case["fused"] = rng.random() < 0.4
        return case
    if kind == "attend":
        group, queries = rng.choice([1, 2, 4, 7]), rng.choice([1, 1, 1, 2, 5, 16])
        prefix = rng.choice([0, _log(rng, 1, 16384), _log(rng, 64, 16384)])
        keys = int(1.8e10 / (4 * d * kv * group * queries * n))  # no more products than the largest listed case has
        prefix = min(prefix, keys)
        return {"kind": kind, "format": fmt, "dtype": dtype, "heads": kv * group, "kv_heads": kv, "d": d, "seqs": n,
                "longest": _log(rng, 1, max(1, min(2048, keys - prefix))), "mix": mix, "queries": queries,
                "prefix": prefix}
    vocab = _log(rng, 2, 200000)
    rows = min(_log(rng, 1, 2048), max(1, 2048 * 128256 // vocab))
    return {"kind": kind, "dtype": dtype, "rows": rows, "vocab": vocab,
            "top": min(vocab, rng.choice([0, 1, 5, 20, 32])), "masked": rng.random() < 0.4}


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
    """The position that each sequence's rows are written at."""
    n, at = case["seqs"], case["at"]
    return [at - (i * at) // n for i in range(n)]


def _normal(seed, tag, shape, dtype=torch.float32):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + int(tag))
    return torch.randn(shape, device=DEV, generator=g, dtype=dtype)


def _uint32(values):
    return torch.tensor([int(v) for v in values], dtype=torch.int32, device=DEV)


def _kv_rows(seed, tag, n, kv, d, dtype):
    """Keys with a channel mean, as trained models have, and values of unlike size by token."""
    k = _normal(seed, tag, (n, kv, d)) + 2.0 * _normal(seed, 90, (1, kv, d))
    v = _normal(seed, tag + 1, (n, kv, d)) * torch.exp(0.5 * _normal(seed, tag + 2, (n, kv, 1)))
    return k.to(dtype), v.to(dtype)


def _starts(rows):
    out = [0]
    for r in rows:
        out.append(out[-1] + r)
    return out


def _attend_inputs(case, seed):
    """q [n][queries][heads][d]; the prefix's and every sequence's key and value rows [.][kv_heads][d], f32."""
    n, dtype = case["seqs"], getattr(torch, case["dtype"])
    q = (1.5 * _normal(seed, 1, (n, case["queries"], case["heads"], case["d"]))).to(dtype)
    own_rows = _kv_rows(seed, 10, sum(_lengths(case)), case["kv_heads"], case["d"], torch.float32)
    return q, _kv_rows(seed, 20, case["prefix"], case["kv_heads"], case["d"], torch.float32), own_rows


def _score_inputs(case, seed):
    rows, vocab = case["rows"], case["vocab"]
    x = _normal(seed, 1, (rows, vocab)).mul_(2.5)
    x.add_(_normal(seed, 2, (rows, 1)))
    if case["masked"]:  # a grammar's or a sampler's forbidden tokens
        forbidden = _normal(seed, 3, (1, vocab)) > 1.0
        forbidden[0, 0] = False
        x.masked_fill_(forbidden, float("-inf"))
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 4)
    targets = torch.randint(0, vocab, (rows,), device=DEV, generator=g, dtype=torch.int32)
    return x.to(getattr(torch, case["dtype"])), targets


# ---- the plain forms -----------------------------------------------------------

def _quantise(x, fmt):
    """Rows [.][kv_heads][d] -> codes and one f32 scale a row and head."""
    x = x.float()
    levels = LEVELS[fmt]
    top = x.abs().amax(dim=-1, keepdim=True)
    whole = torch.isfinite(top)
    top = torch.where(whole, top, torch.ones_like(top)).clamp_min(FLOOR)
    codes = torch.where(whole, x * (levels / top), torch.zeros_like(x))
    codes = torch.round(codes).to(torch.int8) if fmt == "int8" else codes.to(torch.float8_e4m3fn)
    return codes, torch.where(whole, top / levels, torch.full_like(top, float("nan")))


def _values(codes, scales):
    return codes.float() * scales


def _plain_attend(s):
    n, sq, heads, kv, d = s["seqs"], s["queries"], s["heads"], s["kv_heads"], s["d"]
    group, dtype = heads // kv, s["q"].dtype
    q = s["q"].float().view(n, sq, kv, group, d).permute(2, 0, 1, 3, 4).contiguous()  # [kv][n][sq][group][d]
    pk, pv = (_values(*x).permute(1, 0, 2).contiguous() for x in s["prefix_rows"])    # [kv][prefix][d]
    ok, ov = (_values(*x) for x in s["own_rows"])                                     # [n][longest][kv][d]
    ok, ov = ok.permute(2, 0, 1, 3).contiguous(), ov.permute(2, 0, 1, 3).contiguous()
    longest, prefix = ok.shape[2], pk.shape[1]
    rows = sq * group
    scale = 1.0 / math.sqrt(d)
    sp = torch.matmul(q.view(kv, n * rows, d), pk.transpose(1, 2).contiguous()).view(kv, n, rows, prefix)
    so = torch.matmul(q.view(kv, n, rows, d), ok.transpose(2, 3).contiguous())        # [kv][n][rows][longest]
    limit = (s["lens_dev"].view(n, 1) - sq + 1 + torch.arange(sq, device=DEV).view(1, sq))  # own rows a query sees
    seen = torch.arange(longest, device=DEV).view(1, 1, longest) < limit.view(n, sq, 1)
    seen = seen.view(n, sq, 1, longest).expand(n, sq, group, longest).reshape(n, rows, longest)
    scores = torch.cat([sp, so.masked_fill(~seen, float("-inf"))], dim=-1) * scale
    top = scores.amax(dim=-1, keepdim=True) if scores.shape[-1] else scores.new_zeros(kv, n, rows, 1)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p[..., :prefix].reshape(kv, n * rows, prefix), pv).view(kv, n, rows, d)
    out = out + torch.matmul(p[..., prefix:].contiguous(), ov)
    out = torch.where(total > 0, out / total, torch.where(total == 0, torch.zeros_like(out), out * total))
    return out.view(kv, n, sq, group, d).permute(1, 2, 0, 3, 4).reshape(n, sq, heads, d).to(dtype)


def _order(x):
    """int64 keys that sort as (value, lowest index first), NaN as -inf; all differ."""
    x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x) + 0.0
    bits = x.view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    return bits * (1 << 32) + (x.shape[-1] - 1 - torch.arange(x.shape[-1], device=DEV))


def _plain_score(s):
    logp, entropy, ids, tops = [], [], [], []
    step = max(1, (1 << 28) // s["vocab"])
    for r in range(0, s["rows"], step):
        x = s["logits"][r:r + step].float()
        top = x.amax(dim=-1, keepdim=True)
        e = torch.exp(x - top)
        total = e.sum(dim=-1, keepdim=True)
        lse = torch.log(total)
        shifted = x - top
        t = s["targets"][r:r + step].long().view(-1, 1)
        logp.append((shifted.gather(1, t) - lse)[:, 0])
        inner = torch.where(e > 0, e * shifted, torch.where(torch.isnan(e), e, torch.zeros_like(e)))
        entropy.append((lse - inner.sum(dim=-1, keepdim=True) / total)[:, 0])
        if s["top"]:
            i = torch.topk(_order(x), s["top"], dim=-1, sorted=True).indices
            ids.append(i.to(torch.int32))
            tops.append(shifted.gather(1, i) - lse)
    out = {"logprobs": torch.cat(logp), "entropy": torch.cat(entropy)}
    if s["top"]:
        out["top_ids"], out["top_logprobs"] = torch.cat(ids), torch.cat(tops)
    return out


# ---- the cases -------------------------------------------------------------------

def _bytes(n):
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device=DEV)


def _cache(ctx, fmt, n, capacity, kv, d):
    import quantibbler_amd as qa

    return qa.KvCache(ctx, fmt, n, capacity, kv, d, _bytes(qa.KvCache.size(fmt, n, capacity, kv, d)))


def _cache_inputs(case, seed):
    kv, d, n = case["kv_heads"], case["d"], sum(_lengths(case))
    dtype = getattr(torch, case["dtype"])
    k, v = _kv_rows(seed, 10, n, kv, d, dtype)
    if not case.get("fused"):
        return k, v
    rows = torch.zeros((n, 4 * kv * d + 2 * kv * d), dtype=dtype, device=DEV)  # q | k | v of a projection's rows
    rows[:, 4 * kv * d:5 * kv * d] = k.view(n, kv * d)
    rows[:, 5 * kv * d:] = v.view(n, kv * d)
    return rows[:, 4 * kv * d:5 * kv * d].view(n, kv, d), rows[:, 5 * kv * d:].view(n, kv, d)


def prepare(case, seed):
    s = dict(case, stream=torch.cuda.current_stream())
    ctx = None
    if own:
        import quantibbler_amd as qa

        ctx = s["ctx"] = qa.GpuContext(0)
    if case["kind"] == "score":
        s["logits"], s["targets"] = _score_inputs(case, seed)
        if own:
            from quantibbler_amd.gpu import logprobs_workspace_size

            rows, k = case["rows"], case["top"]
            s["logprobs"], s["entropy"] = (torch.empty(rows, device=DEV) for _ in range(2))
            s["top_ids"] = torch.empty((rows, k), dtype=torch.int32, device=DEV) if k else None
            s["top_logprobs"] = torch.empty((rows, k), device=DEV) if k else None
            s["need"] = logprobs_workspace_size(rows, case["vocab"], k)
            s["ws"] = _bytes(s["need"])
        return s
    fmt, kv, d = case["format"], case["kv_heads"], case["d"]
    if case["kind"] in ("cache", "read"):
        n, rows, at = case["seqs"], _lengths(case), _first_rows(case)
        s["k"], s["v"] = _cache_inputs(case, seed)
        s["n_rows"] = sum(rows)
        s["at_dev"], s["row_start"] = _uint32(at), _uint32(_starts(rows))
        if own:
            s["cache"] = _cache(ctx, fmt, n, max(r + a for r, a in zip(rows, at)) + 1, kv, d)
            s["out"] = [torch.empty((s["n_rows"], kv, d), dtype=s["k"].dtype, device=DEV) for _ in range(2)]
            if case["kind"] == "read":
                s["cache"].write_dev(s["k"], s["v"], case["dtype"], s["at_dev"], s["n_rows"],
                                     row_start=s["row_start"], stream=s["stream"])
                del s["k"], s["v"]
        elif case["kind"] == "read":
            s["codes"] = _quantise(s.pop("k"), fmt), _quantise(s.pop("v"), fmt)
        return s
    n, longest, lens = case["seqs"], case["longest"], _lengths(case)
    s["q"], prefix, own_rows = _attend_inputs(case, seed)
    s["lens_dev"] = _uint32(lens)
    starts = _starts(lens)
    if own:
        s["cache"] = _cache(ctx, fmt, n, longest, kv, d)
        s["cache"].write_dev(*own_rows, "float32", _uint32([0] * n), starts[-1], row_start=_uint32(starts),
                             stream=s["stream"])
        s["shared"] = None
        if case["prefix"]:
            s["shared"] = _cache(ctx, fmt, 1, case["prefix"], kv, d)
            s["shared"].write_dev(*prefix, "float32", _uint32([0]), case["prefix"], stream=s["stream"])
        s["out"] = torch.empty_like(s["q"])
        s["need"] = s["cache"].attention_workspace_size(case["heads"], n, seq_q=case["queries"], max_len=longest,
                                                        prefix_len=case["prefix"])
        s["ws"] = _bytes(s["need"])
        return s
    s["prefix_rows"] = [_quantise(x, fmt) for x in prefix]
    s["own_rows"] = []
    for x in own_rows:
        codes, scales = _quantise(x, fmt)
        wide = torch.zeros((n, longest, kv, d), dtype=codes.dtype, device=DEV)
        wide_scales = torch.zeros((n, longest, kv, 1), device=DEV)
        for i in range(n):
            wide[i, :lens[i]] = codes[starts[i]:starts[i + 1]]
            wide_scales[i, :lens[i]] = scales[starts[i]:starts[i + 1]]
        s["own_rows"].append((wide, wide_scales))
    return s


def run(s):
    kind = s["kind"]
    if kind == "score":
        if not own:
            return _plain_score(s)
        from quantibbler_amd.gpu import logprobs_dev

        logprobs_dev(s["ctx"], s["logits"], s["rows"], s["vocab"], s["targets"], s["logprobs"], s["entropy"],
                     s["ws"], s["need"], top_k=s["top"], top_ids=s["top_ids"], top_logprobs=s["top_logprobs"],
                     dtype=s["dtype"], stream=s["stream"])
        out = {"logprobs": s["logprobs"], "entropy": s["entropy"]}
        if s["top"]:
            out["top_ids"], out["top_logprobs"] = s["top_ids"], s["top_logprobs"]
        return out
    if kind == "attend":
        if not own:
            return _plain_attend(s)
        s["cache"].attention_dev(s["q"], s["dtype"], s["heads"], s["lens_dev"], s["out"], s["ws"], s["need"],
                                 seq_q=s["queries"], prefix=s["shared"], prefix_len=s["prefix"], stream=s["stream"])
        return s["out"]
    dtype = getattr(torch, s["dtype"])
    if not own:
        pairs = s["codes"] if kind == "read" else (_quantise(s["k"], s["format"]), _quantise(s["v"], s["format"]))
        return [_values(*p).to(dtype) for p in pairs]
    if kind == "cache":
        s["cache"].write_dev(s["k"], s["v"], s["dtype"], s["at_dev"], s["n_rows"], row_start=s["row_start"],
                             row_stride=s["k"].stride(0), stream=s["stream"])
    s["cache"].read_dev(*s["out"], s["dtype"], s["at_dev"], s["n_rows"], row_start=s["row_start"], stream=s["stream"])
    return s["out"]


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * n}
    kv, d = case["kv_heads"], case["d"]
    if case["kind"] in ("cache", "read"):
        n = 2 * sum(_lengths(case)) * kv
        once = n * (d * e + d + 4)
        return {"bytes": once * (2 if case["kind"] == "cache" else 1), "flops": 2 * n * d}
    n, sq = case["seqs"], case["queries"]
    seen = sum(max(0, x - sq + t + 1) for x in _lengths(case) for t in range(sq)) + n * sq * case["prefix"]
    return {"bytes": 2 * (sum(_lengths(case)) + case["prefix"]) * kv * (d + 4) + 2 * n * sq * case["heads"] * d * e,
            "flops": 4 * d * case["heads"] * seen}


# ---- 64 bits ------------------------------------------------------------------------

def _stored(x, fmt):
    """The values a cache stands for, from the definition: the scale and the scaled input are f32 numbers, the code the
    nearest of its kind, even at a tie."""
    x = x.to(torch.float32)
    top = x.abs().max(dim=-1, keepdim=True).values.clamp(min=FLOOR)
    scaled = (x * (LEVELS[fmt] / top)).double()
    step = torch.ones_like(scaled)
    if fmt == "fp8":  # three bits behind the leading one, none below 2^-9
        step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(scaled / step) * step * (top / LEVELS[fmt]).double()


def exact(case, seed):
    if case["kind"] == "score":
        x, targets = _score_inputs(case, seed)
        parts = {"logprobs": [], "entropy": [], "top_ids": [], "top_logprobs": []}
        step = max(1, (1 << 25) // case["vocab"])
        for r in range(0, case["rows"], step):
            lp = torch.log_softmax(x[r:r + step].double(), dim=-1)
            parts["logprobs"].append(lp.gather(1, targets[r:r + step].long()[:, None])[:, 0])
            parts["entropy"].append(-torch.nan_to_num(lp.exp() * lp, nan=0.0).sum(dim=-1))
            if case["top"]:
                value, index = torch.sort(lp, dim=-1, descending=True, stable=True)
                parts["top_ids"].append(index[:, :case["top"]].to(torch.int32))
                parts["top_logprobs"].append(value[:, :case["top"]])
        return {name: torch.cat(p) for name, p in parts.items() if p}
    if case["kind"] in ("cache", "read"):
        return [_stored(x, case["format"]) for x in _cache_inputs(case, seed)]
    q, prefix, own_rows = _attend_inputs(case, seed)
    pk, pv = (_stored(x, case["format"]) for x in prefix)
    k, v = (_stored(x, case["format"]) for x in own_rows)
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
