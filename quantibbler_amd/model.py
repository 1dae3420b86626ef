"""Model directory reader: the host half of the reference's directory load
(crates/quantibbler-qpk1/src/loader.rs:172-320 `load`, composed by
crates/quantibbler-server/src/model/mod.rs:582-597 and
engine/mod.rs:639-760 `ModelWeights::from_layers`), for the files a
quantized model directory holds:

* ``config.toml`` -- geometry (vocab_size, d_model, n_layers, n_heads,
  n_kv_heads, head_dim, rms_norm_eps, rope_theta), the norm inventory
  ``norm_slots`` and ``weight_tying``;
* ``manifest.toml`` -- the layer names, ``[layer_files]`` (name -> qpk1 path)
  and ``[sidecar]`` (embedding, lm_head, norms, optional dtype f32|bf16);
* the qpk1 layer streams (parsed and uploaded by ``qbk_factor_from_qpk1``)
  and the raw little-endian remainder tensors.

The norm sidecar is laid out by inventory (engine/mod.rs:517-560
BlockRefs::resolve): per block, the declared slots in order -- ``input``,
``post_attention``, ``post_feedforward`` are d_model floats, ``q_norm`` and
``k_norm`` head_dim floats -- then the final norm's d_model floats.

Only what the fixtures and the hot path use is read; the blob format and the
reference's long list of directory refusals are out of scope.  Errors raise
``ModelError`` naming the file.
"""
from __future__ import annotations

import ast
import os
import re
from dataclasses import dataclass, field

import numpy as np

from ._lib import KernelError


class ModelError(ValueError):
    """A model directory that cannot be read (the reference's load error)."""


def read_toml(path: str) -> dict:
    """The TOML subset the reference's model files use: comments, [tables],
    bare or double-quoted keys, strings, numbers, booleans and (multi-line)
    arrays of those."""
    out: dict = {}
    table = out
    pending = ""
    try:
        with open(path, encoding="utf-8") as f:
            lines = f.read().splitlines()
    except OSError as e:
        raise ModelError(f"{path}: {e}") from None
    for raw in lines:
        line = _strip_comment(raw).strip()
        if not line and not pending:
            continue
        if pending:
            pending += " " + line
            if pending.count("[") > pending.count("]"):
                continue
            line, pending = pending, ""
        m = re.fullmatch(r"\[\s*([A-Za-z0-9_.\-]+)\s*\]", line)
        if m:
            table = out.setdefault(m.group(1), {})
            continue
        m = re.fullmatch(r'("(?:[^"\\]|\\.)*"|[A-Za-z0-9_\-]+)\s*=\s*(.*)', line)
        if not m:
            raise ModelError(f"{path}: cannot read line {raw!r}")
        key, val = m.group(1), m.group(2)
        if val.count("[") > val.count("]"):
            pending = line
            continue
        if key.startswith('"'):
            key = ast.literal_eval(key)
        table[key] = _value(path, val)
    if pending:
        raise ModelError(f"{path}: unterminated array")
    return out


def _strip_comment(line: str) -> str:
    in_str = False
    for i, ch in enumerate(line):
        if ch == '"' and (i == 0 or line[i - 1] != "\\"):
            in_str = not in_str
        elif ch == "#" and not in_str:
            return line[:i]
    return line


def _value(path, text):
    t = text.strip()
    if t in ("true", "false"):
        return t == "true"
    try:
        return ast.literal_eval(t)
    except (ValueError, SyntaxError):
        raise ModelError(f"{path}: cannot read value {text!r}") from None


_SLOT_WIDTH = {"input": "d", "post_attention": "d", "post_feedforward": "d", "q_norm": "h", "k_norm": "h"}
_DTYPES = {"f32": np.float32, "bf16": np.uint16}


def _remainder(path: str, n: int, dtype: str) -> np.ndarray:
    """A raw little-endian remainder tensor of n values at the declared dtype,
    widened to f32 (bf16 widens exactly)."""
    try:
        raw = np.fromfile(path, dtype="<u2" if dtype == "bf16" else "<f4")
    except OSError as e:
        raise ModelError(f"{path}: {e}") from None
    if raw.size != n:
        raise ModelError(f"{path}: holds {raw.size} {dtype} values; expected {n}")
    if dtype == "bf16":
        return (raw.astype(np.uint32) << 16).view(np.float32)
    return raw.astype(np.float32)


@dataclass
class ModelDir:
    """A model directory read into host memory (f32 remainder tensors, qpk1
    streams by layer name)."""
    path: str
    vocab_size: int
    d_model: int
    n_layers: int
    n_heads: int
    n_kv_heads: int
    head_dim: int
    rms_norm_eps: float
    rope_theta: float
    norm_slots: list
    remainder_dtype: str
    layer_names: list
    streams: dict = field(repr=False)
    embedding: np.ndarray = field(repr=False)
    lm_head: np.ndarray | None = field(repr=False)
    norms: np.ndarray = field(repr=False)

    @classmethod
    def load(cls, path: str) -> "ModelDir":
        cfg = read_toml(os.path.join(path, "config.toml"))
        man = read_toml(os.path.join(path, "manifest.toml"))
        need = ["vocab_size", "d_model", "n_layers", "n_heads", "n_kv_heads", "head_dim",
                "rms_norm_eps", "rope_theta", "norm_slots"]
        for k in need:
            if k not in cfg:
                raise ModelError(f"{path}/config.toml: missing {k}")
        slots = list(cfg["norm_slots"])
        for s in slots:
            if s not in _SLOT_WIDTH:
                raise ModelError(f"{path}/config.toml: unknown norm slot {s!r}")
        side = man.get("sidecar", {})
        dtype = side.get("dtype", "f32")
        if dtype not in _DTYPES:
            raise ModelError(f"{path}/manifest.toml: unknown sidecar dtype {dtype!r}")
        d, h, v, n = int(cfg["d_model"]), int(cfg["head_dim"]), int(cfg["vocab_size"]), int(cfg["n_layers"])
        per_block = sum(d if _SLOT_WIDTH[s] == "d" else h for s in slots)
        files = man.get("layer_files", {})
        names = list(man.get("layers", []))
        streams = {}
        for name in names:
            if name not in files:
                raise ModelError(f"{path}/manifest.toml: layer {name!r} has no [layer_files] entry")
            fp = os.path.join(path, files[name])
            try:
                with open(fp, "rb") as f:
                    streams[name] = f.read()
            except OSError as e:
                raise ModelError(f"{fp}: {e}") from None
        emb = _remainder(os.path.join(path, side.get("embedding", "e1.f32.bin")), v * d, dtype)
        head = None
        if "lm_head" in side and side["lm_head"] != side.get("embedding"):
            head = _remainder(os.path.join(path, side["lm_head"]), v * d, dtype)
        norms = _remainder(os.path.join(path, side.get("norms", "norms.f32.bin")), per_block * n + d, dtype)
        return cls(path=path, vocab_size=v, d_model=d, n_layers=n, n_heads=int(cfg["n_heads"]),
                   n_kv_heads=int(cfg["n_kv_heads"]), head_dim=h, rms_norm_eps=float(cfg["rms_norm_eps"]),
                   rope_theta=float(cfg["rope_theta"]), norm_slots=slots, remainder_dtype=dtype,
                   layer_names=names, streams=streams, embedding=emb.reshape(v, d),
                   lm_head=None if head is None else head.reshape(v, d), norms=norms)

    def head_rows(self) -> np.ndarray:
        """The lm_head rows, or the embedding when tied (engine/mod.rs:788)."""
        return self.embedding if self.lm_head is None else self.lm_head

    def block_norms(self, b: int) -> dict:
        """Block b's norm weights by slot name (engine/mod.rs:517-560)."""
        d, h = self.d_model, self.head_dim
        per_block = sum(d if _SLOT_WIDTH[s] == "d" else h for s in self.norm_slots)
        at = b * per_block
        out = {}
        for s in self.norm_slots:
            w = d if _SLOT_WIDTH[s] == "d" else h
            out[s] = self.norms[at:at + w]
            at += w
        return out

    def final_norm(self) -> np.ndarray:
        return self.norms[-self.d_model:]

    def block_layers(self, b: int) -> list:
        """Block b's seven qpk1 streams in the order q, k, v, o, gate, up,
        down (engine/mod.rs:517-531: names layers.{b}.inner.*)."""
        out = []
        for suffix in ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj",
                       "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj"):
            name = f"layers.{b}.inner.{suffix}"
            if name not in self.streams:
                raise ModelError(f"block {b}: missing packed layer {name!r}")
            out.append(self.streams[name])
        return out


def _bf16_values(a) -> np.ndarray:
    """f32 values rounded to their bf16 values (round to nearest even; NaN
    kept), as engine/mod.rs:695-706 holds the remainder tensors under bf16
    serving."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    nan = (u & 0x7FFFFFFF) > 0x7F800000
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint32)
    r = np.where(nan, (u >> 16) | 0x40, r).astype(np.uint32)
    return (r << 16).view(np.float32)


def _memory_of(stream):
    """torch's allocations within come from the pool of ``stream`` (as the
    device calls take it): no other stream's work is still using them, and
    once freed they go to work that this stream runs later."""
    import torch

    if not stream:
        stream = torch.cuda.default_stream()
    elif not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(stream if isinstance(stream, int) else stream.cuda_stream)
    return torch.cuda.stream(stream)


class DeviceModel:
    """The transformer trunk on the device at bf16 serving (Engine::forward,
    engine/mod.rs:802-806, and forward_prefill's per-token loop, :811-822):
    embedding row -> every DecoderBlock over its KV cache -> final norm ->
    lm_head logits, all device-resident.  ``attention`` picks every block's
    face once, as the engine does at load (engine/mod.rs:953-968): "sage"
    (the sage decode attention; prefill on the block-scaled SageAttention)
    or "exact" (f32 attention over the cache, one sequence, prefill token by
    token).  ``serving`` is the engine's serving dtype: "bf16" (remainder
    tensors rounded to bf16, the GEMV / GEMM projections) or "fp32" (the
    tensors as stored, apply's f64 products, f32 norms; one sequence, prefill
    token by token).  Built from a ModelDir; torch supplies the device
    buffers (plumbing only -- every step runs in libqbk)."""

    def __init__(self, ctx, md: ModelDir, capacity: int, block_size: int = 64, n_seqs: int = 1,
                 attention: str = "sage", serving: str = "bf16"):
        import torch

        from .gpu import DecoderBlock, FactorLayer, LmHead

        self.ctx, self.md, self.capacity, self.n_seqs = ctx, md, int(capacity), int(n_seqs)
        if serving not in ("bf16", "fp32"):
            raise ValueError(f"serving must be 'bf16' or 'fp32', got {serving!r}")
        self.serving = serving
        # bf16 serving rounds the remainder tensors to bf16 (engine/mod.rs:695-706)
        rnd = _bf16_values if serving == "bf16" else (lambda a: np.ascontiguousarray(a, np.float32))
        dev = torch.device("cuda")
        self.layers, self.blocks = [], []
        for b in range(md.n_layers):
            layers = [FactorLayer.from_qpk1(ctx, s) for s in md.block_layers(b)]
            self.layers.append(layers)
            norms = {k: rnd(v) for k, v in md.block_norms(b).items()}
            self.blocks.append(DecoderBlock(ctx, layers, norms["input"], norms["post_attention"], md.n_heads,
                                            md.n_kv_heads, md.head_dim, md.rope_theta, md.rms_norm_eps,
                                            capacity, block_size, norms.get("q_norm"), norms.get("k_norm"),
                                            n_seqs=self.n_seqs))
            self.blocks[-1].set_attention_face(attention)
            if serving == "fp32":
                self.blocks[-1].set_serving("fp32")
        self.attention = attention
        self.embedding = torch.from_numpy(rnd(md.embedding)).to(dev)
        self.final_norm = torch.from_numpy(rnd(md.final_norm())).to(dev)
        self.head = LmHead.from_rows(ctx, rnd(md.head_rows()))
        self.h = torch.empty(md.d_model, dtype=torch.float32, device=dev)
        self.hn = torch.empty(md.d_model, dtype=torch.float32, device=dev)
        self.logits = torch.empty(md.vocab_size, dtype=torch.float32, device=dev)
        self.pos = 0                        # sequence 0's, the one step() serves
        self.positions = [0] * self.n_seqs  # every sequence's
        self._shared = None                 # share_prefix's caches and buffers
        self._batch = {}                    # n -> (h, hn, logits, workspace) of step_batch

    def reset(self):
        for b in self.blocks:
            b.reset()
        self.pos = 0
        self.positions = [0] * self.n_seqs
        self._wait_shared()
        self._shared = None

    def _wait_shared(self):
        """Steps behind a shared prefix, on whatever stream, are through with its memory."""
        import torch

        if self._shared is not None:
            torch.cuda.synchronize()

    def prefill(self, tokens, stream=None, seq: int = 0):
        """forward_prefill (engine/mod.rs:811-822) of a new sequence (held as
        sequence ``seq``) in one pass per block: the tokens' embedding rows
        through every block's prefill (batched projections, causal
        block-scaled SageAttention), then the final norm and logits of the
        last position -- the logits a token-at-a-time prefill ends with.
        Returns them (a device tensor, overwritten by the next call);
        decoding continues with step() (sequence 0) or step_batch()."""
        from .gpu import rms_norm_dev

        md = self.md
        h, n, _ = self._prefill_rows(tokens, stream, seq)
        rms_norm_dev(self.ctx, h[n - 1], 1, md.d_model, self.final_norm, md.rms_norm_eps, self.hn, stream,
                     self.serving)
        self.head.logits_dev(self.hn, 1, self.logits, stream)
        return self.logits

    def _prefill_rows(self, tokens, stream, seq):
        """A new sequence's tokens through every block: the rows that leave
        the last one, their number, and the workspace (kept while it is read)."""
        import torch

        from .gpu import embed

        md = self.md
        ids = [int(t) for t in tokens]
        n = len(ids)
        need = max(b.prefill_workspace_size(n) for b in self.blocks)
        with _memory_of(stream):
            h = torch.empty((n, md.d_model), dtype=torch.float32, device="cuda")
            ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        embed(self.ctx, self.embedding, md.vocab_size, md.d_model, ids, h, stream)
        for b in self.blocks:
            b.prefill_seq_dev(int(seq), h, n, ws, need, stream)
        self.positions[int(seq)] = n
        if int(seq) == 0:
            self.pos = n
        return h, n, ws

    SCORE_ROWS = 256  # rows of logits held at a time

    def score(self, tokens, stream=None, seq: int = 0, top_k: int = 0):
        """How likely each token of a new sequence is after those before it
        (held as sequence ``seq``, as prefill leaves it): device tensors
        logprobs and entropy [len(tokens) - 1], in nats, row i of token
        i + 1, and with top_k the likeliest tokens there, ids and log
        probabilities [len(tokens) - 1][top_k].  The mean of -logprobs is
        the log of the sequence's perplexity.  Returns once they are written."""
        import torch

        from .gpu import logprobs_dev, logprobs_workspace_size, rms_norm_dev

        md, k = self.md, int(top_k)
        ids = [int(t) for t in tokens]
        if len(ids) < 2:
            raise ValueError(f"a score needs at least two tokens, got {len(ids)}")
        if not 0 <= k <= min(64, md.vocab_size):  # as logprobs_dev, before the sequence is replaced
            raise KernelError(f"logprobs top_k must be at most 64 and the vocabulary of {md.vocab_size}, got {k}")
        h, n, ws = self._prefill_rows(ids, stream, seq)
        targets = torch.tensor(ids[1:], dtype=torch.int32, device="cuda")
        torch.cuda.current_stream().synchronize()  # the targets are there, whatever stream reads them
        step = min(n - 1, self.SCORE_ROWS)
        hn = torch.empty((step, md.d_model), dtype=torch.float32, device="cuda")
        logits = torch.empty((step, md.vocab_size), dtype=torch.float32, device="cuda")
        logp, ent = (torch.empty(n - 1, dtype=torch.float32, device="cuda") for _ in range(2))
        top_ids = torch.empty((n - 1, k), dtype=torch.int32, device="cuda") if k else None
        tops = torch.empty((n - 1, k), dtype=torch.float32, device="cuda") if k else None
        need = logprobs_workspace_size(step, md.vocab_size, k)
        lws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        for r in range(0, n - 1, step):
            m = min(step, n - 1 - r)
            rms_norm_dev(self.ctx, h[r:r + m], m, md.d_model, self.final_norm, md.rms_norm_eps, hn, stream,
                         self.serving)
            self.head.logits_dev(hn, m, logits, stream)
            logprobs_dev(self.ctx, logits, m, md.vocab_size, targets[r:r + m], logp[r:r + m], ent[r:r + m], lws, need,
                         top_k=k, top_ids=top_ids[r:r + m] if k else None, top_logprobs=tops[r:r + m] if k else None,
                         stream=stream)
        torch.cuda.synchronize()  # what was allocated here is free again for any stream
        return (logp, ent, top_ids, tops) if k else (logp, ent)

    def step_batch(self, tokens, stream=None):
        """One position of each of sequences 0 .. n - 1 (the batched decode of
        engine/mod.rs:1377-1476): ``tokens`` n host ids, or a device int32
        tensor of n ids (a greedy loop's argmax output, fed back without a
        host round trip).  Returns the logits [n][vocab] (a device tensor,
        overwritten by the next call of the same n)."""
        import torch

        from .gpu import embed, embed_dev, rms_norm_dev

        md = self.md
        dev_ids = hasattr(tokens, "is_cuda")
        n = int(tokens.numel()) if dev_ids else len(tokens)
        if n == 0 or n > self.n_seqs:
            raise ValueError(f"a batch of {n} sequences on a model holding {self.n_seqs}")
        if n not in self._batch:
            wn = max(b.decode_batch_workspace_size(n) for b in self.blocks)
            with _memory_of(stream):
                self._batch[n] = (torch.empty((n, md.d_model), dtype=torch.float32, device="cuda"),
                                  torch.empty((n, md.d_model), dtype=torch.float32, device="cuda"),
                                  torch.empty((n, md.vocab_size), dtype=torch.float32, device="cuda"),
                                  torch.empty(wn, dtype=torch.uint8, device="cuda"), wn)
        h, hn, logits, ws, wn = self._batch[n]
        if dev_ids:
            embed_dev(self.ctx, self.embedding, md.vocab_size, md.d_model, tokens, n, h, stream)
        else:
            embed(self.ctx, self.embedding, md.vocab_size, md.d_model, [int(t) for t in tokens], h, stream)
        pos = self.positions[:n]
        for b in self.blocks:
            b.decode_batch_dev(h, pos, ws, wn, stream)
        rms_norm_dev(self.ctx, h, n, md.d_model, self.final_norm, md.rms_norm_eps, hn, stream)
        self.head.logits_dev(hn, n, logits, stream)
        for i in range(n):
            self.positions[i] += 1
        self.pos = self.positions[0]
        return logits

    def share_prefix(self, tokens, n_seqs: int, capacity: int, fmt: str = "int8", stream=None):
        """Serves ``n_seqs`` (up to 64) requests behind one prompt: the tokens
        are prefilled once (as sequence 0), their cache rows quantised into an
        8-bit cache per block, and every request gets room for ``capacity``
        rows of its own there; step_shared() then steps them together, each
        block reading the prompt's rows for many of them at a time.  bf16 serving;
        prompt and capacity together within the model's capacity.  Returns the
        prompt's last logits, as prefill."""
        import torch

        from .gpu import KvCache

        md, n, kd = self.md, len(tokens), self.md.n_kv_heads * self.md.head_dim
        if self.serving != "bf16":
            raise ValueError("a shared prefix is served in bf16")
        if not 1 <= int(n_seqs) <= 64 or n + int(capacity) > self.capacity:
            raise ValueError(f"{n_seqs} requests of {capacity} rows behind {n} on a model of {self.capacity} positions")

        def size(seqs, rows):
            return KvCache.size(fmt, seqs, rows, md.n_kv_heads, md.head_dim)

        size(1, n), size(int(n_seqs), int(capacity))  # refusals come before sequence 0 is replaced
        self._wait_shared()
        logits = self.prefill(tokens, stream)

        def cache(seqs, rows):
            need = size(seqs, rows)
            return KvCache(self.ctx, fmt, seqs, rows, md.n_kv_heads, md.head_dim,
                           torch.empty(need, dtype=torch.uint8, device="cuda"))

        d, seqs = md.d_model, int(n_seqs)
        with _memory_of(stream):
            pos = torch.zeros(seqs, dtype=torch.int32, device="cuda")
            prefixes, caches = [], []
            for b in self.blocks:
                k, v = b.cache_ptrs()
                prefixes.append(cache(1, n))
                prefixes[-1].write_dev(k, v, "float32", pos, n, row_stride=kd, stream=stream)
                caches.append(cache(seqs, int(capacity)))
            need = max(b.decode_kv_workspace_size(c, seqs, prefix_len=n) for b, c in zip(self.blocks, caches))
            self._shared = {"n": seqs, "prefix": prefixes, "len": n, "own": caches, "pos": pos, "steps": 0,
                            "h": torch.empty((seqs, d), dtype=torch.float32, device="cuda"),
                            "hn": torch.empty((seqs, d), dtype=torch.float32, device="cuda"),
                            "logits": torch.empty((seqs, md.vocab_size), dtype=torch.float32, device="cuda"),
                            "ws": torch.empty(need, dtype=torch.uint8, device="cuda"), "need": need}
        return logits

    def step_shared(self, tokens, stream=None):
        """The next position of every request of share_prefix(): ``tokens`` as
        step_batch's, one a request.  Returns the logits [n][vocab] (a device
        tensor, overwritten by the next call).  A captured step serves this
        shared prefix alone and counts once towards the requests' capacity,
        however often it is replayed; replays past it write no rows."""
        from .gpu import advance_positions_dev, embed, embed_dev, rms_norm_dev

        md, s = self.md, self._shared
        if s is None:
            raise ValueError("step_shared needs share_prefix first")
        dev_ids = hasattr(tokens, "is_cuda")
        n = int(tokens.numel()) if dev_ids else len(tokens)
        if n != s["n"]:
            raise ValueError(f"{n} tokens for {s['n']} requests")
        if s["steps"] >= s["own"][0].capacity:
            raise ValueError(f"the requests hold their {s['steps']} rows already")
        if dev_ids:
            embed_dev(self.ctx, self.embedding, md.vocab_size, md.d_model, tokens, n, s["h"], stream)
        else:
            embed(self.ctx, self.embedding, md.vocab_size, md.d_model, [int(t) for t in tokens], s["h"], stream)
        for b, own, prefix in zip(self.blocks, s["own"], s["prefix"]):
            b.decode_kv_dev(s["h"], s["pos"], n, own, s["ws"], s["need"], prefix=prefix, prefix_len=s["len"],
                            stream=stream)
        advance_positions_dev(self.ctx, s["pos"], n, stream)
        rms_norm_dev(self.ctx, s["h"], n, md.d_model, self.final_norm, md.rms_norm_eps, s["hn"], stream)
        self.head.logits_dev(s["hn"], n, s["logits"], stream)
        s["steps"] += 1
        return s["logits"]

    def step(self, token: int, stream=None):
        """The next position's logits (a device tensor, overwritten by the
        next step) for a host token id."""
        from .gpu import embed, rms_norm_dev

        md = self.md
        embed(self.ctx, self.embedding, md.vocab_size, md.d_model, [int(token)], self.h, stream)
        for b in self.blocks:
            b.decode_dev(self.h, self.pos, stream)
        rms_norm_dev(self.ctx, self.h, 1, md.d_model, self.final_norm, md.rms_norm_eps, self.hn, stream,
                     self.serving)
        self.head.logits_dev(self.hn, 1, self.logits, stream)
        self.pos += 1
        self.positions[0] = self.pos
        return self.logits

    def close(self):
        for b in self.blocks:
            b.close()
        self.head.close()
        for layers in self.layers:
            for L in layers:
                L.close()
