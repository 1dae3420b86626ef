"""CPU: what a step behind a shared prefix means, by the oracle's trunk on rows
rounded as the 8-bit cache rounds them: the ordinary decode of each request,
prompt first.  The reference's gate for logits (relative L1 0.02, cosine
0.999) tells it from the meanings that it could be mistaken for."""
import numpy as np
import pytest

from conftest import GOLDEN  # noqa: F401  (tests/ on the path)

PROMPT, STEPS = 65, 4


def synthetic(orc):
    from test_gpu_trunk import synthetic_model

    return synthetic_model(orc, 808)


def tokens(md, requests):
    rng = np.random.default_rng(31)
    return rng.integers(0, md.vocab_size, PROMPT).tolist(), rng.integers(0, md.vocab_size, (requests, STEPS)).tolist()


class Rows(np.ndarray):
    """Cache rows [row][kv_heads * head_dim] that hold what ``rounded`` makes of a head's row."""

    def __setitem__(self, at, row):
        x = np.asarray(row, np.float32)
        super().__setitem__(at, self.rounded(x.reshape(-1, self.width)).reshape(x.shape))


def rows(cache, width, rounded):
    out = np.zeros_like(cache).view(Rows)
    out.width, out.rounded = width, rounded
    return out


class Requests:
    """A prompt once through the oracle's trunk, and requests behind its rows."""

    def __init__(self, orc, md, prompt, face="sage"):
        self.md = md
        self.trunk = t = orc.Trunk(md, serving="bf16", attention="scalar", capacity=PROMPT + STEPS + 8)
        if face == "exact":
            for token in prompt:
                t.hidden(token)
        else:  # one pass
            h = t.embedding[np.array(prompt)].copy()
            for b, (layers, norms) in enumerate(t.blocks):
                h = orc.block_prefill(layers, norms, h, t.kc[b], t.vc[b], md.n_heads, md.n_kv_heads, md.head_dim,
                                      md.rope_theta, md.rms_norm_eps)
        self.prompt = [(k.copy(), v.copy()) for k, v in zip(t.kc, t.vc)]

    def logits(self, ids, fmt, change=lambda k, v: (k, v), at=PROMPT):
        """[step][vocab] of one request's tokens behind the prompt's rows (changed), its first token at position at."""
        from test_gpu_kv_cache import stored

        rounded = (lambda x: stored(x, fmt)) if fmt else (lambda x: x)
        t, width = self.trunk, self.md.head_dim
        t.kc, t.vc, t.pos = [], [], at
        for pair in self.prompt:
            k, v = (rows(x, width, rounded) for x in pair)
            k[:at], v[:at] = (x[:at] for x in change(*pair))
            t.kc.append(k)
            t.vc.append(v)
        return np.stack([t.step(i) for i in ids]).astype(np.float64)


def apart(a, b):
    """Relative L1 distance of each step's logits."""
    return np.abs(a - b).sum(-1) / np.abs(b).sum(-1)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_the_gate_tells_the_meaning_from_others(orc, fmt):
    md = synthetic(orc)
    prompt, ids = tokens(md, 2)
    r = Requests(orc, md, prompt)
    for seq in ids:
        want = r.logits(seq, fmt)
        assert (apart(want, r.logits(seq, None)) < 1 / 32).all()  # the rounding of the rows
        later = lambda k, v: tuple(np.concatenate([x[:1], x[:-1]]) for x in (k, v))
        for name, other in (("a row fewer", r.logits(seq, fmt, at=PROMPT - 1)), ("no prefix", r.logits(seq, fmt, at=0)),
                            ("a row more", r.logits(seq, fmt, later, PROMPT + 1)),
                            ("keys of other positions", r.logits(seq, fmt, lambda k, v: (np.roll(k, 1, 0), v))),
                            ("another request's tokens", r.logits(seq[::-1], fmt))):
            assert (apart(other, want) > 1 / 16).all(), name
