"""CPU: what rotating heads and verifying drafts refuse before any device use,
with the library's own error type and words, and the frequencies that a Rope
holds.  A stand-in says what a device tensor of its shape would; a call whose
tensors are right comes as far as its context, which is null here."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from quantibbler_amd import KernelError
from quantibbler_amd.gpu import Rope, rotate_heads_dev, verify_drafts_dev, verify_drafts_workspace_size
from test_tensor_checks import CTX, dev, refused

RIGHT = "null qbk_ctx"


# ---- Rope ---------------------------------------------------------------------

def radians(rope):
    return [t / 2.0 ** 64 * 2 * math.pi for t in rope._rope.turns[:rope.rotary_dim // 2]]


@pytest.mark.parametrize("d,rotary", [(2, 2), (128, 128), (128, 32), (80, 20), (256, 256)])
@pytest.mark.parametrize("theta", [10000.0, 500000.0, 1.0])
def test_plain_frequencies(d, rotary, theta):
    rope = Rope(d, theta, rotary_dim=rotary)
    # a turn's fraction is cut off at 2^-64 of a turn
    for i, f in enumerate(radians(rope)):
        assert abs(f - theta ** (-2 * i / rotary)) <= 2.0 ** -50 * f + 2.0 ** -60
    assert rope._rope.size == 1.0 and list(rope._rope.turns[rotary // 2:]) == [0] * (128 - rotary // 2)


def test_scaled_frequencies():
    d, theta = 64, 10000.0
    plain = np.array(radians(Rope(d, theta)))
    near = dict(rtol=1e-12, atol=2.0 ** -60)
    np.testing.assert_allclose(radians(Rope(d, theta, scaling={"kind": "linear", "factor": 4})), plain / 4, **near)
    np.testing.assert_allclose(radians(Rope(d, theta, scaling={"kind": "base", "factor": 3})),
                               (theta * 3 ** (d / (d - 2))) ** (-2 * np.arange(d // 2) / d), **near)
    ramp = np.array(radians(Rope(d, theta, scaling={"kind": "ramp", "factor": 8, "original_len": 1000})))
    turns = 1000 * plain / (2 * math.pi)
    assert (ramp[turns >= 4] == plain[turns >= 4]).all() and (turns >= 4).any()
    np.testing.assert_allclose(ramp[turns <= 1], plain[turns <= 1] / 8, **near)
    middle = (turns > 1) & (turns < 4)
    assert middle.any() and (ramp[middle] < plain[middle]).all() and (ramp[middle] > plain[middle] / 8).all()
    yarn = Rope(d, theta, scaling={"kind": "yarn", "factor": 16, "original_len": 4096})
    f = np.array(radians(yarn))
    assert f[0] == plain[0] and abs(f[-1] - plain[-1] / 16) <= 2.0 ** -60
    assert (np.diff(f / plain) <= 1e-9).all() and yarn._rope.size == 0.1 * math.log(16) + 1


def test_a_pair_that_turns_faster_than_once_a_position():
    """Frequencies past a turn a position count by what they leave of it: positions are whole."""
    rope = Rope(4, 1e-4)
    want = (1e-4 ** (-2 / 4) / (2 * math.pi)) % 1.0
    assert abs(rope._rope.turns[1] / 2.0 ** 64 - want) < 2.0 ** -45


@pytest.mark.parametrize("args,kw,words", [
    ((0, 1e4), {}, "even head_dim up to 256"), ((7, 1e4), {}, "even head_dim up to 256"), ((258, 1e4), {}, "258 and 258"),
    ((64, 1e4), {"rotary_dim": 66}, "64 and 66"), ((64, 1e4), {"rotary_dim": 7}, "64 and 7"),
    ((64, 1e4), {"rotary_dim": 0}, "64 and 0"), ((-2, 1e4), {}, "negative"), ((64, 1e4), {"rotary_dim": -2}, "negative"),
    ((64, 0.0), {}, "theta must be positive"), ((64, -1.0), {}, "theta must be positive"),
    ((64, float("nan")), {}, "theta must be positive"), ((64, float("inf")), {}, "theta must be positive"),
    ((64, 1e-300), {"rotary_dim": 64, "scaling": {"kind": "linear", "factor": 1e-300}}, "pass the range"),
    ((64, 1e4), {"scaling": {"kind": "ntk", "factor": 2}}, "kind must be one of"),
    ((64, 1e4), {"scaling": {"factor": 2}}, "kind must be one of"),
    ((64, 1e4), {"scaling": {"kind": "linear"}}, "missing \\['factor'\\]"),
    ((64, 1e4), {"scaling": {"kind": "linear", "factor": 2, "low": 1}}, "unknown \\['low'\\]"),
    ((64, 1e4), {"scaling": {"kind": "ramp", "factor": 2}}, "missing \\['original_len'\\]"),
    ((64, 1e4), {"scaling": {"kind": "linear", "factor": 0}}, "factor must be positive"),
    ((64, 1e4), {"scaling": {"kind": "linear", "factor": float("inf")}}, "factor must be positive"),
    ((64, 1e4), {"scaling": {"kind": "ramp", "factor": 2, "original_len": 0}}, "by parts needs"),
    ((64, 1e4), {"scaling": {"kind": "ramp", "factor": 2, "original_len": 9, "low": 4, "high": 4}}, "by parts needs"),
    ((64, 1e4), {"scaling": {"kind": "yarn", "factor": 2, "original_len": 9, "low": 0, "high": 4}}, "by parts needs"),
    ((64, 0.5), {"scaling": {"kind": "yarn", "factor": 2, "original_len": 9}}, "theta above 1"),
])
def test_ropes_that_are_refused(args, kw, words):
    with pytest.raises(KernelError, match=words):
        Rope(*args, **kw)


# ---- rotate_heads ----------------------------------------------------------------

N, HEADS, KV, D, WIDE = 6, 4, 2, 32, 300
ROPE = Rope(D, 10000.0)


def words(*shape):
    return dev(*shape, dtype=torch.int32)


def rotate(**kw):
    a = dict(rope=ROPE, q=dev(N, HEADS, D), k=dev(N, KV, D), dtype="float32", n_rows=N, n_heads=HEADS, n_kv_heads=KV,
             pos=words(3), q_out=dev(N, HEADS, D), k_out=dev(N, KV, D), n_seqs=3)
    a.update(kw)
    rotate_heads_dev(CTX, **a)


def test_rotate_takes_what_it_says():
    refused(RIGHT, rotate)
    refused(RIGHT, rotate, q=4096, k=4096, q_out=4096, k_out=4096, pos=4096, row_start=4096, q_norm=4096, k_norm=4096)
    refused(RIGHT, rotate, row_start=words(4), q_norm=dev(D), k_norm=dev(D), before=100)
    wide = dev(N, WIDE)
    refused(RIGHT, rotate, q=wide[:, :HEADS * D], k=wide[:, HEADS * D:], q_stride=WIDE, k_stride=WIDE)
    refused(RIGHT, rotate, n_kv_heads=0, k=None, k_out=None)
    refused(RIGHT, rotate, n_heads=0, q=None, q_out=None)
    b = torch.bfloat16
    refused(RIGHT, rotate, dtype="bfloat16", q=dev(N, HEADS, D, dtype=b), k=dev(N, KV, D, dtype=b),
            q_out=dev(N, HEADS, D, dtype=b), k_out=dev(N, KV, D, dtype=b))
    rotate(n_rows=0)                    # nothing to do
    rotate(n_heads=0, n_kv_heads=0)


@pytest.mark.parametrize("name,bad", [
    ("q", dev(N, HEADS, D, dtype=torch.bfloat16)), ("q", dev(N - 1, HEADS, D)), ("q", dev(N, WIDE)[:, :HEADS * D]),
    ("q", dev(N, HEADS, D, index=1)), ("q", torch.zeros(N, HEADS, D)), ("k", dev(N, KV, D - 1)), ("k", "k"),
    ("q_out", dev(N, HEADS - 1, D)), ("k_out", dev(N, KV, D, dtype=torch.float64)), ("q_norm", dev(D - 1)),
    ("k_norm", dev(D, dtype=torch.bfloat16)), ("k_norm", dev(2 * D)[::2]), ("q_norm", torch.ones(D))])
def test_rotate_refuses_other_tensors(name, bad):
    refused(f"rotate_heads: {name} must be", rotate, **{name: bad})


@pytest.mark.parametrize("kw,says", [
    (dict(pos=words(2)), "positions must be"), (dict(pos=dev(3, dtype=torch.int64)), "positions must be"),
    (dict(row_start=words(3)), "row starts must be"), (dict(dtype="float16"), "'float32' or 'bfloat16' rows"),
    (dict(n_seqs=4, pos=words(4)), "do not split evenly over 4"), (dict(n_seqs=0), "rows of no sequence"),
    (dict(n_rows=-1), "negative"), (dict(before=-1), "negative"), (dict(before=1 << 32), "too many rows"),
    (dict(q=4096, q_stride=HEADS * D - 1), "row stride of 127 does not fit a row of 128"),
    (dict(k_out=4096, k_out_stride=1 << 41), "does not fit a row of 64"), (dict(q_stride=-5), "negative"),
    (dict(q=dev(N, WIDE)[:, WIDE - 127:], q_stride=WIDE), "q must be"), (dict(q=None), "null argument"),
    (dict(q_out=None), "null argument"), (dict(k=None), "null argument"), (dict(pos=None), "null argument"),
    (dict(q_norm=dev(D), eps=-1.0), "eps must not be negative"), (dict(q_norm=dev(D), eps=float("nan")), "eps must not"),
    (dict(n_heads=65537, q=4096, q_out=4096), "up to 65536 heads"),
    (dict(n_rows=1 << 24, n_heads=64, q=4096, q_out=4096, k=4096, k_out=4096, n_seqs=1), "too many rows")])
def test_rotate_refusals(kw, says):
    refused(says, rotate, **kw)


# ---- verify_drafts ---------------------------------------------------------------

R, K, VOCAB = 3, 2, 900
NEED = verify_drafts_workspace_size(R, K, VOCAB, True)


def verify(**kw):
    a = dict(logits=dev(R, K + 1, VOCAB), n=R, drafts=K, vocab=VOCAB, ids=words(R, K), uniforms=dev(R, K + 1),
             tokens=words(R, K + 1), counts=words(R), workspace=dev(NEED, dtype=torch.uint8), workspace_size=NEED,
             draft_logits=dev(R, K, VOCAB), n_drafts=words(R), temperature=dev(R), pos=words(R))
    a.update(kw)
    verify_drafts_dev(CTX, **a)


def test_verify_takes_what_it_says():
    b = torch.bfloat16
    refused(RIGHT, verify)
    refused(RIGHT, verify, draft_logits=None, n_drafts=None, temperature=None, pos=None)
    refused(RIGHT, verify, logits=dev(R, K + 1, VOCAB, dtype=b), draft_logits=dev(R, K, VOCAB, dtype=b), dtype="bfloat16")
    refused(RIGHT, verify, logits=dev(R * (K + 1), 1000)[:, 3:], row_stride=1000, vocab=990,
            draft_logits=dev(R * K, 999)[:, 5:], draft_row_stride=999)
    refused(RIGHT, verify, drafts=0, draft_logits=None, ids=words(R, 0))
    refused(RIGHT, verify, **{name: 4096 for name in ("logits", "ids", "uniforms", "tokens", "counts", "workspace",
                                                      "draft_logits", "n_drafts", "temperature", "pos")})
    verify(n=0)


@pytest.mark.parametrize("name,bad,says", [
    ("logits", dev(R, K, VOCAB), "logits must be"), ("logits", dev(R, K + 1, VOCAB, dtype=torch.bfloat16), "logits must be"),
    ("draft_logits", dev(R, K - 1, VOCAB), "draft_logits must be"), ("draft_logits", torch.zeros(R, K, VOCAB), "draft_logits"),
    ("draft_logits", dev(R, K, VOCAB, dtype=torch.float64), "draft_logits must be"), ("ids", words(R, K - 1), "ids must be"),
    ("ids", dev(R, K, dtype=torch.int64), "ids must be"), ("uniforms", dev(R, K), "uniforms must be"),
    ("uniforms", dev(R, K + 1, dtype=torch.float64), "uniforms must be"), ("tokens", words(R, K), "tokens must be"),
    ("tokens", dev(R, K + 1, dtype=torch.int64), "tokens must be"), ("counts", words(R - 1), "counts must be"),
    ("n_drafts", dev(R, dtype=torch.int64), "n_drafts must be"), ("temperature", dev(R - 1), "temperature must be"),
    ("temperature", dev(R, dtype=torch.bfloat16), "temperature must be"), ("pos", words(R - 1), "positions must be"),
    ("workspace", dev(NEED - 1, dtype=torch.uint8), "workspace must be"), ("logits", dev(R, K + 1, VOCAB, index=1), "logits"),
    ("ids", torch.zeros((R, K), dtype=torch.int32), "ids must be")])
def test_verify_refuses_other_tensors(name, bad, says):
    refused(says, verify, **{name: bad})


@pytest.mark.parametrize("kw,says", [
    (dict(dtype="float16"), "'float32' or 'bfloat16' logits"), (dict(n=-1), "negative"), (dict(drafts=-1), "negative"),
    (dict(vocab=0), "1 <= vocab"), (dict(logits=4096, vocab=1 << 31, draft_logits=4096), "1 <= vocab"),
    (dict(drafts=65, logits=4096, draft_logits=4096, ids=4096, uniforms=4096, tokens=4096), "up to 64 drafts a request, got 65"),
    (dict(drafts=0, draft_logits=4096), "draft logits without drafts"),
    (dict(logits=4096, row_stride=VOCAB - 1), "do not fit rows of 900"),
    (dict(draft_logits=4096, draft_row_stride=1 << 41), "do not fit rows of 900"),
    (dict(workspace_size=NEED - 1), "smaller than the"), (dict(workspace=None), "smaller than the"),
    (dict(workspace=4104), "16-byte aligned"), (dict(logits=None), "null argument"), (dict(ids=None), "null argument"),
    (dict(uniforms=None), "null argument"), (dict(tokens=None), "null argument"), (dict(counts=None), "null argument"),
    (dict(n=1 << 24, logits=4096, draft_logits=4096, ids=4096, uniforms=4096, tokens=4096, counts=4096, n_drafts=4096,
          temperature=4096, pos=4096), "too many rows"),
    (dict(n=1 << 18, logits=4096, draft_logits=4096, ids=4096, uniforms=4096, tokens=4096, counts=4096, n_drafts=4096,
          temperature=4096, pos=4096, vocab=1 << 20), "too many rows")])
def test_verify_refusals(kw, says):
    refused(says, verify, **kw)


def test_workspace_sizes():
    assert verify_drafts_workspace_size(3, 65, 10) == 0 and verify_drafts_workspace_size(3, 2, 0) == 0
    assert verify_drafts_workspace_size(0, 2, 10) == 0
    # a partial result of 16 bytes a chunk of a row at least; with draft logits a sum a chunk and an end a request more
    assert verify_drafts_workspace_size(2, 3, 100) >= 2 * 4 * 16
    assert verify_drafts_workspace_size(2, 3, 100, True) >= 2 * 7 * 16 + 2 * 8 + 2 * 32
    with pytest.raises(KernelError, match="negative"):
        verify_drafts_workspace_size(-1, 2, 10)
