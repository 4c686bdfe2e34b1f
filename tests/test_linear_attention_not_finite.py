"""A token whose key, value or query is not finite spoils, of its own head, results that depend on it and no other."""
import math

import pytest
import torch

from test_attention_ops import launch
from test_linear_attention import describe, describe_grad, make

CASES = [
    # dtype, tokens, the token, channels, channels of the values, state
    ("bfloat16", 6, 3, 64, 64, True), ("bfloat16", 300, 200, 64, 64, True), ("bfloat16", 64, 63, 128, 128, False), ("bfloat16", 100, 97, 128, 96, False),
    ("bfloat16", 100, 40, 256, 256, True), ("bfloat16", 100, 70, 256, 256, False), ("float16", 130, 100, 64, 64, True), ("float16", 70, 50, 256, 256, True),
    ("float16", 100, 99, 128, 128, False), ("bfloat16", 1100, 900, 64, 64, True), ("bfloat16", 12, 9, 32, 40, False),
]


def spoilt(t, which, at, x):
    t = dict(t)
    t[which] = t[which].clone()
    t[which][1, at, 2, 5] = x
    return t


@pytest.mark.gpu
@pytest.mark.parametrize("which,x", [("v", math.inf), ("v", math.nan), ("k", -math.inf), ("k", math.nan), ("q", math.nan)])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_tokens_in_front_keep_their_results(case, which, x, tmp_path):
    dtype, tokens, at, dim, e, state = case
    t = make((dtype, "BSND", 2, tokens, 4, 4, dim, e, "slow", state, None))
    text, inputs = describe(t, "BSND", last=state)
    clean = launch(text, inputs, tmp_path)
    text, inputs = describe(spoilt(t, which, at, x), "BSND", last=state)
    got = launch(text, inputs, tmp_path)
    others = [0, 1, 3]
    for a, o in zip(clean, got):
        assert torch.equal(a[0], o[0])
    assert torch.equal(clean[0][1, :, others], got[0][1, :, others])
    assert torch.equal(clean[0][1, :at, 2], got[0][1, :at, 2])
    if which == "q":
        assert torch.isnan(got[0][1, at, 2]).all() and torch.equal(clean[0][1, at + 1:, 2], got[0][1, at + 1:, 2])
        assert not state or torch.equal(clean[1], got[1])
    else:
        bad = ~torch.isfinite(got[0][1, at:, 2])
        assert bad[..., 5].all() if which == "v" else bad.all()
        if which == "v":   # (other channels of the values never meet it)
            assert torch.equal(clean[0][1, :, 2, 6:], got[0][1, :, 2, 6:])
        if state:
            assert torch.equal(clean[1][1, others], got[1][1, others]) and not torch.isfinite(got[1][1, 2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["dout", "q", "k", "v"])
@pytest.mark.parametrize("case", [c for c in CASES if c[1] > 8], ids=lambda c: "-".join(str(x) for x in c))
def test_gradients_that_do_not_depend_on_it(case, which, tmp_path):
    """dq of the tokens in front (their own dout apart), dk and dv of those behind."""
    dtype, tokens, at, dim, e, state = case
    t = make((dtype, "BSND", 2, tokens, 4, 4, dim, e, "slow", state, None))
    text, inputs = describe_grad(t, "BSND")
    clean = launch(text, inputs, tmp_path)
    text, inputs = describe_grad(spoilt(t, which, at, math.inf), "BSND")
    got = launch(text, inputs, tmp_path)
    others = [0, 1, 3]
    for n, a, o in zip(("dq", "dk", "dv", "dstate"), clean, got):
        assert torch.equal(a[0], o[0]), n
        if n == "dstate":
            assert torch.equal(a[1, others], o[1, others])
            continue
        assert torch.equal(a[1, :, others], o[1, :, others]), n
        if n == "dq":
            assert torch.equal(a[1, :at, 2], o[1, :at, 2]), n
        else:
            assert torch.equal(a[1, at + 1:, 2], o[1, at + 1:, 2]), n
    # what each does meet
    met = {"dout": ("dq", "dk", "dv"), "q": ("dk", "dv"), "k": ("dq", "dv"), "v": ("dq", "dk")}[which]
    for n, o in zip(("dq", "dk", "dv"), got):
        assert torch.isfinite(o[1, at, 2]).all() == (n not in met), n
