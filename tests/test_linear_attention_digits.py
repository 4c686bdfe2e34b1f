"""Digits of linear attention's states: float32 whatever the decay, how long the text and how large the state given."""
import pytest
import torch

import linear_reference as ref
from akg_amd import driver
from test_attention_ops import launch, normal
from test_attention_use import empties
from test_linear_attention import decays, describe, describe_grad, make

F = torch.float64
STEP = 2.0 ** -24   # half a step of float32, relative to the value


def faded(state, g, tokens):
    """exp(g tokens) times the state [.., heads, channels, channels]."""
    return state.to(F) * torch.exp(g.to(F) * tokens)[:, None, None]


def fade_bound(exact, g, tokens, chunk):
    """A chunk's factor: exponent g n in turns of log 2 off by 2.5 half steps (g log2 e, times n, the constant), the power of two
    by two; each product with it by one. So 2.5 |g| tokens + 3 a chunk of half steps in all, and what is below float32."""
    y = (g.to(F).abs() * tokens)[:, None, None]
    return exact.abs() * (3 * y + 3 * (tokens / chunk + 1) + 8) * STEP + 1e-36


STRONG = torch.tensor([-0.001, -0.02, -0.05, -0.08, -0.12, -0.17, -0.22, -0.3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,e,tokens,batch", [("bfloat16", 64, 64, 128, 2), ("bfloat16", 64, 64, 100, 2), ("float16", 64, 40, 130, 2), ("bfloat16", 256, 256, 96, 2),
                                                      ("float16", 256, 64, 96, 2), ("bfloat16", 128, 128, 200, 32), ("bfloat16", 64, 64, 900, 1), ("bfloat16", 32, 64, 6, 2)])
def test_a_state_keeps_its_digits_however_fast_it_fades(dtype, dim, e, tokens, batch, tmp_path):
    """Tokens that add nothing behind a large state: what is left of it, with the digits of float32, whatever share that is; and the
    results, which read it."""
    g = STRONG
    t = {"q": normal((batch, tokens, 8, dim), dtype, 1), "k": torch.zeros((batch, tokens, 8, dim)).to(getattr(torch, dtype)),
         "v": normal((batch, tokens, 8, e), dtype, 3), "log_decay": g, "state": normal((batch, 8, dim, e), "float32", 4, 1e4)}
    text, inputs = describe(t, "BSND", scale=2.0 ** -12)
    out, last = launch(text, inputs, tmp_path)
    exact = faded(t["state"], g, tokens)
    off, bound = (last.to(F) - exact).abs(), fade_bound(exact, g, tokens, 32 if tokens > 8 else 1)
    assert (off <= bound).all(), float((off / bound).max())
    seen = torch.matmul(t["q"].to(F).transpose(1, 2), t["state"].to(F)) * 2.0 ** -12   # [batch, heads, tokens, channels]
    size = torch.matmul(t["q"].to(F).transpose(1, 2).abs(), t["state"].to(F).abs()) * 2.0 ** -12
    fade = torch.exp(g.to(F)[:, None] * (torch.arange(tokens) + 1))[None, :, :, None]
    back = lambda x: (x * fade).transpose(1, 2)   # noqa: E731
    bound = ref.bound(back(seen), [back(size), back(size)], dtype, dim, tokens)
    off = (out.to(F) - back(seen)).abs()
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tokens", [("bfloat16", 128), ("float16", 100), ("bfloat16", 900)])
def test_the_gradient_of_a_state_keeps_its_digits(dtype, tokens, tmp_path):
    """The same backward: results that nobody needs, and the last state's gradient on its way to the state given."""
    g = STRONG
    t = {n: normal((2, tokens, 8, 64), dtype, 1 + i) for i, n in enumerate(("q", "k", "v"))}
    t.update(dout=torch.zeros_like(t["q"]), log_decay=g, state=normal((2, 8, 64, 64), "float32", 4), dstate=normal((2, 8, 64, 64), "float32", 5, 1e4))
    text, inputs = describe_grad(t, "BSND")
    got = launch(text, inputs, tmp_path)[3]
    exact = faded(t["dstate"], g, tokens)
    bound = fade_bound(exact, g, tokens, 32)
    off = (got.to(F) - exact).abs()
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.gpu
def test_fading_does_not_drift_over_a_long_text(tmp_path):
    """256 chunks in one walk: what the products round goes either way, so the mean over a head's state is off by what its decay's
    exponent is off by. A factor rounded once would be off by the same share every time."""
    batch, heads, tokens = 32, 8, 16384
    g = -(2.0 ** -12) * (1 + torch.arange(heads) / 8.0)
    zeros = lambda h: torch.zeros((batch, tokens, h, 8), dtype=torch.bfloat16)   # noqa: E731
    t = {"q": zeros(heads), "k": zeros(1), "v": zeros(1), "log_decay": g, "state": normal((batch, heads, 8, 8), "float32", 4).abs() + 0.5}
    text, inputs = describe(t, "BSND")
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    assert kernel.workspace_bytes == 0   # (no segments)
    outs = empties(kernel)
    kernel.launch([x.cuda() for x in inputs] + outs)
    exact = faded(t["state"], g, tokens)
    share = ((outs[1].cpu().to(F) - exact) / exact).mean((0, 2, 3))
    bound = (3 * g.to(F).abs() * tokens + 8) * STEP
    once = torch.exp(g.to(F) * 64).float().to(F) ** (tokens // 64) / torch.exp(g.to(F) * tokens) - 1
    assert (once.abs() > 2 * bound).any()   # (that it would show)
    assert (share.abs() <= bound).all(), share


# What is added to a state that is a result goes as three bfloat16 parts: 2^-27 of it is left, two would leave 2^-18. Float32 adds,
# over 1024 tokens with the decays taken here, at most 54 roundings that count of 2^-25.5 on average, and weights off by
# some 4 half steps each: 3e-7 of a state in the mean square.
DIGITS = 2.0 ** -20


def kept(dtype):
    t = make((dtype, "BSND", 2, 1024, 4, 2, 64, 64, "slow", True, None))
    t["state"], t["dstate"] = t["state"] * 0, t["dstate"] * 0
    return t


def mean_square(got, exact):
    return float(((got.to(F) - exact).square().mean((0, 2, 3)) / exact.square().mean((0, 2, 3))).sqrt().max())


def test_two_parts_would_show():
    t = kept("bfloat16")
    g = decays("slow", 4).to(F)
    k, v = (t[n].to(F).transpose(1, 2).repeat_interleave(2, 1) for n in ("k", "v"))
    at = torch.arange(1024)
    inside, behind = (torch.exp(g[:, None] * n)[None, :, :, None] for n in (63 - at % 64, 1023 - at - (63 - at % 64)))
    exact = (k * inside * behind).transpose(2, 3) @ v
    rest, left = (v * inside).float(), {}
    whole = torch.zeros_like(v)
    for n in (1, 2, 3):
        part = rest.to(torch.bfloat16).float()
        rest, whole = rest - part, whole + part.to(F)
        left[n] = mean_square((k * behind).transpose(2, 3) @ whole, exact)
    assert left[3] < DIGITS / 16 and left[2] > 2 * DIGITS


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tokens", [("bfloat16", 1024), ("bfloat16", 960), ("float16", 1024)])
def test_what_is_added_to_a_state_keeps_its_digits(dtype, tokens, tmp_path):
    """Of a state that is a result, forward and backward. (float16: its keys are two parts themselves, without a rest; the product of
    the second with the third part of what is added, 2^-26 of it, is left out.)"""
    t = kept(dtype)
    t = {n: x[:, :tokens].contiguous() if n in ("q", "k", "v", "dout") else x for n, x in t.items()}
    text, inputs = describe(t, "BSND")
    off = mean_square(launch(text, inputs, tmp_path)[1], ref.forward(t["q"], t["k"], t["v"], t["log_decay"])["last"])
    assert off <= DIGITS, off
    text, inputs = describe_grad(t, "BSND")
    off = mean_square(launch(text, inputs, tmp_path)[3], ref.gradient(t["dout"], t["q"], t["k"], t["v"], t["log_decay"])["dstate"][0])
    assert off <= DIGITS, off
