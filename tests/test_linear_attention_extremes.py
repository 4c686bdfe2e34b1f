"""Linear attention where numbers are extreme: decays above 0, decays of -infinity before states that are not finite, values that are
not finite behind the tokens whose results are looked at."""
import math

import pytest
import torch

import linear_reference as ref
from test_attention_ops import close, launch
from test_linear_attention import check_forward, check_gradient, describe, describe_grad, make

GROWING = [
    # dtype, layout, batch, tokens, heads, kv heads, channels, channels of the values, decay, state, lengths; the largest log decay. It times
    # the tokens rounded up to 16, at most 64, stays below 88
    (("bfloat16", "BSND", 2, 9, 4, 2, 64, 64, "none", True, None), 2.0), (("bfloat16", "BSND", 2, 9, 2, 2, 64, 64, "none", False, None), 5.0),
    (("bfloat16", "BNSD", 1, 33, 2, 1, 64, 40, "none", True, None), 1.5), (("bfloat16", "BSND", 3, 65, 4, 4, 128, 128, "none", False, "padded"), 1.0),
    (("bfloat16", "BSND", 2, 17, 2, 2, 256, 256, "none", True, "zero"), 1.5), (("bfloat16", "BSND", 1, 50, 4, 2, 32, 32, "none", False, None), 0.5),
    (("float16", "BSND", 2, 9, 2, 1, 64, 64, "none", True, None), 0.5), (("float16", "BNSD", 1, 33, 2, 2, 256, 64, "none", False, None), 0.1),
    (("bfloat16", "BSND", 1, 1200, 2, 2, 64, 64, "none", True, None), 0.02), (("bfloat16", "BSND", 2, 6, 2, 2, 64, 64, "none", True, None), 8.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case,most", GROWING, ids=lambda c: "-".join(str(x) for x in c) if isinstance(c, tuple) else str(c))
def test_decays_above_zero(case, most, tmp_path):
    """States that grow: as the definition has it, also where a chunk has few tokens."""
    t, layout = make(case), case[1]
    heads = case[4]
    t["log_decay"] = most * (1 + torch.arange(heads, dtype=torch.float32)) / heads
    scale = 2.0 ** -10 if case[0] == "float16" else None
    text, inputs = describe(t, layout, scale=scale)
    check_forward(t, layout, launch(text, inputs, tmp_path), scale=scale)
    if case[3] > 8:
        text, inputs = describe_grad(t, layout, scale=scale)
        check_gradient(t, layout, launch(text, inputs, tmp_path), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [100, 700, 6000])
def test_growing_behind_tokens_that_add_nothing(tokens, tmp_path):
    """Half of the text adds nothing to a state of nothing, in segments too, over which exp(g tokens) is no float32 number."""
    t = make(("bfloat16", "BSND", 1, tokens, 2, 2, 64, 64, "none", False, None))
    quiet = tokens - 60
    t["log_decay"] = torch.tensor([1.0, 1.2])
    t["k"][:, :quiet] = 0
    text, inputs = describe(t, "BSND")
    got = launch(text, inputs, tmp_path)
    assert (got[0][:, :quiet] == 0).all()
    x = {n: v[:, quiet:] if n in ("q", "k", "v") else v for n, v in t.items()}
    r = ref.forward(x["q"], x["k"], x["v"], x["log_decay"])
    # chunks begin elsewhere in the whole text: a term that is in a masked product here may be in the state there, where each is
    # rounded by itself, so that the sizes of the terms count, not those of their sums
    close(got[0][:, quiet:], r["out"], ref.bound(r["out"], [r["rough"][1]] * 2, "bfloat16", 64, tokens), "out")
    close(got[1], r["last"], ref.state_bound(r["last_rough"], 64, tokens), "last state")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tokens,dim", [("bfloat16", 1, 64), ("float16", 6, 96), ("bfloat16", 70, 64), ("float16", 70, 256), ("bfloat16", 1200, 64), ("bfloat16", 6000, 64)])
@pytest.mark.parametrize("pool", [False, True])
def test_nothing_is_left_of_a_state_where_the_decay_is_infinite(dtype, tokens, dim, pool, tmp_path):
    """An entry of a pool may hold anything where a head forgets everything; a sequence without tokens leaves it as it is."""
    t = make((dtype, "BSND", 3, tokens, 4, 2, dim, dim, "all", True, None))
    t["lengths"] = torch.tensor([tokens, 0, max(1, tokens - 5)], dtype=torch.int32)
    if pool:
        t["slots"] = torch.tensor([2, 0, 1], dtype=torch.int32)
    text, inputs = describe(t, "BSND")
    clean = launch(text, inputs, tmp_path)
    forgets = torch.isinf(t["log_decay"])
    t["state"][:, forgets] = torch.tensor([math.nan, math.inf, -math.inf]).repeat(dim * dim)[:dim * dim].view(dim, dim)
    text, inputs = describe(t, "BSND")
    out, last = launch(text, inputs, tmp_path)
    assert torch.equal(out, clean[0])
    idle = 0 if pool else 1
    others = [i for i in range(3) if i != idle]
    assert torch.equal(last[others], clean[1][others])
    assert torch.equal(last[idle].view(torch.int32), t["state"][idle].view(torch.int32))
    if not pool and tokens > 8:
        t["state"] = t["state"] * 1
        text, inputs = describe_grad(t, "BSND", wanted=[0], name="Fused_QueriesOnly")
        dirty = launch(text, inputs, tmp_path)[0]
        t["state"][:, forgets] = 0
        text, inputs = describe_grad(t, "BSND", wanted=[0], name="Fused_QueriesOnly")
        assert torch.equal(dirty, launch(text, inputs, tmp_path)[0])
