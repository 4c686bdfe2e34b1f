"""Linear attention where numbers are extreme: decays above 0."""
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
