"""Descriptions that return some of attention's gradients: the launches and products of the others are left out, and what is
returned has the bits that the description of all three gives."""
import json

import pytest
import torch

import attention_reference as ref
from akg_amd import driver, op_desc
from test_attention_ops import NAMES, attention_case, builder, given, normal

TORCH = {v: k for k, v in NAMES.items()}
SUBSETS = [(0,), (1,), (2,), (0, 1), (0, 2), (1, 2)]


def text_of(asked, tensors, extra, options):
    b = builder("Fused_Grad_" + "".join(str(i) for i in asked))
    args = [given(b, x) for x in tensors]
    grads = op_desc.attention_grad(b, *args, **{n: given(b, x) for n, x in extra.items()}, **options)
    return b.dumps([grads[i] for i in asked])


def launches(asked, directory, dtype="bfloat16", batch=2, seq=4096, heads=32, hkv=8, dim=128):
    """Names of the kernels that run, the last one `kernel`, and the source."""
    x = lambda h: torch.empty((batch, seq, h, dim), dtype=TORCH[dtype], device="meta")   # noqa: E731
    tensors = [x(heads), x(heads), x(hkv), x(hkv), x(heads), torch.empty((batch, heads, seq), device="meta")]
    kernel = driver.HipKernel(text_of(asked, tensors, {}, {"causal": True}), out_dir=str(directory))
    name = "Fused_Grad_" + "".join(str(i) for i in asked)
    meta = json.load(open(str(directory / (name + ".json")), encoding="utf-8"))
    return [p["kernelName"][len(name) + 1:] for p in meta.get("earlier_phases", [])] + ["kernel"], kernel.source


def test_what_nobody_asks_for_is_not_launched(tmp_path):
    assert launches((0, 1, 2), tmp_path)[0] == ["queries", "kernel"]
    names, source = launches((0,), tmp_path)
    assert names == ["kernel"] and "backward_keys" not in source
    assert launches((0,), tmp_path, dtype="float16")[0] == ["values", "kernel"]
    for asked in ((1,), (2,), (1, 2)):
        names, source = launches(asked, tmp_path)
        assert names == ["rows", "kernel"]
        assert "backward_queries<akg_C, 4, 1>" in source and "backward_queries<akg_C, 8, 0>" not in source
    # small ones: dq stands beside dk and dv only where both sides are asked for
    small = dict(batch=8, seq=200, heads=12, hkv=12, dim=64)
    for asked in ((0, 1, 2), (0, 1), (0, 2)):
        names, source = launches(asked, tmp_path, **small)
        assert names == ["rows", "kernel"] and "akg_Q" in source and "akg_K" in source
    assert launches((0,), tmp_path, **small)[0] == ["kernel"]
    assert launches((1,), tmp_path, **small)[0] == ["rows", "kernel"]
    # rows in ranges: no join where there is only dq
    few = dict(batch=1, seq=1024, heads=16, hkv=4)
    assert launches((0, 1, 2), tmp_path, **few)[0] == ["queries", "keys", "kernel"]
    assert launches((0,), tmp_path, **few)[0] == ["kernel"]
    assert launches((2,), tmp_path, **few)[0] == ["rows", "keys", "kernel"]


CASES = [
    ("float16", "BSND", 2, 70, 90, 4, 2, 64, 64, True, None, None),
    ("bfloat16", "BNSD", 2, 65, 130, 4, 2, 128, 40, False, "float32", "padded"),
    ("float16", "BSND", 1, 600, 600, 8, 2, 64, 64, True, None, "padded"),       # rows of dk and dv in ranges
    ("bfloat16", "BSND", 1, 300, 300, 40, 8, 128, 128, True, None, None),
    ("float16", "BSND", 1, 700, 90, 4, 2, 192, 192, True, "bool", "padded"),    # dk and dv by workgroups of their own, in ranges
    ("bfloat16", "BSND", 1, 130, 200, 160, 160, 192, 256, False, None, None),
    ("float16", "BSND", 1, 700, 700, 40, 40, 64, 64, True, None, None),         # a launch each
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_some_gradients_have_the_bits_of_all(case, tmp_path):
    t, extra, options, m, ql, kl = attention_case(case)
    dtype = TORCH[case[0]]
    r = ref.forward(t["q"], t["k"], t["v"], mask=m, qlens=ql, klens=kl, **options)
    tensors = [normal(r["out"].shape, case[0], 5), t["q"], t["k"], t["v"], r["out"].to(dtype), r["lse"].float()]
    device = [x.contiguous().cuda() for x in tensors + list(extra.values())]

    def run(asked):
        kernel = driver.HipKernel(text_of(asked, tensors, extra, options), out_dir=str(tmp_path))
        outs = [torch.full(d.shape, float("nan"), dtype=dtype, device="cuda") for d in kernel.outputs]
        kernel.launch(device + outs)
        torch.cuda.synchronize()
        return outs

    whole = run((0, 1, 2))
    assert all(torch.isfinite(x).all() for x in whole)
    for asked in SUBSETS:
        for i, x in zip(asked, run(asked)):
            assert torch.equal(x, whole[i]), (asked, i)
