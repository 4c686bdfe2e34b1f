"""Gradients of linear attention described for any number of tokens or sequences: the results of static descriptions, bit for bit."""
import pytest
import torch

from akg_amd import driver
from dynamic_cases import open_extent
from test_attention_use import empties
from test_linear_attention import describe_grad, make


def tensors(batch, tokens):
    return make(("bfloat16", "BSND", batch, tokens, 4, 2, 64, 40, "slow", True, None))


@pytest.mark.gpu
@pytest.mark.parametrize("open_,sizes", [("tokens", [(2, 65), (2, 190), (2, 9), (2, 1500), (2, 2100)]), ("batch", [(1, 70), (3, 70), (40, 70)])])
def test_gradient_of_open_extents(open_, sizes, tmp_path):
    many = 7919
    of = dict(batch=2, tokens=many) if open_ == "tokens" else dict(batch=many, tokens=70)
    t = {n: x.to("meta") if x.dim() == 4 else x for n, x in tensors(1, 70).items()}
    for n in ("q", "k", "v", "dout"):
        t[n] = t[n].new_empty((of["batch"], of["tokens"]) + tuple(t[n].shape[2:]))
    for n in ("state", "dstate"):
        t[n] = t[n].new_empty((of["batch"],) + tuple(t[n].shape[1:]))
    dyn = driver.HipDynamicKernel(open_extent(describe_grad(t, "BSND", name="Fused_OpenLinearGrad")[0], (many,)), out_dir=str(tmp_path))
    sources = []
    for batch, tokens in sizes:
        text, inputs = describe_grad(tensors(batch, tokens), "BSND", name="Fused_StaticLinearGrad")
        static = driver.HipKernel(text, out_dir=str(tmp_path))
        ins, expect, got = [x.contiguous().cuda() for x in inputs], empties(static), empties(static)
        static.launch(ins + expect)
        used = dyn.launch_packed([x.data_ptr() for x in ins + got], [list(x.shape) for x in ins + got], torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, o) for a, o in zip(expect, got)), (batch, tokens)
        sources.append(used.source)
    assert sources[0] == sources[1]
