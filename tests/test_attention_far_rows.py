"""Keys of one tile that lie nearly 2 GiB apart: the gradient's kernel of keys and values takes as many of them as its 32-bit
offsets reach."""
import pytest
import torch

import attention_reference as ref
from akg_amd import driver, op_desc
from test_attention_ops import builder, close, given, refused


def gradient_text(heads, dim=128, keys=128, queries=4):
    b = builder("Fused_FarGrad")
    shape = lambda n: [1, n, heads, dim]   # noqa: E731
    dout, q = b.input(shape(queries), "bfloat16"), b.input(shape(queries), "bfloat16")
    k, v = b.input(shape(keys), "bfloat16"), b.input(shape(keys), "bfloat16")
    return b.dumps(op_desc.attention_grad(b, dout, q, k, v, b.input(shape(queries), "bfloat16"), b.input([1, heads, queries], "float32")))


def test_tiles_of_keys_within_32_bit_offsets(tmp_path):
    # a tile of 128 keys ends below 2^31 bytes up to 65533 heads of 128 channels; one of 64 up to 131067
    def tile(heads):
        source = driver.HipKernel(gradient_text(heads), out_dir=str(tmp_path)).source
        return 128 if "backward_keys<akg_C, 4," in source else 64 if "backward_keys<akg_C, 2," in source else 0
    assert tile(65000) == 128 and tile(65533) == 128
    assert tile(65534) == 64 and tile(70000) == 64 and tile(131067) == 64
    refused(gradient_text(131068), -4, "2 GiB")


@pytest.mark.gpu
def test_gradients_of_keys_two_gib_apart(tmp_path):
    keys, queries, heads, dim = 128, 4, 70000, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn((1, keys, heads, dim), generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    dout, q = (torch.randn((1, queries, heads, dim), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    out, lse = torch.zeros_like(q), torch.zeros((1, heads, queries), device="cuda")
    chosen = [0, 34999, 69999]
    part = [x[:, :, chosen].cpu() for x in (dout, q, k, v)]
    r = ref.forward(*part[1:])
    out[:, :, chosen], lse[:, chosen] = r["out"].to(torch.bfloat16).cuda(), r["lse"].float().cuda()
    b = builder("Fused_FarGrad")
    args = [dout, q, k, v, out, lse]
    kernel = driver.HipKernel(b.dumps(op_desc.attention_grad(b, *[given(b, x) for x in args])), out_dir=str(tmp_path))
    outs = [torch.full_like(x, float("nan")) for x in (q, k, v)]
    kernel.launch(args + outs)
    torch.cuda.synchronize()
    exact, size = ref.gradient(*part, r["out"].to(torch.bfloat16), r["lse"].float())
    for n, x in zip(("dq", "dk", "dv"), outs):
        close(x[:, :, chosen].cpu(), exact[n]["exact"], ref.gradient_bound(exact[n], "bfloat16", size, dim), n)
