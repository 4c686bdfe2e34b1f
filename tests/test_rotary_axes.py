"""Rotary positions of several axes: against float64 on the host for every order of axes and rates, layout, type and shape of
positions; one axis against no axes; refusals."""
import pytest
import torch

import linear_reference as ref
from akg_amd import driver, op_desc
from attention_reference import half_step
from dynamic_cases import open_extent
from test_attention_ops import builder, close, given, launch, normal, refused
from test_attention_use import empties

CASES = [
    # dtype, layout, batch, seq, heads, kv heads, channels, turned, sections, order, rates, interleaved, inverse, positions
    ("bfloat16", "BSND", 2, 5, 3, 1, 64, 0, [8, 12, 12], "blocks", "shared", False, False, "int32"),
    ("bfloat16", "BSND", 1, 300, 32, 8, 128, 0, [16, 24, 24], "cycle", "shared", False, False, "int32"),
    ("float32", "BNSD", 3, 33, 4, 2, 96, 64, [16, 16], "blocks", "own", True, True, "int64"),
    ("float16", "BSND", 3, 17, 9, 2, 80, 40, [5, 8, 7], "cycle", "own", True, False, "shared"),
    ("float16", "BNSD", 1, 130, 8, 0, 128, 32, [1, 0, 15], "blocks", "own", False, True, "far"),
    ("float32", "BSND", 1, 1, 1, 0, 2, 0, [0, 1], "cycle", "shared", False, False, "int32"),
    ("float32", "BSND", 2, 7, 2, 1, 13, 6, [1, 2], "blocks", "shared", False, False, "one batch"),
    ("bfloat16", "BSND", 4, 100, 16, 2, 256, 0, [3, 125], "cycle", "own", False, False, "negative"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_axes(case, tmp_path):
    dtype, layout, batch, seq, heads, kv, dim, turned, sections, order, rates, interleaved, inverse, kind = case
    shape = lambda h: (batch, seq, h, dim) if layout == "BSND" else (batch, h, seq, dim)   # noqa: E731
    xs = [normal(shape(h), dtype, 11 + h) for h in (heads, kv) if h]
    first = {"far": 1000000, "negative": -150}.get(kind, 0)
    rows = 1 if kind in ("shared", "one batch") else batch
    positions = torch.stack([first + (torch.arange(seq) * (a + 3)) % (29 + 11 * a) + torch.arange(rows)[:, None] * 13 * (a + 1) for a in range(len(sections))])
    positions = positions if kind == "int64" else positions.to(torch.int32)
    b = builder()
    options = dict(layout=layout, base=500000.0, rotary_dims=turned, interleaved=interleaved, inverse=inverse, magnitude=1.25)
    handed = positions[:, 0].contiguous() if kind == "shared" else positions
    outs = op_desc.rotary_embedding(b, [given(b, x) for x in xs], given(b, handed), sections=sections, axis_order=order, axis_rates=rates, **options)
    got = launch(b.dumps(outs), xs + [handed], tmp_path)
    u, r = half_step(dtype), turned or dim
    for x, y in zip(xs, got):
        exact = ref.rotary_axes(x, positions, sections, order, rates, **options)
        # the result rounded (u); sine, cosine, products and sums off by a few 2^-24 of the pair's size
        bound = u * exact.abs() * 1.01 + 2.0 ** -20 * float(x.double().abs().amax()) * 2.5 + (2.0 ** -25 if dtype == "float16" else 0)
        close(y, exact, bound, "rotary")
        assert torch.equal(y[..., r:], x[..., r:])   # what is not turned is copied


@pytest.mark.gpu
@pytest.mark.parametrize("order,rates", [("blocks", "shared"), ("cycle", "own")])
def test_one_axis_and_equal_axes_are_plain_positions(order, rates, tmp_path):
    x = normal((2, 19, 4, 64), "bfloat16", 3)
    at = torch.arange(38, dtype=torch.int32).view(2, 19) * 701

    def turned(positions, **options):
        b = builder()
        return launch(b.dumps(op_desc.rotary_embedding(b, [given(b, x)], given(b, positions), **options)), [x, positions], tmp_path)[0]
    plain = turned(at)
    assert torch.equal(plain, turned(at[None].contiguous(), sections=[32], axis_order=order, axis_rates=rates))
    if rates == "shared":
        assert torch.equal(plain, turned(torch.stack([at] * 3), sections=[10, 0, 22], axis_order=order, axis_rates=rates))


@pytest.mark.gpu
def test_turned_back_captured_and_open(tmp_path):
    """There and back in one graph, replayed on new positions; and the same through the calling form for open extents."""
    def text_of(seq, name):
        b = builder(name)
        x, p = b.input([2, seq, 4, 64], "float32"), b.input([2, 2, seq], "int32")
        there = op_desc.rotary_embedding(b, [x], p, sections=[20, 12])
        return b.dumps(there + op_desc.rotary_embedding(b, there, p, sections=[20, 12], inverse=True))
    kernel = driver.HipKernel(text_of(19, "Fused_AxesThereAndBack"), out_dir=str(tmp_path))
    x, p = normal((2, 19, 4, 64), "float32", 3).cuda(), (torch.arange(76, dtype=torch.int32).view(2, 2, 19) * 37).cuda()
    outs = empties(kernel)
    kernel.prepare()
    kernel.launch([x, p] + outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernel.launch([x, p] + outs)
    for turn in range(3):
        p.add_(1001)
        for o in outs:
            o.fill_(7)
        graph.replay()
        alone = empties(kernel)
        kernel.launch([x, p] + alone)
        torch.cuda.synchronize()
        assert all(torch.equal(a, o) for a, o in zip(alone, outs))
        close(outs[1].cpu(), x.cpu().double(), 2.0 ** -20 * x.abs().double().amax().cpu(), "there and back")
    dyn = driver.HipDynamicKernel(open_extent(text_of(7919, "Fused_OpenAxes"), 7919), out_dir=str(tmp_path))
    got = empties(kernel)
    dyn.launch_packed([t.data_ptr() for t in [x, p] + got], [list(t.shape) for t in [x, p] + got], torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for a, o in zip(outs, got))


def test_refusals():
    def turned(dim=64, positions=("int32", [3, 5]), sections=(8, 12, 12), **options):
        b = builder()
        return b.dumps(op_desc.rotary_embedding(b, [b.input([2, 5, 4, dim], "bfloat16")], b.input(positions[1], positions[0]), sections=sections, **options))
    driver.translate(turned())
    driver.translate(turned(positions=("int64", [3, 2, 5]), axis_order="cycle", axis_rates="own"))
    driver.translate(turned(positions=("int64", [3, 1, 5])))
    refused(turned(sections=(8, 12, 11)), -3, "half of rotary_dims")
    refused(turned(sections=(8, 12, 12), rotary_dims=32), -3, "half of rotary_dims")
    refused(turned(sections=(8, 28, -4)), -3, "whole numbers of pairs")
    refused(turned(sections=()), -3, "list")
    refused(turned(sections=[0] * 15 + [16] * 2), -3, "16 axes")
    refused(turned(positions=("int32", [5])), -3, "axes")
    refused(turned(positions=("int32", [2, 5])), -3, "axes")
    refused(turned(positions=("int32", [2, 3, 5])), -3, "axes")
    refused(turned(positions=("int32", [3, 3, 5])), -3, "axes")
    refused(turned(positions=("int32", [3, 2, 6])), -3, "axes")
    refused(turned(positions=("float32", [3, 5])), -3, "int32 or int64")
    refused(turned(axis_order="rows"), -3, "axis_order")
    refused(turned(axis_rates="none"), -3, "axis_rates")
