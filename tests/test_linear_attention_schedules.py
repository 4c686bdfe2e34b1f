"""Every schedule of linear attention that real sizes choose, at sizes that the host can check: which one a case chose is asserted, so
that a schedule which is no longer chosen is no longer taken for tested."""
import re

import pytest
import torch

import linear_reference as ref
from akg_amd import driver
from test_attention_use import empties
from test_linear_attention import check_forward, check_gradient, describe, describe_grad, make


def schedules(source):
    """Of every walk: (32-token tiles of a chunk, wavefronts of columns, wavefronts that share a state's rows, wavefronts that fetch, one
    chunk's tiles only, three parts of what is added)."""
    walks = re.findall(r"linear::Config<([^>]*)>", source)
    return [tuple(int(x) for x in w.split(", ")[3:7]) + tuple(x == "true" for x in w.split(", ")[7:9]) for w in walks]


def parts(source):
    return "three" if "_starts" in source else "joined" if "_states" in source else "one"


FORWARD = [
    # dtype, layout, batch, tokens, heads, kv heads, channels, channels of the values, decay, states, lengths; schedule, launches
    (("bfloat16", "BSND", 2, 300, 4, 2, 64, 64, "slow", False, "padded"), (2, 1, 1, 4, False, False), "one"),
    (("bfloat16", "BSND", 9, 200, 32, 32, 64, 64, "slow", False, "padded"), (2, 2, 1, 2, False, False), "one"),
    (("bfloat16", "BNSD", 9, 200, 32, 16, 64, 64, "mixed", True, "padded"), (2, 2, 1, 2, False, True), "one"),
    (("float16", "BSND", 8, 70, 33, 33, 64, 40, "slow", False, "zero"), (1, 2, 1, 2, False, False), "one"),
    (("float16", "BSND", 9, 200, 32, 16, 64, 64, "slow", True, "padded"), (1, 2, 1, 2, False, True), "one"),
    (("bfloat16", "BSND", 8, 200, 32, 32, 128, 128, "slow", False, "padded"), (2, 4, 1, 4, False, False), "one"),
    (("bfloat16", "BSND", 8, 200, 32, 16, 128, 128, "all", True, "zero"), (2, 4, 1, 4, False, True), "one"),
    (("bfloat16", "BSND", 4, 1003, 16, 4, 96, 80, "slow", True, "padded"), (2, 3, 1, 4, False, True), "joined"),
    (("bfloat16", "BSND", 16, 100, 16, 8, 256, 256, "slow", False, "padded"), (1, 4, 1, 4, False, False), "one"),
    (("bfloat16", "BNSD", 16, 100, 16, 8, 256, 256, "mixed", True, "zero"), (1, 2, 2, 4, False, True), "one"),
    (("bfloat16", "BSND", 2, 1000, 4, 4, 256, 256, "slow", True, "padded"), (1, 2, 2, 4, False, True), "joined"),
    (("float16", "BSND", 8, 100, 32, 16, 128, 128, "slow", False, "padded"), (1, 4, 1, 4, False, False), "one"),
    (("float16", "BSND", 8, 100, 32, 16, 128, 128, "slow", True, None), (1, 4, 1, 4, False, True), "one"),
    (("float16", "BSND", 16, 100, 16, 8, 256, 256, "slow", False, "padded"), (1, 2, 2, 4, True, False), "one"),
    (("float16", "BSND", 16, 100, 16, 8, 256, 256, "slow", True, "padded"), (1, 2, 2, 4, True, True), "one"),
    (("float16", "BSND", 2, 1000, 4, 4, 256, 256, "slow", True, "padded"), (1, 2, 2, 4, True, True), "joined"),
    (("bfloat16", "BSND", 1, 4096, 16, 16, 128, 128, "slow", True, None), (2, 4, 1, 4, False, True), "three"),
    (("bfloat16", "BSND", 1, 4096, 4, 4, 128, 128, "slow", False, None), (2, 2, 1, 4, False, False), "three"),
    (("bfloat16", "BSND", 1, 2048, 2, 2, 256, 256, "none", False, None), (1, 2, 1, 4, False, False), "three"),
    (("bfloat16", "BSND", 4, 2048, 8, 8, 256, 256, "slow", False, "padded"), (1, 4, 1, 4, False, False), "three"),
]
GRADIENT = [
    (("bfloat16", "BSND", 8, 200, 12, 12, 64, 64, "slow", False, "padded"), (2, 2, 1, 2, False, False), "one"),
    (("float16", "BSND", 8, 200, 12, 12, 64, 64, "slow", True, "padded"), (1, 2, 1, 2, False, True), "one"),
    (("bfloat16", "BSND", 8, 200, 32, 32, 128, 128, "slow", False, "padded"), (2, 4, 1, 4, False, False), "one"),
    (("bfloat16", "BNSD", 8, 200, 32, 16, 128, 128, "mixed", True, "zero"), (2, 4, 1, 4, False, True), "one"),
    (("float16", "BSND", 8, 100, 32, 32, 128, 128, "slow", False, "padded"), (1, 4, 1, 4, False, False), "one"),
    (("bfloat16", "BSND", 16, 100, 16, 8, 256, 256, "slow", False, "padded"), (1, 4, 1, 4, False, False), "one"),
    (("bfloat16", "BSND", 8, 100, 16, 8, 256, 256, "slow", True, "zero"), (1, 2, 2, 4, False, True), "one"),
    (("float16", "BSND", 8, 70, 16, 8, 256, 256, "slow", False, "padded"), (1, 2, 2, 4, True, False), "one"),
    (("float16", "BSND", 8, 70, 16, 8, 256, 256, "slow", True, "padded"), (1, 2, 2, 4, True, True), "one"),
    (("bfloat16", "BSND", 2, 1500, 2, 1, 256, 256, "slow", True, "padded"), (1, 2, 2, 4, False, True), "joined"),
]


def run(text, inputs, expected, launches, tmp_path, monkeypatch):
    """Results of the usual launch, and of the one without allocations where that has kernels of its own."""
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    source = kernel.source.split("// Generated by")   # (in front of each translation unit)
    assert schedules(source[1])[-1] == expected and parts(source[1]) == launches, (schedules(source[1]), parts(source[1]))
    # The bounds are those of the chunks that the schedule has: a term of the same chunk is rounded with the others of its masked
    # product, 2^-8 of their sum, one of an earlier chunk by itself in the state, 2^-8 of it; with chunks of 64 the first token behind 32
    # would have the former where chunks of 32 have the latter.
    monkeypatch.setattr(ref, "CHUNK", 32 * expected[0])
    ins, outs = [x.contiguous().cuda() for x in inputs], empties(kernel)
    kernel.launch(ins + outs)
    torch.cuda.synchronize()
    results = [[o.cpu() for o in outs]]
    if kernel.workspace_bytes > 16 << 20 and len(source) > 2:
        outs = empties(kernel)
        kernel.launch_static_scratch_ptrs([x.data_ptr() for x in ins + outs], torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        results.append([o.cpu() for o in outs])
    return results


@pytest.mark.gpu
@pytest.mark.parametrize("case,expected,launches", FORWARD, ids=lambda c: "-".join(str(x) for x in c) if isinstance(c, tuple) else c)
def test_forward(case, expected, launches, tmp_path, monkeypatch):
    t, layout = make(case), case[1]
    text, inputs = describe(t, layout, last=case[9])
    for got in run(text, inputs, expected, launches, tmp_path, monkeypatch):
        check_forward(t, layout, got)


@pytest.mark.gpu
@pytest.mark.parametrize("case,expected,launches", GRADIENT, ids=lambda c: "-".join(str(x) for x in c) if isinstance(c, tuple) else c)
def test_gradient(case, expected, launches, tmp_path, monkeypatch):
    t, layout = make(case), case[1]
    text, inputs = describe_grad(t, layout)
    for got in run(text, inputs, expected, launches, tmp_path, monkeypatch):
        check_gradient(t, layout, got)


def test_a_prompt_and_a_gradient_without_allocations_have_launches_of_their_own(tmp_path):
    """(that the cases above launch them)"""
    def launched(case, f, **options):
        dtype, layout, batch, tokens, heads, kv, dim, e = case[:8]
        meta = lambda h, d: torch.empty((batch, tokens, h, d), dtype=getattr(torch, dtype), device="meta")   # noqa: E731
        t = {"q": meta(heads, dim), "k": meta(kv, dim), "v": meta(kv, e), "dout": meta(heads, e), "log_decay": torch.zeros(heads)}
        if case[9]:
            t["state"] = t["dstate"] = torch.empty((batch, heads, dim, e), device="meta")
        kernel = driver.HipKernel(f(t, layout, **options)[0], out_dir=str(tmp_path))
        return kernel.workspace_bytes > 16 << 20 and "_within_kernel" in kernel.source
    assert launched(FORWARD[-1][0], describe, last=False) and launched(GRADIENT[-1][0], describe_grad)
