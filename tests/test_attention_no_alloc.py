"""Launches without allocations of attention, its gradient and cache attention whose usual schedule shares an axis through more
than 16 MiB: they run with fewer ranges, or none."""
import json

import pytest
import torch

import attention_reference as ref
from akg_amd import driver, op_desc
from test_attention_ops import CACHE_ORDER, NAMES, attention_case, builder, cache_case, close, describe_attention, describe_cache, given, normal
from test_attention_use import empties, layer_inputs, training_layer
from test_cache_attention_scales import as_reference, tight_bound

LIMIT = 16 << 20


def attention_text(batch, q, k, heads, hkv, dim, causal=True):
    b = builder("Fused_AttentionWithin")
    x = [b.input([batch, n, h, dim], "bfloat16") for n, h in ((q, heads), (k, hkv), (k, hkv))]
    return b.dumps(op_desc.attention(b, *x, causal=causal))


def gradient_text(batch, seq, heads, hkv, dim, dtype="bfloat16"):
    b = builder("Fused_GradWithin")
    shape = lambda h: [batch, seq, h, dim]   # noqa: E731
    x = [b.input(shape(h), dtype) for h in (heads, heads, hkv, hkv, heads)]
    return b.dumps(op_desc.attention_grad(b, *x, b.input([batch, heads, seq], "float32"), causal=True))


def cache_text(batch, q, heads, hkv, dim, page, per):
    b = builder("Fused_CacheWithin")
    x = [b.input([batch, q, heads, dim], "bfloat16")] + [b.input([batch * per, hkv, page, dim], "int8") for _ in range(2)]
    x += [b.input([batch * per, hkv], "float32") for _ in range(2)] + [b.input([batch, per], "int32"), b.input([batch], "int32")]
    return b.dumps([op_desc.cache_attention(b, *x)])


@pytest.mark.parametrize("text", [
    attention_text(1, 64, 4096, 32, 8, 128), attention_text(1, 2000, 1030, 8, 2, 256, causal=False), gradient_text(1, 1024, 16, 4, 128), gradient_text(1, 2048, 32, 8, 128),
    gradient_text(1, 4096, 32, 4, 128, "float16"), gradient_text(2, 2048, 32, 8, 256), cache_text(1, 512, 32, 8, 128, 64, 256), cache_text(2, 300, 32, 8, 256, 64, 128)])
def test_a_schedule_within_16_mib_stands_beside_the_usual_one(text, tmp_path):
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    assert kernel.workspace_bytes > LIMIT and "_within_kernel" in kernel.source
    meta = json.load(open(str(tmp_path / (kernel.kernel_name[:-len("_kernel")] + ".json")), encoding="utf-8"))
    assert "_within" not in meta["kernelName"] and not any("_within" in p["kernelName"] for p in meta.get("earlier_phases", []))


def test_there_is_one_schedule_where_16_mib_suffice(tmp_path):
    for text in (attention_text(8, 1, 8192, 32, 8, 128), gradient_text(2, 4096, 32, 8, 128), cache_text(32, 1, 32, 8, 128, 64, 256)):
        kernel = driver.HipKernel(text, out_dir=str(tmp_path))
        assert kernel.workspace_bytes <= LIMIT and "_within" not in kernel.source


def without_allocations(kernel, device):
    """Results of a launch through the fixed array, and of a captured one replayed twice."""
    kernel.prepare()
    outs, again = empties(kernel), empties(kernel)
    stream = torch.cuda.current_stream().cuda_stream
    kernel.launch_static_scratch_ptrs([x.data_ptr() for x in device + outs], stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernel.launch_static_scratch_ptrs([x.data_ptr() for x in device + again], torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        for x in again:
            x.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(outs, again))
    return [x.cpu() for x in outs]


@pytest.mark.gpu
@pytest.mark.parametrize("case", [("bfloat16", "BSND", 1, 64, 4096, 32, 8, 128, 128, True, None, "padded"),
                                  ("float16", "BSND", 1, 2000, 1030, 8, 2, 64, 256, False, None, None)], ids=lambda c: "-".join(str(x) for x in c))
def test_attention_within(case, tmp_path):
    t, extra, options, m, ql, kl = attention_case(case)
    text, inputs = describe_attention(t, extra, options)
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    assert "_within" in kernel.source
    out, lse = without_allocations(kernel, [x.contiguous().cuda() for x in inputs])
    r = ref.forward(t["q"], t["k"], t["v"], mask=m, qlens=ql, klens=kl, **options)
    close(out, r["out"], ref.forward_bound(r, case[0]), "out")
    some = ~torch.isinf(r["lse"])
    assert ((lse[some].double() - r["lse"][some]).abs() <= ref.lse_bound(r) + 2.0 ** -23 * r["lse"][some].abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [("bfloat16", "BSND", 1, 1024, 1024, 16, 4, 128, 128, True, None, "padded"),
                                  ("float16", "BNSD", 1, 2048, 1500, 8, 4, 128, 128, False, None, None)], ids=lambda c: "-".join(str(x) for x in c))
def test_gradient_within(case, tmp_path):
    t, extra, options, m, ql, kl = attention_case(case)
    r = ref.forward(t["q"], t["k"], t["v"], mask=m, qlens=ql, klens=kl, **options)
    dtype = ref.TYPES[case[0]]
    tensors = [normal(r["out"].shape, case[0], 8), t["q"], t["k"], t["v"], r["out"].to(dtype), r["lse"].float()]
    b = builder("Fused_GradWithin")
    grads = op_desc.attention_grad(b, *[given(b, x) for x in tensors], **{n: given(b, x) for n, x in extra.items()}, **options)
    kernel = driver.HipKernel(b.dumps(grads), out_dir=str(tmp_path))
    assert "_within" in kernel.source
    got = without_allocations(kernel, [x.contiguous().cuda() for x in tensors + list(extra.values())])
    exact, size = ref.gradient(*tensors, mask=m, qlens=ql, klens=kl, **options)
    for n, x in zip(("dq", "dk", "dv"), got):
        close(x, exact[n]["exact"], ref.gradient_bound(exact[n], case[0], size, 128), n)


@pytest.mark.gpu
def test_cache_within(tmp_path):
    t = cache_case(("bfloat16", 1, 300, 32, 8, 128, 64, 130, [8200], None))
    t = {n: t[n] for n in CACHE_ORDER}
    kernel = driver.HipKernel(describe_cache(t), out_dir=str(tmp_path))
    assert "_within" in kernel.source
    got = without_allocations(kernel, [x.cuda() for x in t.values()])[0]
    # (every 37th query against float64)
    part = dict(t)
    rows = torch.arange(0, 300, 37)
    whole = torch.empty(t["q"].shape, dtype=torch.float64)
    bound = torch.empty(t["q"].shape, dtype=torch.float64)
    for i in rows.tolist():
        part["q"], part["lengths"] = t["q"][:, i:i + 1].contiguous(), t["lengths"] - 300 + 1 + i
        r = ref.cache_attention(**as_reference(part))
        whole[:, i:i + 1], bound[:, i:i + 1] = r["out"], tight_bound(part, r, "bfloat16")
    close(got[:, rows], whole[:, rows], bound[:, rows], "cache attention")


@pytest.mark.gpu
def test_a_training_layer_within(tmp_path):
    """The gradient as a stage of a longer description."""
    t = layer_inputs("bfloat16", 1, 1024, 16, 4, 128)
    text, names = training_layer(t, False)
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    order = [t[n] for n in ("q", "k", "v", "dout", "positions")]
    got = dict(zip(names, without_allocations(kernel, [x.cuda() for x in order])))
    g, size = ref.gradient(t["dout"], got["q1"], got["k1"], t["v"], got["out"], got["lse"], causal=True)
    for name, key in (("dq1", "dq"), ("dk1", "dk"), ("dv", "dv")):
        close(got[name], g[key]["exact"], ref.gradient_bound(g[key], "bfloat16", size, 128), name)
