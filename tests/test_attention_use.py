"""The operators of an attention layer as a program uses them: behind one another in one description, captured into a graph, on
another stream, through the calling form for open extents, without allocations, on tensors at odd addresses, on tensors
longer than 32-bit offsets, on blocks that this library's row quantisation wrote."""
import json

import pytest
import torch

import attention_reference as ref
from akg_amd import driver, op_desc
from dynamic_cases import open_extent
from test_attention_ops import CACHE, CACHE_ORDER, NAMES, attention_case, builder, cache_case, close, describe_attention, describe_cache, given, normal

TORCH = {v: k for k, v in NAMES.items()}


def empties(kernel):
    return [torch.empty(d.shape, dtype=TORCH[d.dtype], device="cuda") for d in kernel.outputs]


def training_layer(t, lengths, causal=True):
    """Rotary positions, attention, its gradient and the positions' own, every tensor between them an output."""
    b = builder("Fused_AttentionLayer")
    q, k, v, dout, positions = (given(b, t[n]) for n in ("q", "k", "v", "dout", "positions"))
    n = given(b, t["lengths"]) if lengths else None
    options = dict(query_lengths=n, key_lengths=n, causal=causal)
    turned = op_desc.rotary_embedding(b, [q, k], positions, base=10000.0)
    out, lse = op_desc.attention(b, *turned, v, **options)
    dq, dk, dv = op_desc.attention_grad(b, dout, *turned, v, out, lse, **options)
    back = op_desc.rotary_embedding(b, [dq, dk], positions, base=10000.0, inverse=True)
    names = ["q1", "k1", "out", "lse", "dq1", "dk1", "dv", "dq", "dk"]
    return b.dumps(turned + [out, lse, dq, dk, dv] + back), names


def layer_inputs(dtype, batch=2, seq=75, heads=4, kv=2, dim=64):
    t = {"q": normal((batch, seq, heads, dim), dtype, 1, 2.0), "k": normal((batch, seq, kv, dim), dtype, 2), "v": normal((batch, seq, kv, dim), dtype, 3),
         "dout": normal((batch, seq, heads, dim), dtype, 4)}
    t["positions"] = torch.arange(seq, dtype=torch.int32) + 1000
    t["lengths"] = torch.tensor([seq] + [seq - 20] * (batch - 1), dtype=torch.int32)
    return t


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_a_training_layer_in_one_description(dtype, tmp_path):
    t = layer_inputs(dtype)
    text, names = training_layer(t, True)
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    assert kernel.family == "staged"
    outs = empties(kernel)
    order = [t[n] for n in ("q", "k", "v", "dout", "positions", "lengths")]
    kernel.launch([x.cuda() for x in order] + outs)
    got = {n: x.cpu() for n, x in zip(names, outs)}
    lengths = t["lengths"].tolist()
    u = ref.half_step(dtype)
    # every step against float64 on what it was given
    for name, x in (("q1", t["q"]), ("k1", t["k"])):
        exact = ref.rotary(x, t["positions"])
        close(got[name], exact, u * exact.abs() * 1.01 + 2.0 ** -19 * float(x.abs().max()), name)
    r = ref.forward(got["q1"], got["k1"], t["v"], causal=True, qlens=lengths, klens=lengths)
    close(got["out"], r["out"], ref.forward_bound(r, dtype), "out")
    g, size = ref.gradient(t["dout"], got["q1"], got["k1"], t["v"], got["out"], got["lse"], causal=True, qlens=lengths, klens=lengths)
    for name, key in (("dq1", "dq"), ("dk1", "dk"), ("dv", "dv")):
        close(got[name], g[key]["exact"], ref.gradient_bound(g[key], dtype, size, 64), name)
    for name, x in (("dq", got["dq1"]), ("dk", got["dk1"])):
        exact = ref.rotary(x, t["positions"], inverse=True)
        close(got[name], exact, u * exact.abs() * 1.01 + 2.0 ** -19 * float(x.abs().max()), name)


def test_a_training_layer_is_cut_at_its_operators(tmp_path):
    text, _ = training_layer(layer_inputs("bfloat16"), True)
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    meta = json.load(open(str(tmp_path / "Fused_AttentionLayer.json"), encoding="utf-8"))
    assert kernel.family == "staged" and len(meta["stages"]) == 4
    # an elementwise op in front and behind: kernels of their own around the operator
    b = builder("Fused_Scaled")
    x = b.input([2, 40, 4, 64], "float16")
    half = b.mul(x, b.const(0.5, "float16"))
    out = op_desc.attention(b, half, x, x, lse=False)[0]
    kernel = driver.HipKernel(b.dumps([b.add(out, x)]), out_dir=str(tmp_path))
    meta = json.load(open(str(tmp_path / "Fused_Scaled.json"), encoding="utf-8"))
    assert kernel.family == "staged" and len(meta["stages"]) == 3


@pytest.mark.gpu
def test_elementwise_ops_around_attention_of_one_tensor(tmp_path):
    x = normal((2, 40, 4, 64), "float16", 6)
    b = builder("Fused_Scaled")
    i = given(b, x)
    half = b.mul(i, b.const(0.5, "float16"))
    out = op_desc.attention(b, half, i, i, lse=False)[0]
    kernel = driver.HipKernel(b.dumps([b.add(out, i)]), out_dir=str(tmp_path))
    outs = empties(kernel)
    kernel.launch([x.cuda()] + outs)
    r = ref.forward((x.float() * 0.5).to(torch.float16), x, x)
    u = ref.half_step("float16")
    exact = r["out"] + x.double()
    close(outs[0].cpu(), exact, ref.forward_bound(r, "float16") * (1 + u) + u * exact.abs() * 1.01 + 2.0 ** -25, "sum")


@pytest.mark.gpu
def test_results_of_the_gradient_that_nobody_asks_for(tmp_path):
    """dk alone, and dq alone, equal what the description with all three gives."""
    case = ("bfloat16", "BSND", 2, 70, 90, 4, 2, 64, 64, True, None, None)
    t, _, options, _, _, _ = attention_case(case)
    r = ref.forward(t["q"], t["k"], t["v"], **options)
    given_tensors = [normal(r["out"].shape, "bfloat16", 5), t["q"], t["k"], t["v"], r["out"].to(torch.bfloat16), r["lse"].float()]
    results = {}
    for asked in ((0, 1, 2), (1,), (0,)):
        b = builder("Fused_Grad%d" % len(asked) + str(asked[0]))
        grads = op_desc.attention_grad(b, *[given(b, x) for x in given_tensors], **options)
        kernel = driver.HipKernel(b.dumps([grads[i] for i in asked]), out_dir=str(tmp_path))
        outs = empties(kernel)
        kernel.launch([x.contiguous().cuda() for x in given_tensors] + outs)
        results[asked] = [o.cpu() for o in outs]
    assert torch.equal(results[(1,)][0], results[(0, 1, 2)][1]) and torch.equal(results[(0,)][0], results[(0, 1, 2)][0])


def several(tmp_path):
    """(kernel, inputs on the device) of every operator: split and whole, with lengths, a mask, a cache."""
    jobs = []

    def add(text, inputs):
        jobs.append((driver.HipKernel(text, out_dir=str(tmp_path)), [x.cuda() for x in inputs]))
    t = layer_inputs("float16")
    text, _ = training_layer(t, True)
    add(text, [t[n] for n in ("q", "k", "v", "dout", "positions", "lengths")])
    for case in (("bfloat16", "BSND", 2, 1, 3000, 8, 2, 64, 64, True, None, "padded"), ("float16", "BNSD", 2, 150, 130, 4, 4, 128, 128, False, "float32", None)):
        t, extra, options, _, _, _ = attention_case(case)
        add(*describe_attention(t, extra, options))
    for case in (CACHE[2], CACHE[9]):
        t = cache_case(case)
        t = {n: t[n] for n in CACHE_ORDER}
        add(describe_cache(t), list(t.values()))
    return jobs


@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream(tmp_path):
    """All of them in one graph on a side stream, replayed four times on new inputs with eager launches between: bit for bit
    the eager results (no sum depends on an order that may change)."""
    jobs = several(tmp_path)
    static = [([x.clone() for x in ins], empties(k)) for k, ins in jobs]
    for k, _ in jobs:
        k.prepare()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for (k, _), (ins, outs) in zip(jobs, static):
            k.launch(ins + outs)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for (k, _), (ins, outs) in zip(jobs, static):
            k.launch(ins + outs)
    for turn in range(4):
        for ins, outs in static:
            for x in ins:
                if x.is_floating_point():
                    x.mul_(1.0 - 0.125 * turn)
            for o in outs:
                o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for (k, _), (ins, outs) in zip(jobs, static):
            alone = empties(k)
            k.launch(ins + alone)
            torch.cuda.synchronize()
            for i, (a, o) in enumerate(zip(alone, outs)):
                assert torch.equal(a.view(torch.uint8), o.view(torch.uint8)), (turn, k.kernel_name, i)


@pytest.mark.gpu
def test_without_allocations(tmp_path):
    for k, ins in several(tmp_path):
        k.prepare()
        first, second = empties(k), empties(k)
        k.launch(ins + first)
        k.launch_static_scratch_ptrs([x.data_ptr() for x in ins + second], torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for a, o in zip(first, second):
            assert torch.equal(a.view(torch.uint8), o.view(torch.uint8)), k.kernel_name


@pytest.mark.gpu
def test_open_extents(tmp_path):
    """One description for any number of queries and keys, or tokens: the results of the static ones, and one code object for
    sizes that need the same kernel."""
    def attention_of(q, k, name):
        b = builder(name)
        x = [b.input([2, n, h, 64], "bfloat16") for n, h in ((q, 4), (k, 2), (k, 2))]
        return b.dumps(op_desc.attention(b, *x, causal=True))
    dyn = driver.HipDynamicKernel(open_extent(attention_of(7919, 7907, "Fused_OpenAttention"), (7919, 7907)), out_dir=str(tmp_path))
    seen = []
    for q, k in ((65, 65), (90, 100), (1, 4000)):
        ins = [normal((2, n, h, 64), "bfloat16", 40 + i).cuda() for i, (n, h) in enumerate(((q, 4), (k, 2), (k, 2)))]
        static = driver.HipKernel(attention_of(q, k, "Fused_StaticAttention"), out_dir=str(tmp_path))
        expect, got = empties(static), empties(static)
        static.launch(ins + expect)
        special = dyn.specialize([list(x.shape) for x in ins])
        assert [d.shape for d in special.outputs] == [list(o.shape) for o in got]
        used = dyn.launch_packed([x.data_ptr() for x in ins + got], [list(x.shape) for x in ins + got], torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for a, o in zip(expect, got):
            assert torch.equal(a, o)
        seen.append(used.source)
    assert seen[0] == seen[1] != seen[2]


def at_odd_address(x):
    """A contiguous copy of `x` one element behind the start of its storage."""
    whole = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
    view = whole[1:].view(x.shape)
    view.copy_(x)
    return view


@pytest.mark.gpu
def test_tensors_at_odd_addresses(tmp_path):
    for k, ins in several(tmp_path):
        expect = empties(k)
        k.launch(ins + expect)
        moved = [at_odd_address(o) for o in expect]
        for m in moved:
            m.fill_(0)
        k.launch([at_odd_address(x) for x in ins] + moved)
        torch.cuda.synchronize()
        for a, o in zip(expect, moved):
            assert torch.equal(a, o), k.kernel_name


@pytest.mark.gpu
def test_keys_and_blocks_behind_32_bit_offsets(tmp_path):
    # 2.3 GB of keys and as much of values of one sequence; the last key heads are checked
    sk, heads, dim = 140001, 64, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn((1, 2, heads, dim), generator=g, device="cuda").to(torch.bfloat16)
    k, v = (torch.randn((1, sk, heads, dim), generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    b = builder("Fused_LongKeys")
    kernel = driver.HipKernel(b.dumps(op_desc.attention(b, given(b, q), given(b, k), given(b, v), causal=True)), out_dir=str(tmp_path))
    outs = empties(kernel)
    kernel.launch([q, k, v] + outs)
    torch.cuda.synchronize()
    part = [x[:, :, 62:].cpu() for x in (q, k, v)]
    r = ref.forward(*part, causal=True)
    close(outs[0][:, :, 62:].cpu(), r["out"], ref.forward_bound(r, "bfloat16"), "long keys")
    del k, v
    # a pool of 2.3 GB a side whose last blocks are the live ones
    case = ("bfloat16", 2, 1, 8, 4, 128, 64, 5, [320, 130], None)
    t = cache_case(case)
    blocks = 70000
    for n in ("key", "value"):
        small = t[n + "_cache"]
        t[n + "_cache"] = torch.zeros((blocks,) + tuple(small.shape[1:]), dtype=torch.int8, device="cuda")
        t[n + "_cache"][-small.shape[0]:] = small.cuda()
        scale = torch.zeros((blocks, 4))
        scale[-small.shape[0]:] = t[n + "_scale"]
        t[n + "_scale"] = scale
    first = blocks - 13
    t["block_table"] += first
    t = {n: t[n] for n in CACHE_ORDER}
    kernel = driver.HipKernel(describe_cache(t), out_dir=str(tmp_path))
    outs = empties(kernel)
    kernel.launch([x.cuda() for x in t.values()] + outs)
    torch.cuda.synchronize()
    near = {n: (x[first:].cpu() if n.endswith(("_cache", "_scale")) else x) for n, x in t.items()}
    near["table"] = near.pop("block_table") - first
    r = ref.cache_attention(**near)
    close(outs[0].cpu(), r["out"], ref.cache_bound(r, "bfloat16"), "far blocks")


@pytest.mark.gpu
def test_blocks_that_the_row_quantisation_wrote(tmp_path):
    """Keys and values of a prefill, turned by their positions, quantised block by block with this library's row quantisation
    (a row is a block of one key head), then attended by the last token."""
    batch, blocks, hkv, heads, page, dim = 2, 5, 2, 8, 32, 64
    rows, cols = batch * blocks * hkv, page * dim
    b = builder("Fused_QuantBlocks")
    x = b.input([rows, cols], "bfloat16")
    s = b.cast(x, "float32")
    scale = b.div(b.reduce("ReduceMax", b.unary("Abs", s), [1], False), b.const(127.0, "float32"))
    q8 = b.cast(b.div(s, b.reshape(scale, [rows, 1])), "int8")
    quant = driver.HipKernel(b.dumps([q8, scale]), out_dir=str(tmp_path))
    cache = {}
    for n, seed in (("key", 51), ("value", 52)):
        outs = empties(quant)
        dense = normal((batch * blocks, hkv, page, dim), "bfloat16", seed)
        quant.launch([dense.view(rows, cols).cuda()] + outs)
        cache[n + "_cache"], cache[n + "_scale"] = outs[0].view(batch * blocks, hkv, page, dim), outs[1].view(batch * blocks, hkv)
        torch.cuda.synchronize()
        back = cache[n + "_cache"].cpu().double() * cache[n + "_scale"].cpu().double()[..., None, None]
        # half a step of the scale, and the division's and the scale's own roundings of a number up to 127
        assert ((back - dense.double()).abs() <= cache[n + "_scale"].cpu().double()[..., None, None] * (0.5 + 127 * 2.0 ** -22)).all()
    t = {"q": normal((batch, 1, heads, dim), "bfloat16", 53, 2.0), **cache}
    t["block_table"] = torch.arange(batch * blocks, dtype=torch.int32).view(batch, blocks)
    t["lengths"] = torch.tensor([blocks * page, blocks * page - 17], dtype=torch.int32)
    t = {n: t[n].cuda() for n in CACHE_ORDER}
    kernel = driver.HipKernel(describe_cache(t), out_dir=str(tmp_path))
    outs = empties(kernel)
    kernel.launch(list(t.values()) + outs)
    host = {n: x.cpu() for n, x in t.items()}
    host["table"] = host.pop("block_table")
    r = ref.cache_attention(**host)
    close(outs[0].cpu(), r["out"], ref.cache_bound(r, "bfloat16"), "cache attention")
