"""Linear attention with a decay for each head and its gradient: against float64 on the host at the sizes, lengths, decays and
states where a chunk ends, a walk is cut into segments, nothing is left or nothing is forgotten; refusals; use in graphs,
pools, pieces and a training layer."""
import json
import math

import pytest
import torch

import linear_reference as ref
from akg_amd import driver, op_desc
from dynamic_cases import open_extent
from test_attention_ops import NAMES, builder, close, given, launch, normal, refused
from test_attention_use import at_odd_address, empties

F = torch.float64


def decays(kind, heads):
    i = torch.arange(heads, dtype=torch.float32)
    return {"slow": torch.log1p(-torch.exp2(-5 - 4 * i / heads)), "none": torch.zeros(heads), "fast": -0.3 - i, "steep": -40.0 - 100 * i,
            "all": torch.where(i % 2 == 0, torch.tensor(-math.inf), -0.01 * (i + 1)), "mixed": -0.7 * i ** 2 / heads,
            "tiny": torch.full((heads,), -1e-6)}[kind]


def spread_lengths(kind, batch, seq):
    if kind is None:
        return None
    if kind == "zero":
        return ([0, seq, 1, -3, seq + 5] * batch)[:batch]
    return [max(1, seq - 29 * b) for b in range(batch)]


def make(case, poison=True):
    """Tensors of a case (name: tensor), NaN behind the lengths."""
    dtype, layout, batch, seq, heads, kv, dim, e, decay, state, kind = case
    shape = lambda h, d: (batch, seq, h, d) if layout == "BSND" else (batch, h, seq, d)   # noqa: E731
    t = {"q": normal(shape(heads, dim), dtype, 1), "k": normal(shape(kv, dim), dtype, 2), "v": normal(shape(kv, e), dtype, 3),
         "dout": normal(shape(heads, e), dtype, 4), "log_decay": decays(decay, heads)}
    lengths = spread_lengths(kind, batch, seq)
    if state:
        t["state"] = normal((batch, heads, dim, e), "float32", 5, 4.0)
        t["dstate"] = normal((batch, heads, dim, e), "float32", 6)
    if lengths is not None:
        t["lengths"] = torch.tensor(lengths, dtype=torch.int32)
        for n in ("q", "k", "v", "dout"):
            for b in range(batch):
                rows = t[n][b] if layout == "BSND" else t[n][b].transpose(0, 1)
                rows[min(max(lengths[b], 0), seq):] = math.nan
    return t


def cleaned(t, layout):
    """The tensors with zeros for what lies behind the lengths."""
    return {n: torch.nan_to_num(x) if x.is_floating_point() and n != "log_decay" else x for n, x in t.items()}


def describe(t, layout, last=True, name="Fused_Linear", wanted=None, **options):
    b = builder(name)
    order = [n for n in ("q", "k", "v", "log_decay", "state", "slots", "lengths") if n in t]
    g = {n: given(b, t[n]) for n in order}
    outs = op_desc.linear_attention(b, g["q"], g["k"], g["v"], g["log_decay"], state=g.get("state"), slots=g.get("slots"), lengths=g.get("lengths"),
                                    layout=layout, last_state=last, **options)
    return b.dumps(outs if wanted is None else [outs[i] for i in wanted]), [t[n] for n in order]


def describe_grad(t, layout, wanted=None, name="Fused_LinearGrad", **options):
    b = builder(name)
    order = [n for n in ("dout", "q", "k", "v", "log_decay", "state", "dstate", "lengths") if n in t]
    g = {n: given(b, t[n]) for n in order}
    outs = op_desc.linear_attention_grad(b, g["dout"], g["q"], g["k"], g["v"], g["log_decay"], state=g.get("state"), dstate=g.get("dstate"),
                                         lengths=g.get("lengths"), layout=layout, **options)
    return b.dumps(outs if wanted is None else [outs[i] for i in wanted]), [t[n] for n in order]


FORWARD = [
    # dtype, layout, batch, seq, heads, kv heads, channels, channels of the values, decay, state, lengths
    ("bfloat16", "BSND", 1, 1, 1, 1, 8, 8, "slow", False, None),
    ("float16", "BSND", 2, 1, 4, 2, 64, 64, "fast", True, None),
    ("bfloat16", "BNSD", 3, 1, 8, 8, 128, 128, "all", True, "zero"),
    ("bfloat16", "BSND", 2, 8, 6, 3, 40, 72, "mixed", True, "padded"),
    ("float16", "BNSD", 5, 5, 2, 1, 256, 24, "none", True, "zero"),
    ("bfloat16", "BSND", 40, 2, 16, 16, 96, 256, "slow", True, None),
    ("float16", "BSND", 1, 3, 1, 1, 8, 136, "steep", False, None),
    ("bfloat16", "BSND", 1, 9, 1, 1, 16, 8, "slow", True, None),
    ("float16", "BSND", 2, 32, 2, 2, 64, 64, "slow", False, None),
    ("bfloat16", "BNSD", 2, 33, 4, 2, 64, 32, "fast", True, None),
    ("float16", "BSND", 1, 63, 3, 1, 80, 48, "mixed", True, None),
    ("bfloat16", "BSND", 2, 64, 2, 1, 128, 128, "none", True, None),
    ("bfloat16", "BSND", 5, 65, 4, 4, 40, 104, "all", True, "zero"),
    ("float16", "BNSD", 3, 130, 6, 2, 128, 128, "slow", True, "padded"),
    ("bfloat16", "BSND", 1, 255, 2, 2, 256, 256, "slow", True, None),
    ("float16", "BSND", 1, 200, 2, 1, 256, 192, "fast", False, None),
    ("bfloat16", "BSND", 2, 1100, 4, 2, 64, 64, "slow", True, "padded"),      # segments
    ("float16", "BNSD", 3, 800, 2, 2, 96, 40, "none", True, "zero"),
    ("bfloat16", "BNSD", 1, 2049, 3, 3, 128, 80, "all", True, None),
    ("bfloat16", "BSND", 1, 1500, 2, 1, 200, 160, "steep", False, None),
    ("bfloat16", "BSND", 1, 3001, 1, 1, 32, 32, "tiny", True, None),
]


def check_forward(t, layout, got, **options):
    dtype = NAMES[t["q"].dtype]
    c = cleaned(t, layout)
    r = ref.forward(c["q"], c["k"], c["v"], c["log_decay"], state=c.get("state"), slots=c.get("slots"), lengths=c.get("lengths"), layout=layout, **options)
    close(got[0], r["out"], ref.bound(r["out"], r["rough"], dtype, r["channels"], r["seq"]), "out")
    if len(got) > 1 and "slots" not in c:
        close(got[1], r["last"], ref.state_bound(r["last_rough"], r["channels"], r["seq"], r["seq"] > 8), "last state")
    return r


@pytest.mark.gpu
@pytest.mark.parametrize("case", FORWARD, ids=lambda c: "-".join(str(x) for x in c))
def test_linear_attention(case, tmp_path):
    t, layout = make(case), case[1]
    text, inputs = describe(t, layout)
    check_forward(t, layout, launch(text, inputs, tmp_path))


GRADIENT = [
    ("bfloat16", "BSND", 1, 1, 1, 1, 8, 8, "slow", True, None),
    ("float16", "BSND", 2, 33, 2, 2, 64, 64, "slow", False, None),
    ("bfloat16", "BNSD", 2, 64, 4, 2, 128, 128, "none", True, None),
    ("bfloat16", "BSND", 5, 70, 4, 4, 40, 104, "all", True, "zero"),
    ("float16", "BSND", 3, 130, 6, 2, 80, 128, "mixed", True, "padded"),
    ("bfloat16", "BSND", 1, 200, 2, 1, 256, 256, "slow", True, None),
    ("float16", "BNSD", 1, 100, 2, 1, 256, 24, "fast", False, None),
    ("bfloat16", "BSND", 2, 1100, 4, 1, 64, 64, "slow", True, "padded"),      # segments
    ("float16", "BNSD", 3, 800, 2, 2, 96, 40, "none", True, "zero"),
    ("bfloat16", "BNSD", 1, 2049, 2, 2, 128, 72, "steep", True, None),
    ("bfloat16", "BSND", 2, 600, 16, 4, 128, 128, "slow", False, "padded"),
]


def check_gradient(t, layout, got, names=("dq", "dk", "dv", "dstate"), **options):
    dtype = NAMES[t["q"].dtype]
    c = cleaned(t, layout)
    r = ref.gradient(c["dout"], c["q"], c["k"], c["v"], c["log_decay"], state=c.get("state"), dstate=c.get("dstate"), lengths=c.get("lengths"), layout=layout, **options)
    channels, seq = max(t["q"].shape[3], t["v"].shape[3]), t["q"].shape[1 if layout == "BSND" else 2]
    for n, x in zip(names, got):
        exact, rough = r[n]
        close(x, exact, ref.state_bound(rough, channels, seq) if n == "dstate" else ref.bound(exact, rough, dtype, channels, seq), n)


@pytest.mark.gpu
@pytest.mark.parametrize("case", GRADIENT, ids=lambda c: "-".join(str(x) for x in c))
def test_gradient(case, tmp_path):
    t, layout = make(case), case[1]
    text, inputs = describe_grad(t, layout)
    check_gradient(t, layout, launch(text, inputs, tmp_path))


# ---- the reference itself -------------------------------------------------------------------------------------------
def test_the_reference_in_chunks_is_the_recurrence():
    g = decays("all", 3)
    a, b, c = (torch.randn((3, 150, d), dtype=F, generator=torch.Generator().manual_seed(d)) for d in (5, 5, 7))
    start = torch.randn((3, 5, 7), dtype=F, generator=torch.Generator().manual_seed(1))
    out, last = ref.recurrence(a, b, c, g, 0.5, 131, start)
    x = ref.walk(a, b, c, g, 0.5, 131, start)
    assert torch.allclose(out, x[0], rtol=1e-12, atol=1e-12) and torch.allclose(last, x[1], rtol=1e-12, atol=1e-12)


def test_the_reference_gradient_is_the_forward_differences():
    case = ("float32", "BSND", 2, 70, 2, 1, 8, 16, "slow", True, "padded")
    t = {n: x.to(F) if x.is_floating_point() else x for n, x in cleaned(make(case), "BSND").items()}
    r = ref.gradient(t["dout"], t["q"], t["k"], t["v"], t["log_decay"], state=t["state"], dstate=t["dstate"], lengths=t["lengths"])

    def loss(**other):
        x = dict(t, **other)
        f = ref.forward(x["q"], x["k"], x["v"], x["log_decay"], state=x["state"], lengths=x["lengths"])
        return float((f["out"] * t["dout"]).sum() + (f["last"] * t["dstate"]).sum())
    for n in ("q", "k", "v", "state"):
        step = torch.randn(t[n].shape, dtype=F, generator=torch.Generator().manual_seed(9))
        slope = (loss(**{n: t[n] + 1e-5 * step}) - loss(**{n: t[n] - 1e-5 * step})) / 2e-5
        assert abs(slope - float((r["d" + n][0] * step).sum())) < 1e-6 * abs(slope) + 1e-6


# ---- as programs use them -------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_gradients_are_the_differences_of_the_result(dtype, tmp_path):
    """The gradient along one direction of every input is the slope of sum(out dout) + sum(last dstate) there."""
    t = make((dtype, "BSND", 2, 150, 4, 2, 32, 48, "slow", True, None))
    text, inputs = describe_grad(t, "BSND")
    got = dict(zip(("q", "k", "v", "state"), launch(text, inputs, tmp_path)))
    exact = ref.gradient(t["dout"], t["q"], t["k"], t["v"], t["log_decay"], state=t["state"], dstate=t["dstate"])
    x = {n: t[n].to(F) for n in t}

    def loss(**other):
        y = dict(x, **other)
        f = ref.forward(y["q"], y["k"], y["v"], y["log_decay"], state=y["state"])
        return float((f["out"] * x["dout"]).sum() + (f["last"] * x["dstate"]).sum())
    for n, g in got.items():
        step = torch.randn(t[n].shape, dtype=F, generator=torch.Generator().manual_seed(9))
        slope = (loss(**{n: x[n] + 1e-4 * step}) - loss(**{n: x[n] - 1e-4 * step})) / 2e-4
        e, rough = exact["d" + n]
        bound = ref.state_bound(rough, 48, 150) if n == "state" else ref.bound(e, rough, dtype, 48, 150)
        assert abs(slope - float((g.to(F) * step).sum())) <= float((bound * step.abs()).sum()) + 1e-6 * abs(slope), n


@pytest.mark.gpu
def test_tokens_after_a_prompt_in_a_pool(tmp_path):
    """A prompt of three sequences leaves its states in entries of a pool; tokens go on from there, in place; what a sequence
    without an entry leaves is nothing, and other entries stay as they were."""
    heads, dim, e, seq = 4, 64, 96, 100
    g = decays("slow", heads)
    pool = normal((6, heads, dim, e), "float32", 1, 2.0)
    slots = torch.tensor([4, 0, 9], dtype=torch.int32)
    parts = [{"q": normal((3, n, heads, dim), "bfloat16", 10 + n), "k": normal((3, n, 2, dim), "bfloat16", 20 + n), "v": normal((3, n, 2, e), "bfloat16", 30 + n)}
             for n in (seq, 1, 3, 400)]
    where = pool.cuda()
    state = pool.to(F)
    for x in parts:
        t = dict(x, log_decay=g, state=pool, slots=slots)
        text, _ = describe(t, "BSND")
        kernel = driver.HipKernel(text, out_dir=str(tmp_path))
        out = empties(kernel)[0]
        kernel.launch([t["q"].cuda(), t["k"].cuda(), t["v"].cuda(), g.cuda(), where, slots.cuda(), out, where])
        before = dict(t, state=state)
        r = check_forward(before, "BSND", [out.cpu()])
        n = t["q"].shape[1]
        after = where.cpu()
        for b in range(2):
            close(after[slots[b]], r["last"][b], ref.state_bound(r["last_rough"][b], dim, n, n > 8), "entry")
        others = [i for i in range(6) if i not in (4, 0)]
        assert torch.equal(after[others], pool[others])
        state = after.to(F)


@pytest.mark.gpu
def test_a_text_in_pieces_is_the_text(tmp_path):
    """Two pieces, the first one's state given to the second in place, against the whole; and their gradients, the second
    piece's for its state given to the first."""
    t = make(("bfloat16", "BSND", 2, 300, 4, 2, 64, 64, "slow", True, None))
    cut = lambda a, b: {n: x[:, a:b].contiguous() if n in ("q", "k", "v", "dout") else x for n, x in t.items()}   # noqa: E731
    first, second = cut(0, 170), cut(170, 300)
    text, inputs = describe(first, "BSND")
    out1, middle = launch(text, inputs, tmp_path)
    second["state"] = middle
    text, inputs = describe(second, "BSND")
    out2, last = launch(text, inputs, tmp_path)
    check_forward(t, "BSND", [torch.cat([out1, out2], 1), last])
    text, inputs = describe_grad(second, "BSND")
    later = launch(text, inputs, tmp_path)
    first["dstate"] = later[3]
    text, inputs = describe_grad(first, "BSND")
    sooner = launch(text, inputs, tmp_path)
    check_gradient(t, "BSND", [torch.cat([a, b], 1) for a, b in zip(sooner[:3], later[:3])] + [sooner[3]])


@pytest.mark.gpu
def test_results_that_nobody_asks_for(tmp_path):
    """One result alone equals what the description with all of them gives, bit for bit."""
    for case in (("bfloat16", "BSND", 2, 70, 4, 2, 64, 96, "slow", True, "padded"), ("float16", "BNSD", 1, 900, 2, 2, 64, 64, "mixed", True, None)):
        t, layout = make(case), case[1]
        text, inputs = describe_grad(t, layout)
        whole = launch(text, inputs, tmp_path)
        for i in range(4):
            text, inputs = describe_grad(t, layout, wanted=[i], name="Fused_LinearGradOnly%d" % i)
            assert torch.equal(launch(text, inputs, tmp_path)[0], whole[i]), i
        text, inputs = describe(t, layout)
        whole = launch(text, inputs, tmp_path)
        for i in range(2):
            text, inputs = describe(t, layout, wanted=[i], name="Fused_LinearOnly%d" % i)
            assert torch.equal(launch(text, inputs, tmp_path)[0], whole[i]), i


def several(tmp_path):
    """(kernel, inputs on the device): few tokens, chunks, segments, gradients, shared heads."""
    jobs = []
    for case in (("bfloat16", "BSND", 2, 1, 4, 2, 64, 64, "slow", True, None), ("float16", "BNSD", 2, 90, 4, 2, 64, 40, "fast", True, "padded"),
                 ("bfloat16", "BSND", 2, 1000, 2, 1, 128, 128, "slow", True, None)):
        t = make(case)
        for f in (describe, describe_grad):
            text, inputs = f(t, case[1])
            jobs.append((driver.HipKernel(text, out_dir=str(tmp_path)), [x.contiguous().cuda() for x in inputs]))
    return jobs


@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream(tmp_path):
    jobs = several(tmp_path)
    static = [([torch.nan_to_num(x) if x.is_floating_point() else x.clone() for x in ins], empties(k)) for k, ins in jobs]
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
def test_without_allocations_and_at_odd_addresses(tmp_path):
    for k, ins in several(tmp_path):
        k.prepare()
        first, second = empties(k), empties(k)
        k.launch(ins + first)
        k.launch_static_scratch_ptrs([x.data_ptr() for x in ins + second], torch.cuda.current_stream().cuda_stream)
        moved = [at_odd_address(o) for o in second]
        for m in moved:
            m.fill_(0)
        k.launch([at_odd_address(x) for x in ins] + moved)
        torch.cuda.synchronize()
        for a, o, m in zip(first, second, moved):
            assert torch.equal(a.view(torch.uint8), o.view(torch.uint8)) and torch.equal(a, m), k.kernel_name


@pytest.mark.gpu
@pytest.mark.parametrize("seq", [2048, 3500])
def test_fewer_segments_without_allocations(seq, tmp_path):
    """A gradient whose heads' own gradients (4 KiB a token) and states in front of segments take almost, or more than, 16 MiB."""
    t = make(("bfloat16", "BSND", 1, seq, 4, 2, 128, 128, "slow", False, "padded"))
    text, inputs = describe_grad(t, "BSND")
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    assert kernel.workspace_bytes > seq * 4096 and ("_within" in kernel.source) == (kernel.workspace_bytes > 16 << 20)
    assert seq == 2048 or "_within" in kernel.source
    kernel.prepare()
    ins, outs = [x.cuda() for x in inputs], empties(kernel)
    kernel.launch_static_scratch_ptrs([x.data_ptr() for x in ins + outs], torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    check_gradient(t, "BSND", [o.cpu() for o in outs])


@pytest.mark.gpu
def test_open_extents(tmp_path):
    """One description for any number of tokens: the results of the static ones, and one code object for lengths that need
    the same kernel."""
    def text_of(seq, name):
        b = builder(name)
        x = [b.input([2, seq, h, 64], "bfloat16") for h in (4, 2, 2)]
        return b.dumps(op_desc.linear_attention(b, *x, b.input([4], "float32"), last_state=True))
    dyn = driver.HipDynamicKernel(open_extent(text_of(7919, "Fused_OpenLinear"), (7919,)), out_dir=str(tmp_path))
    seen = []
    for seq in (65, 190, 1, 4000, 5000):
        ins = [normal((2, seq, h, 64), "bfloat16", 40 + i).cuda() for i, h in enumerate((4, 2, 2))] + [decays("slow", 4).cuda()]
        static = driver.HipKernel(text_of(seq, "Fused_StaticLinear"), out_dir=str(tmp_path))
        expect, got = empties(static), empties(static)
        static.launch(ins + expect)
        used = dyn.launch_packed([x.data_ptr() for x in ins + got], [list(x.shape) for x in ins + got], torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for a, o in zip(expect, got):
            assert torch.equal(a, o)
        seen.append(used.source)
    assert seen[0] == seen[1] != seen[2] and seen[3] == seen[4] != seen[0]


@pytest.mark.gpu
def test_tokens_behind_32_bit_offsets(tmp_path):
    """2.2 GB each of queries, keys, values and results: the last head's tokens near the end, which have forgotten the rest."""
    seq, heads, dim = 70001, 128, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((1, seq, heads, dim), generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    decay = torch.full((heads,), -0.5)
    b = builder("Fused_LongLinear")
    kernel = driver.HipKernel(b.dumps(op_desc.linear_attention(b, given(b, q), given(b, k), given(b, v), given(b, decay), last_state=True)), out_dir=str(tmp_path))
    outs = empties(kernel)
    kernel.launch([q, k, v, decay.cuda()] + outs)
    torch.cuda.synchronize()
    part = [x[:, -300:, -2:].cpu() for x in (q, k, v)]
    r = ref.forward(*part, decay[-2:])
    at = slice(200, None)   # (behind 200 tokens that decay by e^-100)
    close(outs[0][:, -100:, -2:].cpu(), r["out"][:, at], ref.bound(r["out"][:, at], [x[:, at] for x in r["rough"]], "bfloat16", dim, seq), "out")
    close(outs[1][:, -2:].cpu(), r["last"], ref.state_bound(r["last_rough"], dim, seq), "last state")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_a_training_layer(dtype, tmp_path):
    """Positions of three axes, linear attention, its gradient, positions turned back: one description, every tensor between
    them checked from what stands in front of it."""
    batch, seq, heads, kv, dim, sections = 2, 150, 4, 2, 64, [8, 12, 12]
    t = {"q": normal((batch, seq, heads, dim), dtype, 1), "k": normal((batch, seq, kv, dim), dtype, 2), "v": normal((batch, seq, kv, dim), dtype, 3),
         "dout": normal((batch, seq, heads, dim), dtype, 4), "log_decay": decays("slow", heads)}
    at = torch.arange(seq)
    t["positions"] = torch.stack([at // 25, at // 5 % 5, at % 5]).to(torch.int32)
    t["lengths"] = torch.tensor([seq, 90], dtype=torch.int32)
    b = builder("Fused_LinearLayer")
    order = ("q", "k", "v", "dout", "positions", "log_decay", "lengths")
    g = {n: given(b, t[n]) for n in order}
    turn = dict(sections=sections, axis_order="cycle")
    turned = op_desc.rotary_embedding(b, [g["q"], g["k"]], g["positions"], **turn)
    out, last = op_desc.linear_attention(b, *turned, g["v"], g["log_decay"], lengths=g["lengths"], last_state=True)
    dq, dk, dv = op_desc.linear_attention_grad(b, g["dout"], *turned, g["v"], g["log_decay"], lengths=g["lengths"])
    again = op_desc.rotary_embedding(b, [dq, dk], g["positions"], inverse=True, **turn)
    got = launch(b.dumps(turned + [out, last, dq, dk, dv] + again), [t[n] for n in order], tmp_path)
    u = ref.half_step(dtype)
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0

    def turns(x, y, inverse):
        exact = ref.rotary_axes(x, t["positions"][:, None], sections, "cycle", "shared", 10000.0, inverse=inverse)
        close(y, exact, u * exact.abs() * 1.01 + 2.0 ** -19 * float(x.abs().max()) + tiny, "turned")
    turns(t["q"], got[0], False)
    turns(t["k"], got[1], False)
    x = dict(t, q=got[0], k=got[1])
    check_forward(x, "BSND", got[2:4])
    check_gradient(x, "BSND", got[4:7])
    turns(got[4], got[7], True)
    turns(got[5], got[8], True)


@pytest.mark.gpu
def test_elementwise_ops_around(tmp_path):
    x = normal((2, 40, 4, 64), "bfloat16", 6)
    g = decays("slow", 4)
    b = builder("Fused_ScaledLinear")
    i, d = given(b, x), given(b, g)
    half = b.mul(i, b.const(0.5, "bfloat16"))
    out = op_desc.linear_attention(b, half, i, i, d)[0]
    got = launch(b.dumps([b.add(out, i)]), [x, g], tmp_path)
    r = ref.forward((x.float() * 0.5).to(torch.bfloat16), x, x, g)
    u = ref.half_step("bfloat16")
    exact = r["out"] + x.double()
    close(got[0], exact, ref.bound(r["out"], r["rough"], "bfloat16", 64, 40) * (1 + u) + u * exact.abs() * 1.01, "sum")


@pytest.mark.gpu
@pytest.mark.parametrize("seq", [3, 100])
def test_large_and_small_values_in_float16(seq, tmp_path):
    """States beyond float16's range with results inside it, beside heads of very small ones."""
    t = make(("float16", "BSND", 1, seq, 2, 2, 32, 32, "none", True, None))
    t["k"] = (t["k"].float() * torch.tensor([600.0, 1e-4])[:, None]).to(torch.float16)
    t["v"] = (t["v"].float() * torch.tensor([2000.0, 3.0])[:, None]).to(torch.float16)
    t["q"] = (t["q"].float() * torch.tensor([3e-5, 200.0])[:, None]).to(torch.float16)
    t["state"] = t["state"] * torch.tensor([1e6, 1e-4])[:, None, None]
    text, inputs = describe(t, "BSND")
    check_forward(t, "BSND", launch(text, inputs, tmp_path))
    if seq > 8:
        text, inputs = describe_grad(t, "BSND")
        t["dout"] = (t["dout"].float() * torch.tensor([1e-4, 100.0])[:, None]).to(torch.float16)
        text, inputs = describe_grad(t, "BSND")
        got = launch(text, inputs, tmp_path)
        keep = [torch.isfinite(x).all() for x in got]
        r = ref.gradient(t["dout"], t["q"], t["k"], t["v"], t["log_decay"], state=t["state"], dstate=t["dstate"])
        for n, x, ok in zip(("dq", "dk", "dv", "dstate"), got, keep):
            exact, rough = r[n]
            fits = exact.abs() < (65000.0 if n != "dstate" else 1e38)
            bound = ref.state_bound(rough, 32, seq) if n == "dstate" else ref.bound(exact, rough, "float16", 32, seq)
            assert ((x.to(F) - exact).abs() <= bound)[fits].all(), n


@pytest.mark.gpu
def test_long_texts_in_a_pool_in_place(tmp_path):
    """Segments, entries of a pool read and written in place: one of them whole, one sequence without an entry, one without
    tokens, whose entry stays as it was, bit for bit, as do those that no sequence has."""
    heads, dim, seq = 2, 64, 3000
    g, pool = decays("slow", heads), normal((5, heads, dim, dim), "float32", 1, 2.0)
    t = {n: normal((3, seq, heads, dim), "bfloat16", 2 + i) for i, n in enumerate(("q", "k", "v"))}
    t = dict(t, log_decay=g, state=pool, slots=torch.tensor([3, -1, 0], dtype=torch.int32), lengths=torch.tensor([seq, 50, 0], dtype=torch.int32))
    text, inputs = describe(t, "BSND", scale=0.25)
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    assert kernel.workspace_bytes > 0
    ins = [x.cuda() for x in inputs]
    out = empties(kernel)[0]
    kernel.launch(ins + [out, ins[4]])
    r = check_forward(t, "BSND", [out.cpu()], scale=0.25)
    after = ins[4].cpu()
    close(after[3], r["last"][0], ref.state_bound(r["last_rough"][0], dim, seq), "entry")
    others = [0, 1, 2, 4]
    assert torch.equal(after[others], pool[others])


@pytest.mark.gpu
@pytest.mark.parametrize("seq,joined", [(700, True), (6000, False)])
def test_the_last_state_over_the_one_given_beside_other_work(seq, joined, tmp_path):
    """Several segments, whose workgroups other work on the card keeps from starting together: in place as apart, bit for bit."""
    heads, dim = 4, 64
    t = dict({n: normal((2, seq, heads, dim), "bfloat16", 2 + i) for i, n in enumerate(("q", "k", "v"))}, log_decay=decays("slow", heads),
             state=normal((2, heads, dim, dim), "float32", 1, 2.0))
    text, inputs = describe(t, "BSND")
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    assert kernel.workspace_bytes > 0 and ("_starts" not in kernel.source) == joined
    kernel.prepare()
    ins, apart = [x.cuda() for x in inputs], empties(kernel)
    kernel.launch(ins + apart)
    torch.cuda.synchronize()
    check_forward(t, "BSND", [x.cpu() for x in apart])
    side, a = torch.cuda.Stream(), torch.randn(2048, 2048, device="cuda")
    for _ in range(6):
        with torch.cuda.stream(side):
            for _ in range(4):
                a @ a
        out, where = torch.empty_like(apart[0]), ins[4].clone()
        kernel.launch(ins[:4] + [where] + [out, where])
        torch.cuda.synchronize()
        assert torch.equal(out, apart[0]) and torch.equal(where, apart[1])


@pytest.mark.gpu
@pytest.mark.parametrize("seq", [2, 150, 2000])
def test_one_entry_read_by_several_sequences(seq, tmp_path):
    """A prefix that sequences share: the same entry for all of them, and none left behind."""
    heads, dim = 2, 64
    g, pool = decays("mixed", heads), normal((3, heads, dim, dim), "float32", 1, 2.0)
    t = dict({n: normal((3, seq, heads, dim), "bfloat16", 2 + i) for i, n in enumerate(("q", "k", "v"))}, log_decay=g)
    text, inputs = describe(dict(t, state=pool, slots=torch.tensor([1, 1, 1], dtype=torch.int32)), "BSND", last=False, name="Fused_SharedEntry")
    shared = launch(text, inputs, tmp_path)[0]
    text, inputs = describe(dict(t, state=pool[1:2].expand(3, -1, -1, -1).contiguous()), "BSND", last=False, name="Fused_OwnState")
    assert torch.equal(shared, launch(text, inputs, tmp_path)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("seq", [70, 1600])
@pytest.mark.parametrize("given_", ["state", "dstate"])
def test_gradient_with_one_of_the_states(seq, given_, tmp_path):
    t = make(("bfloat16", "BSND", 2, seq, 4, 2, 64, 40, "slow", True, "padded"))
    del t["state" if given_ == "dstate" else "dstate"]
    text, inputs = describe_grad(t, "BSND", scale=0.5)
    got = launch(text, inputs, tmp_path)
    assert len(got) == (4 if given_ == "state" else 3)
    check_gradient(t, "BSND", got, scale=0.5)


@pytest.mark.gpu
def test_one_handle_on_two_streams(tmp_path):
    """Launches of one handle with a workspace that overlap on two streams: each has the results it has alone."""
    t = make(("bfloat16", "BSND", 2, 1500, 2, 1, 128, 128, "slow", True, None))
    for f in (describe, describe_grad):
        text, inputs = f(t, "BSND")
        kernel = driver.HipKernel(text, out_dir=str(tmp_path))
        assert kernel.workspace_bytes > 0
        kernel.prepare()
        sets = [[x.cuda() for x in inputs], [x.cuda() * (0.5 if x.is_floating_point() and x.dim() == 4 else 1) for x in inputs]]
        alone, both = [empties(kernel) for _ in sets], [empties(kernel) for _ in sets]
        for ins, outs in zip(sets, alone):
            kernel.launch(ins + outs)
            torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(5):
            for stream, ins, outs in zip(streams, sets, both):
                with torch.cuda.stream(stream):
                    kernel.launch(ins + outs)
        torch.cuda.synchronize()
        for a, o in zip(alone, both):
            assert all(torch.equal(x, y) for x, y in zip(a, o))


@pytest.mark.gpu
@pytest.mark.parametrize("seq,at,kept", [(6, 3, 3), (300, 200, 128), (2500, 1700, 1664)])
def test_values_that_are_not_finite_stay_in_their_head(seq, at, kept, tmp_path):
    """Infinity and NaN in one head of one sequence: every other head and sequence has its results, bit for bit, and so have the
    head's own tokens in front of the chunk (of few tokens: in front of the token)."""
    t = make(("bfloat16", "BSND", 2, seq, 4, 4, 64, 64, "slow", True, None))
    text, inputs = describe(t, "BSND")
    clean = launch(text, inputs, tmp_path)
    for n, x in (("v", math.inf), ("k", math.nan)):
        t[n][1, at, 2, 5] = x
    text, inputs = describe(t, "BSND")
    got = launch(text, inputs, tmp_path)
    for a, o in zip(clean, got):
        assert torch.equal(a[0], o[0])
    for h in (0, 1, 3):
        assert torch.equal(clean[0][1, :, h], got[0][1, :, h]) and torch.equal(clean[1][1, h], got[1][1, h])
    assert torch.equal(clean[0][1, :kept, 2], got[0][1, :kept, 2]) and torch.isnan(got[0][1, at:, 2]).all()


# ---- what is refused ------------------------------------------------------------------------------------------------
def text_of(dtype="bfloat16", q=(2, 9, 4, 64), k=(2, 9, 2, 64), v=(2, 9, 2, 32), decay=([4], "float32"), state=None, slots=None, lengths=None, grad=False, dout=None,
            dstate=None, **options):
    b = builder()
    ins = [b.input(list(s), dtype) for s in (q, k, v)] + [b.input(*decay)]
    more = {n: b.input(*s) for n, s in (("state", state), ("slots", slots), ("lengths", lengths), ("dstate", dstate)) if s is not None}
    if grad:
        return b.dumps(op_desc.linear_attention_grad(b, b.input(list(dout or (2, 9, 4, 32)), dtype), *ins, **more, **options))
    return b.dumps(op_desc.linear_attention(b, *ins, **more, **options))


def test_refusals():
    driver.translate(text_of())
    driver.translate(text_of(grad=True))
    state = ([2, 4, 64, 32], "float32")
    driver.translate(text_of(state=state, slots=([2], "int32"), lengths=([2], "int32"), last_state=True))
    driver.translate(text_of(state=([7, 4, 64, 32], "float32"), slots=([2], "int32"), last_state=True))
    driver.translate(text_of(grad=True, state=state, dstate=state, lengths=([2], "int32")))
    refused(text_of(dtype="float32"), -3, "float16 or bfloat16")
    refused(text_of(k=(2, 8, 2, 64)), -3, "batch or sequence")
    refused(text_of(v=(3, 9, 2, 32)), -3, "batch or sequence")
    refused(text_of(k=(2, 9, 3, 64), v=(2, 9, 3, 32)), -3, "multiple of them")
    refused(text_of(v=(2, 9, 4, 32)), -3, "same heads")
    refused(text_of(k=(2, 9, 2, 32)), -3, "channels")
    refused(text_of(decay=([2], "float32")), -3, "log_decay")
    refused(text_of(decay=([4], "float16")), -3, "log_decay")
    refused(text_of(state=([3, 4, 64, 32], "float32")), -3, "states must be")
    refused(text_of(state=([2, 4, 32, 64], "float32")), -3, "states must be")
    refused(text_of(state=([2, 4, 64, 32], "bfloat16")), -3, "float32")
    refused(text_of(slots=([2], "int32")), -3, "slots")
    refused(text_of(state=state, slots=([3], "int32")), -3, "slots")
    refused(text_of(state=state, slots=([2], "int64")), -3, "slots")
    refused(text_of(lengths=([3], "int32")), -3, "lengths")
    refused(text_of(scale=0.0), -3, "scale")
    refused(text_of(layout="SBND"), -3, "layout")
    refused(text_of(grad=True, dout=(2, 9, 4, 64)), -3, "shape of the result")
    refused(text_of(grad=True, dout=(2, 8, 4, 32)), -3, "shape of the result")
    refused(text_of(grad=True, dstate=([2, 4, 64, 64], "float32")), -3, "gradient must be")
    for channels in (12, 264):
        refused(text_of(q=(2, 9, 4, channels), k=(2, 9, 2, channels)), -4, "multiple of 8")
        refused(text_of(v=(2, 9, 2, channels)), -4, "multiple of 8")
    refused(text_of(q=(1, 9, 1 << 17, 128), k=(1, 9, 1, 128), v=(1, 9, 1, 8), decay=([1 << 17], "float32")), -4, "2 GiB")
    refused(text_of(q=(1 << 20, 9, 64, 8), k=(1 << 20, 9, 64, 8), v=(1 << 20, 9, 64, 8), decay=([64], "float32")), -4, "more threads")
    doc = json.loads(text_of())
    doc["op_desc"][0]["output_desc"][0]["shape"][3] = 64
    refused(json.dumps(doc), -3, "does not follow")


def test_bytes_count_the_entries_of_a_pool_that_sequences_have(tmp_path):
    def moved(entries, **options):
        text = text_of(state=([entries, 4, 64, 32], "float32"), slots=([2], "int32"), **options)
        return driver.HipKernel(text, out_dir=str(tmp_path)).algorithmic_bytes
    for last in (False, True):
        assert moved(2, last_state=last) == moved(70, last_state=last)
    assert moved(2, last_state=True) - moved(2) == 4 * 2 * 4 * 64 * 32


def test_long_texts_of_few_heads_are_cut_into_segments(tmp_path):
    def kernel(seq, batch=1, **options):
        return driver.HipKernel(text_of(q=(batch, seq, 4, 64), k=(batch, seq, 4, 64), v=(batch, seq, 4, 64), **options), out_dir=str(tmp_path))
    assert kernel(8192).workspace_bytes > 0 and kernel(200).workspace_bytes == 0
    assert "linear::tokens" in kernel(8).source and "linear::walk" in kernel(9).source
    a, b = kernel(4096), kernel(5000)
    assert a.family == "linear_attention" and a.source == b.source and b.cache_hit
