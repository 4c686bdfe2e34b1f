"""Pools of states: several ops of one description over one pool, launches without allocations in place, descriptions of any number of
entries, pools behind 32-bit offsets."""
import pytest
import torch

import linear_reference as ref
from akg_amd import driver, op_desc
from dynamic_cases import open_extent
from test_attention_ops import builder, close, given, normal, refused
from test_attention_use import empties
from test_linear_attention import decays, describe

F = torch.float64


def steps(pool_is_a_result, other_slots=False):
    """A prompt and a drafted step behind it over one pool."""
    b = builder("Fused_TwoSteps")
    x = [[b.input([2, n, 2, 64], "bfloat16") for _ in range(3)] for n in (70, 3)]
    g, pool, slots = b.input([2], "float32"), b.input([5, 2, 64, 64], "float32"), b.input([2], "int32")
    out1, pool1 = op_desc.linear_attention(b, *x[0], g, state=pool, slots=slots, last_state=True)
    out2, pool2 = op_desc.linear_attention(b, *x[1], g, state=pool1, slots=b.input([2], "int32") if other_slots else slots, last_state=True)
    return b.dumps([out1] + [pool1] * pool_is_a_result + [out2, pool2])


def test_a_pool_between_two_ops_is_a_result():
    driver.translate(steps(True))
    driver.translate(steps(True, True))
    refused(steps(False), -3, "has to be a result")
    refused(steps(False, True), -3, "has to be a result")
    b = builder()
    x = [b.input([2, 9, 2, 64], "bfloat16") for _ in range(3)]
    out, pool = op_desc.linear_attention(b, *x, b.input([2], "float32"), state=b.input([5, 2, 64, 64], "float32"), slots=b.input([2], "int32"), last_state=True)
    refused(b.dumps([out, b.mul(pool, b.const(0.5, "float32"))]), -3, "has to be a result")


@pytest.mark.gpu
def test_two_steps_over_one_pool_in_one_description(tmp_path):
    g, pool = decays("slow", 2), normal((5, 2, 64, 64), "float32", 1, 2.0)
    x = [[normal((2, n, 2, 64), "bfloat16", 10 * n + i) for i in range(3)] for n in (70, 3)]
    slots = [torch.tensor([3, 1], dtype=torch.int32), torch.tensor([1, 4], dtype=torch.int32)]
    kernel = driver.HipKernel(steps(True, True), out_dir=str(tmp_path))
    where = pool.cuda()
    outs = empties(kernel)
    order = [t.cuda() for t in x[0] + x[1]] + [g.cuda(), where, slots[0].cuda(), slots[1].cuda()]
    kernel.launch(order + [outs[0], where, outs[2], where])
    torch.cuda.synchronize()
    state = pool.to(F)
    for n, (a, s, got) in enumerate(zip(x, slots, (outs[0], outs[2]))):
        r = ref.forward(*a, g, state=state, slots=s)
        bound = ref.bound(r["out"], r["rough"], "bfloat16", 64, 70)
        if n:   # (the state that it starts from is off by what the first step's may be)
            bound = bound + ref.state_bound(size, 64, 70).amax() * a[0].to(F).abs().sum(-1, keepdim=True) * 64 ** -0.5
        close(got.cpu(), r["out"], bound, "out")
        size = r["last_rough"]
        for b in range(2):
            state[int(s[b])] = r["last"][b]
    after = where.cpu()
    for i in (0, 2):
        assert torch.equal(after[i], pool[i])
    for i in (1, 3, 4):
        assert ((after[i].to(F) - state[i]).abs() <= ref.state_bound(size.amax() + state[i].abs(), 64, 80)).all(), i


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 100, 1500, 6000])
def test_in_place_without_allocations(tokens, tmp_path):
    """As apart, bit for bit (with the launches that need no more than the library's own scratch: against themselves)."""
    heads, dim = 2, 64
    t = dict({n: normal((3, tokens, heads, dim), "bfloat16", 2 + i) for i, n in enumerate(("q", "k", "v"))}, log_decay=decays("slow", heads),
             state=normal((6, heads, dim, dim), "float32", 1, 2.0), slots=torch.tensor([5, 0, 7], dtype=torch.int32),
             lengths=torch.tensor([tokens, tokens // 2, tokens], dtype=torch.int32))
    text, inputs = describe(t, "BSND")
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    kernel.prepare()
    ins, stream = [x.cuda() for x in inputs], torch.cuda.current_stream().cuda_stream
    apart = empties(kernel)
    apart[1].copy_(ins[4])
    kernel.launch_static_scratch_ptrs([x.data_ptr() for x in ins + apart], stream)
    out, where = torch.empty_like(apart[0]), ins[4].clone()
    kernel.launch_static_scratch_ptrs([x.data_ptr() for x in ins[:4] + [where] + ins[5:] + [out, where]], stream)
    torch.cuda.synchronize()
    assert torch.equal(out, apart[0]) and torch.equal(where, apart[1])
    others = [1, 2, 3, 4]
    assert torch.equal(where[others].cpu(), t["state"][others]) and not torch.equal(where[5].cpu(), t["state"][5])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 40])
def test_descriptions_of_any_number_of_entries(tokens, tmp_path):
    """An open number of entries: the results of the static description, one code object for two of them."""
    def text_of(entries, name):
        b = builder(name)
        x = [b.input([2, tokens, 2, 64], "bfloat16") for _ in range(3)]
        return b.dumps(op_desc.linear_attention(b, *x, b.input([2], "float32"), state=b.input([entries, 2, 64, 64], "float32"), slots=b.input([2], "int32"), last_state=True))
    dyn = driver.HipDynamicKernel(open_extent(text_of(7919, "Fused_OpenPool"), (7919,)), out_dir=str(tmp_path))
    sources = []
    for entries in (3, 11):
        ins = [normal((2, tokens, 2, 64), "bfloat16", 4 + i).cuda() for i in range(3)] + [decays("slow", 2).cuda(), normal((entries, 2, 64, 64), "float32", 9).cuda(),
               torch.tensor([entries - 1, entries], dtype=torch.int32).cuda()]
        static = driver.HipKernel(text_of(entries, "Fused_StaticPool"), out_dir=str(tmp_path))
        expect, got = empties(static), empties(static)
        for o in (expect, got):
            o[1].zero_()
        static.launch(ins + expect)
        used = dyn.launch_packed([x.data_ptr() for x in ins + got], [list(x.shape) for x in ins + got], torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, o) for a, o in zip(expect, got))
        sources.append(used.source)
    assert sources[0] == sources[1]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 70, 1500])
def test_entries_behind_32_bit_offsets(tokens, tmp_path):
    """A pool of 5.2 GB, in place, of which the last entries are read and left."""
    heads, dim, entries = 2, 128, 40000
    pool = torch.zeros((entries, heads, dim, dim), device="cuda")
    first = normal((2, heads, dim, dim), "float32", 1, 2.0)
    slots = torch.tensor([entries - 1, 33333], dtype=torch.int32)
    for s, x in zip(slots.tolist(), first):
        pool[s] = x.cuda()
    t = dict({n: normal((2, tokens, heads, dim), "bfloat16", 2 + i) for i, n in enumerate(("q", "k", "v"))}, log_decay=decays("slow", heads))
    b = builder("Fused_LargePool")
    ins = [t[n] for n in ("q", "k", "v", "log_decay")]
    d = [given(b, x) for x in ins]
    kernel = driver.HipKernel(b.dumps(op_desc.linear_attention(b, *d, state=b.input([entries, heads, dim, dim], "float32"), slots=b.input([2], "int32"), last_state=True)),
                              out_dir=str(tmp_path))
    out = torch.empty((2, tokens, heads, dim), dtype=torch.bfloat16, device="cuda")
    kernel.launch([x.cuda() for x in ins] + [pool, slots.cuda(), out, pool])
    torch.cuda.synchronize()
    r = ref.forward(t["q"], t["k"], t["v"], t["log_decay"], state=first)
    close(out.cpu(), r["out"], ref.bound(r["out"], r["rough"], "bfloat16", dim, tokens), "out")
    for s, e, size in zip(slots.tolist(), r["last"], r["last_rough"]):
        close(pool[s].cpu(), e, ref.state_bound(size, dim, tokens, tokens > 8), "entry")
        pool[s] = 0
    assert not pool.any()
