"""float16 gradients of attention over the range of float16: gradients of scores beyond 65504 where dq, dk and dv fit, and
probabilities of some 10^5 keys, far below float16's normal numbers."""
import math

import pytest
import torch

import attention_reference as ref
from akg_amd import op_desc
from test_attention_ops import attention_case, behind_lengths, builder, close, given, launch, normal

MOST = 65504.0

# case as in the tests of the operators, standard deviation of dout, of the values, of the queries
LARGE = [
    (("float16", "BSND", 1, 32, 32, 1, 1, 64, 64, False, None, None), 16384.0, 1.0, 2.0),
    (("float16", "BSND", 1, 300, 300, 2, 2, 128, 128, True, None, None), 580.0, 16.0, 2.0),
    (("float16", "BNSD", 1, 300, 300, 2, 1, 128, 128, True, None, None), 6400.0, 2.0, 1.0),
    (("float16", "BSND", 2, 77, 90, 4, 2, 64, 40, False, "float32", "padded"), 4000.0, 6.0, 1.0),
    (("float16", "BSND", 1, 600, 600, 8, 2, 64, 64, True, None, "padded"), 4000.0, 3.0, 1.0),      # rows of dk and dv in ranges
    (("float16", "BNSD", 2, 65, 130, 2, 2, 192, 256, False, "bool", None), 500.0, 24.0, 1.0),        # dk and dv by workgroups of their own
    (("float16", "BSND", 1, 700, 700, 40, 40, 64, 64, True, None, None), 2400.0, 6.0, 1.0),        # dq in a launch of its own
]


def large_case(case, dout_size, v_size, q_size):
    t, extra, options, m, ql, kl = attention_case(case)
    t["q"] = (t["q"].float() * (q_size / 2.0)).to(torch.float16)
    t["v"] = (t["v"].float() * v_size).to(torch.float16)
    r = ref.forward(t["q"], t["k"], t["v"], mask=m, qlens=ql, klens=kl, **options)
    dout = (normal(r["out"].shape, "float32", 8) * dout_size).clamp(-60000.0, 60000.0).to(torch.float16)
    return t, extra, options, m, ql, kl, dout, r["out"].to(torch.float16), r["lse"].float()


def largest_score_gradient(t, options, m, ql, kl, dout, out):
    """max |p (dp - delta)| in float64."""
    layout = options["layout"]
    dout, out = (ref.heads_of(behind_lengths(x, ql, layout, 0.0), layout) for x in (dout, out))
    q = ref.heads_of(t["q"], layout)
    k, v = (ref.used_keys(ref.heads_of(t[n], layout), kl).repeat_interleave(q.shape[1] // ref.heads_of(t["k"], layout).shape[1], 1) for n in "kv")
    p, _, _ = ref.probabilities(q, k, 1 / math.sqrt(q.shape[3]), options["causal"], m, ql, kl)
    return float((p * (dout @ v.transpose(2, 3) - (dout * out).sum(-1, keepdim=True))).abs().max())


def range_bounds(exact, t, dout, out, options, size, sq, sk):
    """As ref.gradient_bound, but for the steps of the smallest float16. A row's gradients of scores are at most B = sum |dout| max
    |v| + |delta|, computed times a power of two that puts B into [2^13, 2^14) (dk: the largest row of a key head): steps of
    2^-24 there are off by at most 2^-25 2^-13 B = 2^-38 B. Probabilities times 2^13 are off by 2^-38. float32 sums over n
    positions, sixteen at a time: (n / 16 + 16) 2^-24 of the sizes added."""
    layout = options["layout"]
    g, o = ref.heads_of(dout, layout).abs(), ref.heads_of(out, layout)
    v, k = ref.heads_of(t["v"], layout).abs(), ref.heads_of(t["k"], layout).abs()
    hkv = k.shape[1]
    group = g.shape[1] // hkv
    top_v = v.amax((2, 3)).repeat_interleave(group, 1)[:, :, None, None]
    b = g.sum(-1, keepdim=True) * top_v + (g * o.abs()).sum(-1, keepdim=True)
    top_b = b.view(b.shape[0], hkv, group, -1).amax((2, 3))[:, :, None, None]
    scale = 1 / math.sqrt(k.shape[3])
    sum_k = k.sum(2, keepdim=True).repeat_interleave(group, 1)
    sum_q = ref.heads_of(t["q"], layout).abs().view(b.shape[0], hkv, group, sq, -1).sum((2, 3))[:, :, None]
    sum_g = g.view(b.shape[0], hkv, group, sq, -1).sum((2, 3))[:, :, None]
    steps = {"dq": b * sum_k * scale, "dk": (top_b * sum_q * scale).expand(-1, -1, sk, -1), "dv": sum_g.expand(-1, -1, sk, -1)}
    u = ref.half_step("float16")
    noise = 2.0 ** -23 * (k.shape[3] + 8) * (size + 2)
    long = {"dq": sk, "dk": sq * group, "dv": sq * group}
    return {n: 1.01 * (u * e["sum"] + noise * e["rough"] + u * e["exact"].abs() + 2.0 ** -38 * ref.back(steps[n], layout)
                       + 2.0 ** -24 * (long[n] / 16 + 16) * e["sum"]) + 2.0 ** -25 for n, e in exact.items()}


def check(t, extra, options, m, ql, kl, dout, out, lse, tmp_path):
    layout = options["layout"]
    named = {"dout": dout, **t, "out": out, "lse": lse}
    for n, lengths in (("dout", ql), ("q", ql), ("out", ql), ("k", kl), ("v", kl)):
        named[n] = behind_lengths(named[n], lengths, layout, math.nan)
    order = ("dout", "q", "k", "v", "out", "lse")
    b = builder()
    more = [given(b, named[n]) for n in order]
    grads = op_desc.attention_grad(b, *more, **{n: given(b, x) for n, x in extra.items()}, **options)
    got = launch(b.dumps(grads), [named[n] for n in order] + list(extra.values()), tmp_path)
    clean = {n: behind_lengths(x, {"q": ql, "k": kl, "v": kl}[n], layout, 0.0) for n, x in t.items()}
    dout, out = (behind_lengths(x, ql, layout, 0.0) for x in (dout, out))
    exact, size = ref.gradient(dout, clean["q"], clean["k"], clean["v"], out, lse, mask=m, qlens=ql, klens=kl, **options)
    seq = 1 if layout == "BSND" else 2
    bounds = range_bounds(exact, clean, dout, out, options, size, t["q"].shape[seq], t["k"].shape[seq])
    for n, x in zip(("dq", "dk", "dv"), got):
        assert float(exact[n]["exact"].abs().max()) < MOST - 500
        close(x, exact[n]["exact"], bounds[n], n)


@pytest.mark.parametrize("large", LARGE, ids=lambda x: "-".join(str(y) for y in x[0]) + "-%g-%g-%g" % x[1:])
def test_the_scores_gradients_of_these_leave_float16(large):
    t, extra, options, m, ql, kl, dout, out, lse = large_case(*large)
    assert largest_score_gradient(t, options, m, ql, kl, dout, out) > MOST
    exact, _ = ref.gradient(dout, t["q"], t["k"], t["v"], out, lse, mask=m, qlens=ql, klens=kl, **options)
    assert max(float(e["exact"].abs().max()) for e in exact.values()) < MOST - 500


@pytest.mark.gpu
@pytest.mark.parametrize("large", LARGE, ids=lambda x: "-".join(str(y) for y in x[0]) + "-%g-%g-%g" % x[1:])
def test_float16_gradients_of_a_large_loss(large, tmp_path):
    check(*large_case(*large), tmp_path)


@pytest.mark.gpu
@pytest.mark.parametrize("dout_size", [2.0 ** -10, 2.0 ** 12])
def test_float16_gradients_over_many_keys(dout_size, tmp_path):
    """One query of nearly equal probabilities, 56.5 steps of 2^-24 each."""
    keys = 296941
    case = ("float16", "BSND", 1, 1, keys, 1, 1, 64, 64, False, None, None)
    check(*large_case(case, dout_size, 1.0, 2.0 ** -5), tmp_path)


@pytest.mark.gpu
@pytest.mark.parametrize("layout,seq,heads,hkv,dim,lengths", [("BSND", 600, 1, 1, 64, None), ("BNSD", 700, 4, 4, 128, [640]), ("BSND", 520, 40, 40, 64, None),
                                                              ("BNSD", 520, 2, 2, 192, None)])
def test_float16_gradients_of_keys_that_the_large_rows_do_not_see(layout, seq, heads, hkv, dim, lengths, tmp_path):
    """The first 64 queries have gradients of some 2^13, the others of 2^-10. Keys from 128 on are seen by the others alone and keep the
    digits of what those leave: dk there is bounded by the rows from 64 below the key's tile of 128 on."""
    case = ("float16", layout, 1, seq, seq, heads, hkv, dim, dim, True, None, None)
    t, _, options, _, _, _ = attention_case(case)
    extra, ql, kl = {}, lengths, lengths
    if lengths:
        extra = {n: torch.tensor(lengths, dtype=torch.int32) for n in ("query_lengths", "key_lengths")}
    r = ref.forward(t["q"], t["k"], t["v"], qlens=ql, klens=kl, **options)
    dout = ref.heads_of(normal(r["out"].shape, "float32", 8), layout)
    dout[:, :, :64] *= 2.0 ** 13
    dout[:, :, 64:] *= 2.0 ** -10
    dout = ref.back(dout, layout).contiguous().to(torch.float16)
    tensors = [dout, t["q"], t["k"], t["v"], r["out"].to(torch.float16), r["lse"].float()]
    b = builder()
    grads = op_desc.attention_grad(b, *[given(b, x) for x in tensors], **{n: given(b, x) for n, x in extra.items()}, **options)
    got = launch(b.dumps(grads), [x.contiguous() for x in tensors] + list(extra.values()), tmp_path)
    exact, size = ref.gradient(*tensors, qlens=ql, klens=kl, **options)
    clean = {n: behind_lengths(x, lengths, layout, 0.0) for n, x in t.items()}
    dout, out = (behind_lengths(x, lengths, layout, 0.0) for x in (dout, r["out"].to(torch.float16)))
    whole = range_bounds(exact, clean, dout, out, options, size, seq, seq)
    late = dout.clone()
    (late if layout == "BNSD" else late.transpose(1, 2))[:, :, :64] = 0
    tight = range_bounds(exact, clean, late, out, options, size, seq, seq)
    for n, x in zip(("dq", "dk", "dv"), got):
        bound = whole[n]
        if n == "dk":
            # (what the first rows leave in the exact value and its sums stays; their steps do not)
            keys = torch.arange(seq).view(1, 1, -1, 1) if layout == "BNSD" else torch.arange(seq).view(1, -1, 1, 1)
            bound = torch.where(keys >= 128, tight[n], whole[n])
        close(x, exact[n]["exact"], bound, n)
