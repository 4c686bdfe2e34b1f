"""Rotary positions, attention, its gradient and attention over an 8-bit cache: each against float64 on the host, at the
sizes, masks and lengths where a tile ends, a row sees nothing or the work is split; their refusals; all of them together."""
import json
import math

import pytest
import torch

import attention_reference as ref
from akg_amd import driver, op_desc

NAMES = {torch.bfloat16: "bfloat16", torch.float16: "float16", torch.float32: "float32", torch.int32: "int32", torch.int64: "int64",
         torch.int8: "int8", torch.bool: "bool"}


def builder(name="Fused_Layer"):
    return op_desc.DescBuilder(name)


def given(b, t):
    return b.input(list(t.shape), NAMES[t.dtype])


def launch(text, inputs, tmp_path, poison=True):
    """Outputs of a description on device copies of `inputs`; every output starts as NaN."""
    kernel = driver.HipKernel(text, out_dir=str(tmp_path))
    dtypes = {v: k for k, v in NAMES.items()}
    outs = [torch.full(d.shape, math.nan, dtype=dtypes[d.dtype], device="cuda") for d in kernel.outputs]
    kernel.launch([t.contiguous().cuda() for t in inputs] + outs)
    torch.cuda.synchronize()
    return [o.cpu() for o in outs]


def normal(shape, dtype, seed, factor=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * factor).to(ref.TYPES[dtype])


def close(got, exact, bound, what):
    got = got.to(torch.float64)
    assert torch.isfinite(got).all(), "%s: not finite" % what
    off = (got - exact).abs()
    worst = float((off / bound).max())
    assert (off <= bound).all(), "%s: %.3g of the bound, off by %.3g" % (what, worst, float(off.max()))


# ---- rotary ---------------------------------------------------------------------------------------------------------
WAVES = {"kind": "wavelength", "factor": 8.0, "original_length": 8192, "low": 1.0, "high": 4.0}
ROTARY = [
    # dtype, layout, batch, seq, heads, kv heads, channels, turned, interleaved, inverse, scaling, positions
    ("bfloat16", "BSND", 2, 5, 3, 1, 64, 0, False, False, None, "int32"),
    ("float32", "BSND", 1, 1, 1, 0, 2, 0, False, False, None, "int32"),
    ("float32", "BNSD", 2, 33, 4, 2, 96, 64, True, True, {"kind": "linear", "factor": 4.0}, "int64"),
    ("float16", "BSND", 3, 17, 9, 2, 80, 40, True, False, WAVES, "int32"),
    ("float16", "BNSD", 1, 130, 8, 8, 128, 32, False, True, WAVES, "far"),
    ("bfloat16", "BSND", 1, 1, 32, 8, 128, 0, False, False, WAVES, "far"),
    ("float32", "BSND", 1, 7, 2, 1, 13, 6, False, False, None, "shared"),
    ("bfloat16", "BSND", 4, 300, 16, 2, 256, 0, False, False, None, "negative"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: "-".join(str(x) for x in c[:10]))
def test_rotary_positions(case, tmp_path):
    dtype, layout, batch, seq, heads, kv, dim, turned, interleaved, inverse, scaling, kind = case
    shape = lambda h: (batch, seq, h, dim) if layout == "BSND" else (batch, h, seq, dim)   # noqa: E731
    xs = [normal(shape(h), dtype, 11 + h) for h in (heads, kv) if h]
    first = {"far": 1000000, "negative": -150}.get(kind, 0)
    positions = torch.arange(first, first + seq, dtype=torch.int64)
    if kind != "shared":
        positions = positions + torch.arange(batch)[:, None] * 1009
    if kind != "int64":
        positions = positions.to(torch.int32)
    b = builder()
    options = dict(layout=layout, base=500000.0, rotary_dims=turned, interleaved=interleaved, inverse=inverse, scaling=scaling, magnitude=1.25)
    outs = op_desc.rotary_embedding(b, [given(b, x) for x in xs], given(b, positions), **options)
    got = launch(b.dumps(outs), xs + [positions], tmp_path)
    u = ref.half_step(dtype)
    for x, y in zip(xs, got):
        exact = ref.rotary(x, positions, **options)
        # the result rounded (u); sine and cosine off by a few 2^-24, each product and sum by 2^-24; the angle itself by
        # 2^-31 turns. The reference's own angle is a float64 product: 2^-53 of at most 2^20 turns. float16's smallest steps.
        size = ref.rotary(x.abs(), torch.zeros_like(positions), **options).abs().amax() if x.numel() else 0
        bound = u * exact.abs() * 1.01 + 2.0 ** -20 * float(size) + (2.0 ** -25 if dtype == "float16" else 0)
        close(y, exact, bound, "rotary")
        r = turned or dim
        assert torch.equal(y[..., r:], x[..., r:])   # what is not turned is copied


@pytest.mark.gpu
def test_rotary_turned_back_gives_the_input(tmp_path):
    x = normal((2, 19, 4, 64), "float32", 3)
    positions = torch.arange(19, dtype=torch.int32) * 70001
    b = builder()
    p = given(b, positions)
    # (in description order: the positions are input 0)
    there = op_desc.rotary_embedding(b, [given(b, x)], p, interleaved=True)
    again = op_desc.rotary_embedding(b, there, p, interleaved=True, inverse=True)
    got = launch(b.dumps(again), [positions, x], tmp_path)
    close(got[0], x.double(), 2.0 ** -20 * x.abs().double().amax(), "there and back")


# ---- attention ------------------------------------------------------------------------------------------------------
# dtype, layout, batch, queries, keys, heads, key heads, channels, channels of the values, causal, mask, lengths
ATTENTION = [
    ("bfloat16", "BSND", 1, 1, 1, 1, 1, 8, 8, False, None, None),
    ("float16", "BSND", 2, 33, 65, 2, 2, 64, 64, False, None, None),
    ("bfloat16", "BNSD", 2, 130, 130, 4, 2, 128, 128, True, None, None),
    ("bfloat16", "BSND", 3, 77, 77, 6, 2, 40, 72, True, None, "padded"),
    ("float16", "BNSD", 3, 100, 63, 3, 1, 80, 64, True, None, "padded"),      # more queries than keys: rows that see nothing
    ("float16", "BSND", 2, 64, 200, 4, 4, 64, 128, False, "float32", None),
    ("bfloat16", "BNSD", 2, 70, 129, 4, 1, 96, 96, True, "bool", "padded"),
    ("float16", "BSND", 2, 50, 300, 2, 2, 32, 32, False, "float16", None),
    ("bfloat16", "BSND", 2, 9, 257, 6, 3, 64, 64, False, "rows", None),         # rows whose mask leaves nothing
    ("float16", "BSND", 1, 40, 64, 2, 1, 64, 64, False, "lowest", None),
    ("bfloat16", "BSND", 2, 1, 5000, 8, 2, 128, 128, True, None, "padded"),   # split along the keys
    ("float16", "BNSD", 1, 3, 1111, 4, 4, 64, 48, True, "float32", None),
    ("bfloat16", "BSND", 2, 48, 48, 2, 1, 256, 256, True, None, None),
    ("float16", "BSND", 1, 300, 300, 40, 8, 64, 64, True, None, None),
    ("bfloat16", "BSND", 4, 65, 65, 2, 2, 64, 64, True, None, "zero"),
    ("bfloat16", "BSND", 1, 2100, 2100, 32, 2, 64, 64, True, None, None),     # eight wavefronts to a workgroup
]


def lengths_of(kind, batch, sq, sk):
    if kind is None:
        return None, None
    if kind == "zero":
        return [0, sq, 1, -3][:batch], [sk, 0, 1, 9][:batch]
    return [max(1, sq - 7 * b) for b in range(batch)], [max(1, sk - 11 * b) for b in range(batch)]


def mask_of(kind, batch, heads, sq, sk):
    g = torch.Generator().manual_seed(99)
    if kind is None:
        return None
    if kind == "bool":
        return torch.rand((batch, 1, sq, sk), generator=g) < 0.7
    if kind == "float32":
        m = torch.randn((1, heads, sq, sk), generator=g)
        m[torch.rand(m.shape, generator=g) < 0.3] = -math.inf
        return m
    if kind == "float16":
        return torch.randn((batch, 1, 1, sk), generator=g).to(torch.float16)
    if kind == "rows":
        m = torch.rand((batch, heads, sq, sk), generator=g) < 0.5
        m[:, :, ::3] = False
        return m
    # the type's lowest value: all keys of a row alike, which is a mean over them
    m = torch.zeros((1, 1, sq, sk), dtype=torch.float32)
    m[..., 10:] = torch.finfo(torch.float32).min
    m[:, :, ::2] = torch.finfo(torch.float32).min
    return m


def attention_case(case, seed=5):
    dtype, layout, batch, sq, sk, h, hkv, dk, dv, causal, mask, lengths = case
    shape = lambda s, n, d: (batch, s, n, d) if layout == "BSND" else (batch, n, s, d)   # noqa: E731
    t = {"q": normal(shape(sq, h, dk), dtype, seed, 2.0), "k": normal(shape(sk, hkv, dk), dtype, seed + 1), "v": normal(shape(sk, hkv, dv), dtype, seed + 2)}
    m = mask_of(mask, batch, h, sq, sk)
    ql, kl = lengths_of(lengths, batch, sq, sk)
    options = dict(layout=layout, causal=causal)
    extra = {}
    if m is not None:
        extra["mask"] = m
    if ql is not None:
        extra["query_lengths"], extra["key_lengths"] = (torch.tensor(x, dtype=torch.int32) for x in (ql, kl))
    return t, extra, options, m, ql, kl


def describe_attention(t, extra, options, lse=True):
    b = builder()
    qkv = [given(b, t[n]) for n in "qkv"]
    more = {n: given(b, x) for n, x in extra.items()}
    return b.dumps(op_desc.attention(b, *qkv, lse=lse, **more, **options)), [t[n] for n in "qkv"] + list(extra.values())


def behind_lengths(x, lengths, layout, value):
    """`x` with `value` in the rows behind the lengths."""
    if lengths is None:
        return x
    x = x.clone()
    for b, n in enumerate(lengths):
        (x[b] if layout == "BSND" else x[b].transpose(0, 1))[max(n, 0):] = value
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(str(x) for x in c))
def test_attention(case, tmp_path):
    t, extra, options, m, ql, kl = attention_case(case)
    layout = options["layout"]
    # nothing behind the lengths may reach a result
    for n, lengths in (("q", ql), ("k", kl), ("v", kl)):
        t[n] = behind_lengths(t[n], lengths, layout, math.nan)
    text, inputs = describe_attention(t, extra, options)
    out, lse = launch(text, inputs, tmp_path)
    clean = [behind_lengths(t[n], lengths, layout, 0.0) for n, lengths in (("q", ql), ("k", kl), ("v", kl))]
    r = ref.forward(*clean, mask=m, qlens=ql, klens=kl, **options)
    close(out, r["out"], ref.forward_bound(r, case[0]), "out")
    empty = torch.isinf(r["lse"])
    assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all()
    # (a sum with the lowest value of float32 is itself rounded to float32)
    assert ((lse[~empty].double() - r["lse"][~empty]).abs() <= ref.lse_bound(r) + 2.0 ** -23 * r["lse"][~empty].abs()).all()


@pytest.mark.gpu
def test_attention_without_its_log_sums(tmp_path):
    t, extra, options, m, ql, kl = attention_case(ATTENTION[2])
    text, inputs = describe_attention(t, extra, options, lse=False)
    whole, whole_inputs = describe_attention(t, extra, options)
    assert torch.equal(launch(text, inputs, tmp_path)[0], launch(whole, whole_inputs, tmp_path)[0])


# ---- its gradient ---------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(str(x) for x in c))
def test_attention_gradient(case, tmp_path):
    t, extra, options, m, ql, kl = attention_case(case)
    dtype, layout = case[0], options["layout"]
    r = ref.forward(t["q"], t["k"], t["v"], mask=m, qlens=ql, klens=kl, **options)
    out, lse = r["out"].to(ref.TYPES[dtype]), r["lse"].float()
    dout = normal(out.shape, dtype, 8)
    gradient_against_formula(dtype, t, dout, out, lse, extra, options, m, ql, kl, tmp_path)


def gradient_against_formula(dtype, t, dout, out, lse, extra, options, m, ql, kl, tmp_path):
    layout = options["layout"]
    b = builder()
    named = {"dout": dout, **t, "out": out, "lse": lse}
    for n, lengths in (("dout", ql), ("q", ql), ("out", ql), ("k", kl), ("v", kl)):
        named[n] = behind_lengths(named[n], lengths, layout, math.nan)
    args = [given(b, named[n]) for n in ("dout", "q", "k", "v", "out", "lse")]
    more = {n: given(b, x) for n, x in extra.items()}
    grads = op_desc.attention_grad(b, *args, **more, **options)
    got = launch(b.dumps(grads), [named[n] for n in ("dout", "q", "k", "v", "out", "lse")] + list(extra.values()), tmp_path)
    exact, size = ref.gradient(dout, t["q"], t["k"], t["v"], out, lse, mask=m, qlens=ql, klens=kl, **options)
    for n, x in zip(("dq", "dk", "dv"), got):
        close(x, exact[n]["exact"], ref.gradient_bound(exact[n], dtype, size, t["q"].shape[3]), n)
    return got


@pytest.mark.gpu
def test_float16_gradients_of_a_small_loss(tmp_path):
    # gradients of 2^-12: a probability of 1 / 300 times such a number is below the normal float16 numbers
    case = ("float16", "BSND", 1, 300, 300, 2, 1, 64, 64, False, None, None)
    t, extra, options, m, ql, kl = attention_case(case)
    r = ref.forward(t["q"], t["k"], t["v"], **options)
    dout = (normal(r["out"].shape, "float16", 8).float() * 2.0 ** -12).to(torch.float16)
    gradient_against_formula("float16", t, dout, r["out"].to(torch.float16), r["lse"].float(), extra, options, m, ql, kl, tmp_path)


@pytest.mark.gpu
def test_gradient_against_differences(tmp_path):
    """The gradient of sum(weight * out) along random directions against a central difference of the float64 forward pass."""
    case = ("bfloat16", "BSND", 2, 40, 56, 4, 2, 64, 64, True, None, "padded")
    t, extra, options, m, ql, kl = attention_case(case)
    r = ref.forward(t["q"], t["k"], t["v"], qlens=ql, klens=kl, **options)
    dout = normal(r["out"].shape, "bfloat16", 21)
    b = builder()
    args = [dout, t["q"], t["k"], t["v"], r["out"].to(torch.bfloat16), r["lse"].float()]
    grads = op_desc.attention_grad(b, *[given(b, x) for x in args], **{n: given(b, x) for n, x in extra.items()}, **options)
    got = launch(b.dumps(grads), args + list(extra.values()), tmp_path)
    weight = behind_lengths(dout, ql, "BSND", 0.0).double()
    exact, _ = ref.gradient(dout, t["q"], t["k"], t["v"], r["out"], r["lse"], qlens=ql, klens=kl, **options)
    for name, key, grad in (("dq", "q", got[0]), ("dk", "k", got[1]), ("dv", "v", got[2])):
        direction = normal(t[key].shape, "float32", 31).double()
        step = 1e-4
        value = {}
        for sign in (1, -1):
            moved = {n: x.double() for n, x in t.items()}
            moved[key] = moved[key] + sign * step * direction
            value[sign] = float((ref.forward(moved["q"], moved["k"], moved["v"], qlens=ql, klens=kl, **options)["out"] * weight).sum())
        difference = (value[1] - value[-1]) / (2 * step)
        # every entry is off by a few half steps of what was summed for it (and delta, from the rounded result, by one of its
        # terms), of independent signs: six standard deviations of their sum; the difference itself by step^2
        u = 2.0 ** -8
        scatter = float(((3 * u * exact[name]["rough"] * direction) ** 2).sum().sqrt())
        assert abs(float((grad.double() * direction).sum()) - difference) <= 6 * scatter + 1e-4 * abs(difference), name


# ---- attention over the cache ----------------------------------------------------------------------------------------
# dtype, batch, queries, heads, key heads, channels, tokens of a block, blocks of a sequence, lengths, what is odd
CACHE = [
    ("bfloat16", 1, 1, 1, 1, 16, 16, 1, [1], None),
    ("float16", 3, 1, 8, 2, 64, 16, 9, [144, 17, 100], None),
    ("bfloat16", 4, 1, 32, 8, 128, 64, 5, [320, 1, 64, 65], None),
    ("bfloat16", 2, 4, 16, 4, 128, 32, 7, [200, 5], None),
    ("float16", 2, 3, 12, 2, 80, 48, 6, [288, 2], None),                # more queries than tokens: rows that see nothing
    ("bfloat16", 2, 2, 64, 2, 96, 128, 4, [512, 300], "scales"),
    ("float16", 3, 1, 8, 2, 256, 16, 40, [640, 0, -4], None),
    ("bfloat16", 2, 1, 8, 1, 192, 64, 3, [1000, 128], "table"),         # a length behind the table, entries outside the pool
    ("float16", 1, 5, 40, 2, 64, 16, 70, [1111], None),                    # a hundred rows
    ("bfloat16", 1, 1, 8, 2, 128, 256, 40, [9999], "scales"),
]


def cache_case(case):
    dtype, batch, sq, h, hkv, dim, page, per, lengths, odd = case
    g = torch.Generator().manual_seed(17)
    total = batch * per + 3
    t = {"q": normal((batch, sq, h, dim), dtype, 4, 2.0)}
    for n in ("key", "value"):
        t[n + "_cache"] = torch.randint(-128, 128, (total, hkv, page, dim), generator=g).to(torch.int8)
        t[n + "_scale"] = torch.rand((total, hkv), generator=g) * 0.02 + 0.01
    if odd == "scales":   # from block to block over many powers of two, and zero
        t["value_scale"] = torch.exp2(torch.randint(-30, 10, (total, hkv), generator=g).float()) * 1.3
        t["value_scale"][::5] = 0.0
    t["block_table"] = torch.randperm(total, generator=g)[:batch * per].to(torch.int32).view(batch, per).clone()
    if odd == "table":
        t["block_table"][0, 1], t["block_table"][1, 0] = total, -1
    t["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    return t


def describe_cache(t):
    b = builder()
    return b.dumps([op_desc.cache_attention(b, *[given(b, x) for x in t.values()])])


CACHE_ORDER = ("q", "key_cache", "value_cache", "key_scale", "value_scale", "block_table", "lengths")


@pytest.mark.gpu
@pytest.mark.parametrize("case", CACHE, ids=lambda c: "-".join(str(x) for x in c))
def test_cache_attention(case, tmp_path):
    t = cache_case(case)
    t = {n: t[n] for n in CACHE_ORDER}
    got = launch(describe_cache(t), list(t.values()), tmp_path)[0]
    r = ref.cache_attention(**{("table" if n == "block_table" else n): x for n, x in t.items()})
    close(got, r["out"], ref.cache_bound(r, case[0]), "cache attention")


# ---- axes that several workgroups share, and masks of a few elements ----------------------------------------------------
SHARED = [
    ("bfloat16", "BSND", 1, 20, 1500, 16, 2, 128, 128, True, None, "padded"),   # 64 rows times 11 ranges of keys: joined by a launch of its own
    ("float16", "BNSD", 2, 3, 700, 4, 4, 64, 64, False, "rows", None),          # 3 rows times 5 ranges: by the last workgroup
    ("float16", "BSND", 1, 40, 900, 8, 1, 256, 256, False, "float32", None),
    ("bfloat16", "BSND", 1, 33, 640, 6, 1, 8, 24, False, None, None),
    ("bfloat16", "BSND", 1, 600, 600, 8, 2, 64, 64, True, None, "padded"),      # the gradients of keys and values: 2400 rows in 4 ranges
    ("float16", "BNSD", 2, 520, 300, 4, 1, 96, 40, False, "bool", None),
    ("float16", "BSND", 4, 300, 70, 8, 1, 256, 128, True, None, "zero"),
    ("float16", "BSND", 1, 3, 5, 1, 1, 64, 64, False, "bool", None),            # a mask of 15 bytes
    ("bfloat16", "BSND", 1, 1, 7, 2, 1, 16, 16, False, "float32", None),
    ("float16", "BSND", 1, 2, 45, 1, 1, 64, 64, False, "float16", None),
    ("bfloat16", "BSND", 2, 40, 33, 2, 2, 64, 64, False, "bool", None),
]


WIDE = [
    ("bfloat16", "BSND", 1, 700, 90, 4, 2, 192, 192, True, None, "padded"),     # dk and dv by workgroups of their own, rows in two ranges
    ("float16", "BNSD", 2, 65, 130, 2, 2, 256, 8, False, "float32", None),
    ("float16", "BSND", 1, 40, 33, 2, 1, 40, 256, True, "bool", "padded"),
    ("bfloat16", "BNSD", 2, 96, 96, 3, 3, 136, 136, False, None, None),
    ("bfloat16", "BSND", 4, 70, 200, 40, 40, 136, 64, True, None, None),        # one group of wavefronts, in one launch with dq
    ("float16", "BSND", 2, 33, 257, 40, 10, 64, 136, False, "bool", "padded"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", WIDE, ids=lambda c: "-".join(str(x) for x in c))
def test_wide_heads(case, tmp_path):
    test_attention(case, tmp_path / "forward")
    test_attention_gradient(case, tmp_path / "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("case", SHARED, ids=lambda c: "-".join(str(x) for x in c))
def test_shared_axes(case, tmp_path):
    test_attention(case, tmp_path / "forward")


@pytest.mark.gpu
@pytest.mark.parametrize("case", SHARED, ids=lambda c: "-".join(str(x) for x in c))
def test_shared_axes_gradient(case, tmp_path):
    test_attention_gradient(case, tmp_path / "gradient")


@pytest.mark.gpu
def test_a_shared_axis_gives_the_same_bits_every_time(tmp_path):
    """The ranges are joined in their order, whichever workgroup ends last."""
    for case in (SHARED[0], SHARED[1]):
        t, extra, options, m, ql, kl = attention_case(case)
        text, inputs = describe_attention(t, extra, options)
        first = launch(text, inputs, tmp_path)
        for _ in range(3):
            assert all(torch.equal(x, y) for x, y in zip(first, launch(text, inputs, tmp_path)))


# ---- refusals and what is chosen, without a GPU -----------------------------------------------------------------------
def refused(text, code, part):
    with pytest.raises(driver.AkgHipError) as e:
        driver.HipKernel(text, out_dir=None)
    assert e.value.code == code and part in str(e.value), str(e.value)


def attention_text(q=(2, 5, 4, 64), k=(2, 7, 2, 64), v=(2, 7, 2, 64), dtype="float16", mask=None, lengths=None, **options):
    b = builder()
    t = [b.input(list(s), dtype) for s in (q, k, v)]
    more = {}
    if mask is not None:
        more["mask"] = b.input(list(mask[0]), mask[1])
    if lengths is not None:
        more["key_lengths"] = b.input(list(lengths[0]), lengths[1])
    return b.dumps(op_desc.attention(b, *t, **more, **options))


@pytest.mark.parametrize("change,code,part", [
    (dict(dtype="float32"), -3, "float16 or bfloat16"),
    (dict(k=(2, 7, 3, 64), v=(2, 7, 3, 64)), -3, "multiple of the key heads"),
    (dict(k=(2, 7, 2, 32)), -3, "channels of a head"),
    (dict(v=(2, 8, 2, 64)), -3, "differ in length or heads"),
    (dict(k=(3, 7, 2, 64), v=(3, 7, 2, 64)), -3, "batch"),
    (dict(q=(2, 5, 4, 12), k=(2, 7, 2, 12), v=(2, 7, 2, 12)), -4, "multiple of 8 up to 256"),
    (dict(q=(2, 5, 4, 264), k=(2, 7, 2, 264)), -4, "multiple of 8 up to 256"),
    (dict(mask=((2, 4, 5, 8), "float32")), -3, "mask must be"),
    (dict(mask=((2, 4, 5, 7), "int32")), -3, "mask must be"),
    (dict(mask=((2, 3, 5, 7), "bool")), -3, "mask must be"),
    (dict(lengths=((2,), "int64")), -3, "key lengths"),
    (dict(lengths=((3,), "int32")), -3, "key lengths"),
    (dict(scale=0.0), -3, "scale"),
    (dict(layout="SBND"), -3, "layout"),
    (dict(q=(2, 0, 4, 64)), -3, "extent of 0"),
])
def test_attention_refusals(change, code, part):
    refused(attention_text(**change), code, part)


def test_wrong_results_and_operands_are_refused():
    doc = json.loads(attention_text())
    doc["op_desc"][0]["input_desc"].pop()
    refused(json.dumps(doc), -3, "operands")
    doc = json.loads(attention_text())
    doc["op_desc"][0]["output_desc"][0]["shape"][1] += 1
    refused(json.dumps(doc), -3, "does not follow")
    doc = json.loads(attention_text())
    doc["op_desc"][0]["output_desc"][1]["data_type"] = "float16"
    refused(json.dumps(doc), -3, "must be float32")
    doc = json.loads(attention_text())
    for a in doc["op_desc"][0]["attr"]:
        if a["name"] == "causal":
            a["value"] = 1
    refused(json.dumps(doc), -3, "bool")


def test_gradient_and_cache_and_rotary_refusals():
    def grad(lse=(2, 4, 5), out=(2, 5, 4, 64), dtype="float32"):
        b = builder()
        dout, q = b.input([2, 5, 4, 64], "float16"), b.input([2, 5, 4, 64], "float16")
        k, v = b.input([2, 7, 2, 64], "float16"), b.input([2, 7, 2, 64], "float16")
        return b.dumps(op_desc.attention_grad(b, dout, q, k, v, b.input(list(out), "float16"), b.input(list(lse), dtype)))
    driver.translate(grad())
    refused(grad(lse=(2, 5, 4)), -3, "lse")
    refused(grad(dtype="float16"), -3, "lse")
    refused(grad(out=(2, 4, 5, 64)), -3, "result and its gradient")

    def cache(dim=64, page=16, kc="int8", ks="float32", table="int32", scales=(9, 2), pool=(9, 2)):
        b = builder()
        x = [b.input([2, 1, 4, dim], "float16"), b.input([*pool, page, dim], kc), b.input([*pool, page, dim], kc), b.input(list(scales), ks),
             b.input(list(scales), ks), b.input([2, 3], table), b.input([2], "int32")]
        return b.dumps([op_desc.cache_attention(b, *x)])
    driver.translate(cache())
    refused(cache(dim=72), -4, "multiple of 16")
    refused(cache(dim=272), -4, "multiple of 16")
    refused(cache(page=24), -4, "multiple of 16")
    refused(cache(kc="float16"), -3, "int8")
    refused(cache(ks="float16"), -3, "scales")
    refused(cache(scales=(9, 4)), -3, "scales")
    refused(cache(table="int64"), -3, "block table")
    refused(cache(pool=(9, 3), scales=(9, 3)), -3, "multiple of the key heads")

    def turned(dim=64, positions=("int32", [5]), dtype="float16", second=None, **options):
        b = builder()
        xs = [b.input([2, 5, 4, dim], dtype)] + ([b.input(second, dtype)] if second else [])
        return b.dumps(op_desc.rotary_embedding(b, xs, b.input(positions[1], positions[0]), **options))
    driver.translate(turned())
    refused(turned(positions=("float32", [5])), -3, "positions")
    refused(turned(positions=("int32", [6])), -3, "positions")
    refused(turned(positions=("int32", [3, 5])), -3, "positions")
    refused(turned(dtype="int32"), -3, "float32")
    refused(turned(rotary_dims=66), -3, "rotary_dims")
    refused(turned(rotary_dims=7), -3, "rotary_dims")
    refused(turned(dim=63), -3, "rotary_dims")
    refused(turned(base=1.0), -3, "base")
    refused(turned(second=[2, 6, 4, 64]), -3, "number of heads only")
    refused(turned(scaling={"kind": "other"}), -3, "scaling")
    refused(turned(scaling={"kind": "wavelength", "factor": 2.0}), -3, "original_length")
    refused(turned(scaling={"kind": "linear", "factor": 0.5}), -3, "factor")


def test_extents_are_arguments_and_code_objects_are_shared(tmp_path):
    texts = [attention_text(q=(2, s, 4, 64), k=(2, s, 2, 64), v=(2, s, 2, 64), causal=True) for s in (40, 41, 57)]
    kernels = [driver.HipKernel(t, out_dir=str(tmp_path)) for t in texts]
    assert [k.family for k in kernels] == ["attention"] * 3
    assert len({k.source for k in kernels}) == 1 and kernels[1].cache_hit and kernels[2].cache_hit


def test_few_rows_over_many_keys_are_split(tmp_path):
    def kernel(q, k):
        return driver.HipKernel(attention_text(q=(1, q, 4, 64), k=(1, k, 2, 64), v=(1, k, 2, 64)), out_dir=str(tmp_path))
    assert kernel(1, 8192).workspace_bytes > 0 and kernel(1, 200).workspace_bytes == 0


def test_launches_of_too_many_threads_are_refused():
    b = builder()
    refused(b.dumps(op_desc.rotary_embedding(b, [b.input([1, 1 << 27, 32, 16], "float16")], b.input([1 << 27], "int32"))), -4, "more threads")
    refused(attention_text(q=(1 << 22, 1, 16, 64), k=(1 << 22, 1, 16, 64), v=(1 << 22, 1, 16, 64)), -4, "more threads")


def test_rows_and_keys_whose_numbers_pass_32_bits_are_refused():
    n = 1 << 30
    refused(attention_text(q=(1, n, 1, 8), k=(1, n, 1, 8), v=(1, n, 1, 8)), -4, "2^31 rows")
    refused(attention_text(q=(1, n, 2, 8), k=(1, 8, 1, 8), v=(1, 8, 1, 8)), -4, "2^31 rows")


def test_small_gradients_are_one_launch_beside_the_rows_own(tmp_path):
    def kernel(s):
        b = builder()
        dout, q, k, v, out = (b.input([2, s, 4, 64], "float16") for _ in range(5))
        return driver.HipKernel(b.dumps(op_desc.attention_grad(b, dout, q, k, v, out, b.input([2, 4, s], "float32"))), out_dir=str(tmp_path))
    assert "akg_K" in kernel(200).source and "akg_K" not in kernel(8192).source


def test_rows_of_the_gradient_are_shared_where_keys_are_few(tmp_path):
    def kernel(s, h, hkv, batch=1):
        b = builder()
        dout, q, out = (b.input([batch, s, h, 64], "float16") for _ in range(3))
        k, v = (b.input([batch, s, hkv, 64], "float16") for _ in range(2))
        return driver.HipKernel(b.dumps(op_desc.attention_grad(b, dout, q, k, v, out, b.input([batch, h, s], "float32"))), out_dir=str(tmp_path))
    assert "backward_join" in kernel(512, 8, 2).source
    assert "backward_join" not in kernel(200, 4, 4).source and "backward_join" not in kernel(2048, 16, 16, 2).source


def test_attributes_that_no_float_holds_are_refused():
    def turned(**changes):
        b = builder()
        doc = json.loads(b.dumps(op_desc.rotary_embedding(b, [b.input([2, 5, 4, 64], "float16")], b.input([5], "int32"),
                                                         scaling={"kind": "linear", "factor": 2.0})))
        for a in doc["op_desc"][0]["attr"]:
            a["value"] = changes.get(a["name"], a["value"])
        return json.dumps(doc)
    driver.translate(turned())
    for name, value in (("rotary_dims", 62.5), ("rotary_dims", 1e30), ("rotary_dims", -2), ("magnitude", 1e300), ("magnitude", -1e39), ("base", math.inf),
                        ("base", math.nan), ("factor", math.inf)):
        refused(turned(**{name: value}), -3, name)
    for scale in (1e300, 1e-60, 0.0, -1.0, math.inf, math.nan):
        refused(attention_text(scale=scale), -3, "scale")
    driver.translate(attention_text(scale=2.0 ** -100))
