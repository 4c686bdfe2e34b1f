"""Attention over the 8-bit cache where the scales of the values' blocks differ by many powers of two: every row's weights are
as good as the block scales times its own probabilities, whatever scales lie on blocks that it does not attend to."""
import math

import pytest
import torch

import attention_reference as ref
from test_attention_ops import CACHE, CACHE_ORDER, cache_case, close, describe_cache, launch, normal

F = torch.float64


def as_reference(t):
    return {("table" if n == "block_table" else n): x for n, x in t.items()}


def heaviest(t):
    """max over the tokens that a row sees of probability times |scale of the value block|, [batch, queries, heads, 1], and the
    tokens seen, [batch, queries, 1, 1]."""
    batch, sq, h, dim = t["q"].shape
    hkv, page = t["key_cache"].shape[1:3]
    weight, count = torch.zeros((batch, sq, h, 1), dtype=F), torch.zeros((batch, sq, 1, 1), dtype=F)
    ones = torch.ones_like(t["value_cache"])
    for b in range(batch):
        n = min(max(int(t["lengths"][b]), 0), t["block_table"].shape[1] * page)
        k, live = ref.dense_cache(t["key_cache"], t["key_scale"], t["block_table"][b], n, page)
        s, _ = ref.dense_cache(ones, t["value_scale"], t["block_table"][b], n, page)
        k, s = k.repeat_interleave(h // hkv, 0), s[..., 0].abs().repeat_interleave(h // hkv, 0)
        for i in range(sq):
            seen = min(max(n - sq + 1 + i, 0), n)
            ok = live[:seen]
            if not bool(ok.any()):
                continue
            x = (k[:, :seen] @ t["q"][b, i].to(F)[..., None])[..., 0] / math.sqrt(dim)
            p = torch.softmax(x.masked_fill(~ok, -math.inf), -1)
            weight[b, i, :, 0], count[b, i] = (p * s[:, :seen]).amax(-1), seen
    return weight, count


def tight_bound(t, r, dtype):
    """|computed - exact|. A probability times its block's scale is rounded to float16: 2^-11 of it, and 2^-25 in units of a power of
    two that is at most twice the row's heaviest, times numbers up to 128, once for every token. Scores: float32 (2^-23
    (channels + 4) (size + 1) relative in every probability); bfloat16 queries are float16 relative to the largest of the row,
    off by 2^-25 of it where that has no digits left, which moves a score by `moved` and every probability by twice that."""
    u = ref.half_step(dtype)
    weight, count = heaviest(t)
    dim = t["q"].shape[3]
    noise = 2.0 ** -23 * (dim + 4) * (r["size"] + 1)
    moved = 0.0
    if dtype == "bfloat16":
        largest_key = float(t["key_scale"].abs().max()) * 128
        moved = dim * 2.0 ** -25 * float(t["q"].abs().max()) * largest_key / math.sqrt(dim)
    result = 2.0 ** -25 if dtype == "float16" else 0.0
    return ((2.0 ** -11 + noise + 2 * moved) * r["spread"] + u * r["out"].abs() + count * 128 * 2.0 ** -25 * 2 * weight) * 1.01 + result + 1e-30


# type, queries, tokens of a block, channels, exponents of two of the scales block by block, scores of a block (+: the even heads
# attend to it, -: the odd ones)
SCALES = [
    ("bfloat16", 1, 16, 64, [0, -20], [-20.0, 20.0]),
    ("float16", 1, 64, 128, [-14, 6], [20.0, -20.0]),                 # the larger scale behind
    ("bfloat16", 2, 64, 128, [0, -16, 0], [-18.0, 18.0, -18.0]),
    ("float16", 4, 16, 80, [-12, 7, -12, 7, -4], [16.0, -16.0, 16.0, -16.0, 0.0]),
    ("bfloat16", 1, 48, 64, [-30, 10], [14.0, -14.0]),                # the even heads: both count
    ("float16", 1, 16, 96, [6, -14] * 100, [-20.0, 20.0] * 100),      # tokens in ranges
    ("bfloat16", 3, 32, 256, [-20, 0, 20], [20.0, 0.0, -20.0]),
    ("float16", 9, 16, 64, [7, -13] * 20, [-9.0, 9.0] * 20),         # several tiles of rows
]


def scales_case(case):
    dtype, sq, page, dim, exponents, scores = case
    g = torch.Generator().manual_seed(5)
    heads, hkv, per = 16, 2, len(exponents)
    sign = torch.where(torch.rand((hkv, dim), generator=g) < 0.5, -1.0, 1.0)
    # head j of a group points along the key heads' signs or against them
    along = torch.tensor([1.0, -1.0] * (heads // 2))[None, None, :, None] * sign.repeat_interleave(heads // hkv, 0)[None, None]
    t = {"q": (along * (1.0 + torch.rand((1, sq, heads, dim), generator=g) / 16)).to(ref.TYPES[dtype])}
    shape = (per, hkv, page, dim)
    keys = torch.randint(90, 128, shape, generator=g) * sign[None, :, None, :]
    side = torch.tensor([1.0 if x >= 0 else -1.0 for x in scores])[:, None, None, None]
    t["key_cache"] = (keys * side).to(torch.int8)
    t["value_cache"] = torch.randint(-128, 128, shape, generator=g).to(torch.int8)
    # (a key of +-127 along the signs with scale s gives a score of 127 s sqrt(channels))
    t["key_scale"] = (torch.tensor(scores).abs() / (127 * math.sqrt(dim)))[:, None].expand(per, hkv).contiguous().float()
    t["value_scale"] = (torch.exp2(torch.tensor(exponents, dtype=torch.float32))[:, None] * (1 + torch.rand((per, hkv), generator=g))).contiguous()
    t["block_table"] = torch.arange(per, dtype=torch.int32).view(1, per)
    t["lengths"] = torch.tensor([per * page - 3], dtype=torch.int32)
    return {n: t[n] for n in CACHE_ORDER}


@pytest.mark.gpu
@pytest.mark.parametrize("case", SCALES, ids=lambda c: "-".join(str(x) for x in c[:4]) + "-%d" % len(c[4]))
def test_scales_of_blocks_that_a_row_does_not_attend_to(case, tmp_path):
    t = scales_case(case)
    got = launch(describe_cache(t), list(t.values()), tmp_path)[0]
    r = ref.cache_attention(**as_reference(t))
    close(got, r["out"], tight_bound(t, r, case[0]), "cache attention")


@pytest.mark.gpu
@pytest.mark.parametrize("case", CACHE, ids=lambda c: "-".join(str(x) for x in c))
def test_cache_attention_within_the_steps_of_its_numbers(case, tmp_path):
    t = cache_case(case)
    t = {n: t[n] for n in CACHE_ORDER}
    got = launch(describe_cache(t), list(t.values()), tmp_path)[0]
    r = ref.cache_attention(**as_reference(t))
    close(got, r["out"], tight_bound(t, r, case[0]), "cache attention")


@pytest.mark.parametrize("case", [c for c in CACHE if c[0] == "float16"], ids=lambda c: "-".join(str(x) for x in c))
def test_the_bound_sees_a_result_rounded_to_fewer_bits(case):
    t = cache_case(case)
    t = {n: t[n] for n in CACHE_ORDER}
    r = ref.cache_attention(**as_reference(t))
    bound = tight_bound(t, r, "float16")
    assert ((r["out"].to(torch.bfloat16).double() - r["out"]).abs() > bound).any()
    assert ((r["out"].to(torch.float16).double() - r["out"]).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("page,queries,per", [(16, 3, 3), (64, 2, 2), (32, 4, 40)])
def test_scales_of_a_block_that_a_query_does_not_see(page, queries, per, bad, tmp_path):
    """The last query's own token opens a block whose scales are no numbers: the queries before it never see that block."""
    case = ("float16", 1, queries, 8, 2, 64, page, per, [(per - 1) * page + 1], None)
    t = cache_case(case)
    t = {n: t[n] for n in CACHE_ORDER}
    last = int(t["block_table"][0, per - 1])
    r = ref.cache_attention(**as_reference(t))
    bound = tight_bound(t, r, "float16")
    t["key_scale"][last] = bad
    t["value_scale"][last] = bad
    got = launch(describe_cache(t), list(t.values()), tmp_path)[0]
    close(got[:, :-1], r["out"][:, :-1], bound[:, :-1], "queries before the last")
    assert not torch.isfinite(got[:, -1]).any()
