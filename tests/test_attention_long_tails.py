"""Rows in which one key has half of the weight or more and very many equal ones have the rest, each far below float16's normal numbers
times the largest: what their roundings add up to stays within the rounding of a probability."""
import math

import pytest
import torch

import attention_reference as ref
from akg_amd import driver, op_desc
from test_attention_ops import CACHE_ORDER, builder, close, describe_cache, given, launch
from test_attention_use import empties

TAIL = math.log(40.5 / 2 ** 24)   # of a key's score to the heavy one's: 40.5 steps of 2^-24


@pytest.mark.gpu
@pytest.mark.parametrize("mask", [False, True])
def test_attention_with_a_long_tail(mask, tmp_path):
    keys, queries, dim = (1 << 17), 16384, 64      # (as many queries as leave the keys in one range)
    q = torch.zeros((1, queries, 1, dim), dtype=torch.float16)
    q[..., 0], q[..., 1] = 1.0, 2.0 ** -8
    k = torch.zeros((1, keys, 1, dim), dtype=torch.float16)
    k[:, 1:, :, 0], k[:, 1:, :, 1] = -13.0, (TAIL + 13.0) * 256
    v = torch.ones((1, keys, 1, dim), dtype=torch.float16)
    v[:, 0] = 0
    b = builder("Fused_Tail")
    x = [given(b, t) for t in (q, k, v)]
    added = torch.zeros((1, 1, 1, keys), dtype=torch.float16)
    out = op_desc.attention(b, *x, scale=1.0, **({"mask": given(b, added)} if mask else {}))
    kernel = driver.HipKernel(b.dumps(out), out_dir=str(tmp_path))
    assert kernel.workspace_bytes == 0   # (the keys are not in ranges)
    outs = empties(kernel)
    kernel.launch([t.cuda() for t in [q, k, v] + ([added] if mask else [])] + outs)
    torch.cuda.synchronize()
    r = ref.forward(q[:, :1], k, v, scale=1.0)
    assert 0.2 < float(r["out"].max()) < 0.3
    # every probability and the result rounded (2^-11 each); float32 in scores and in sums of keys / 32 terms a lane; steps of
    # 2^-24 of the smallest float16 no more than 2^-7 of a heavy key's own
    noise = 2.0 ** -23 * (dim + 4) * (r["size"] + 1) + 2.0 ** -24 * (keys / 32)
    bound = (2 * 2.0 ** -11 + noise) * 1.01 * r["out"] + keys * 2.0 ** -25 * 2.0 ** -7
    for i in (0, 5000, queries - 1):
        close(outs[0][:, i:i + 1].cpu(), r["out"], bound, "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_cache_attention_with_a_long_tail(dtype, tmp_path):
    # all sequences read the same blocks; as many of them as leave a sequence to one workgroup
    batch, hkv, page, per, dim = 256, 8, 16, 2048, 64
    tokens = page * per
    t = {"q": torch.ones((batch, 1, hkv, dim), dtype=ref.TYPES[dtype])}
    key = torch.zeros((per, hkv, page, dim), dtype=torch.int8)
    value = torch.full((per, hkv, page, dim), 100, dtype=torch.int8)
    key[0, :, 0], value[0, :, 0] = 127, 0
    t["key_cache"], t["value_cache"] = key, value
    t["key_scale"] = torch.full((per, hkv), -TAIL / (127 * math.sqrt(dim)))
    t["value_scale"] = torch.full((per, hkv), 2.0 ** -7)
    t["block_table"] = torch.arange(per, dtype=torch.int32).expand(batch, per).contiguous()
    t["lengths"] = torch.full((batch,), tokens, dtype=torch.int32)
    t = {n: t[n] for n in CACHE_ORDER}
    kernel = driver.HipKernel(describe_cache(t), out_dir=str(tmp_path))
    assert kernel.workspace_bytes == 0
    got = launch(describe_cache(t), list(t.values()), tmp_path)[0]
    one = {("table" if n == "block_table" else n): (x[:1] if n in ("q", "block_table", "lengths") else x) for n, x in t.items()}
    r = ref.cache_attention(**one)
    assert 0.04 < float(r["out"].max()) < 0.1
    u = ref.half_step(dtype)
    noise = 2.0 ** -23 * (dim + 4) * (r["size"] + 1) + 2.0 ** -24 * (tokens / 32)
    # steps of 2^-38 of twice the heavy token's weight, 2^-7, times numbers of 100
    bound = (2.0 ** -11 + noise + u) * 1.01 * r["out"] + tokens * 2.0 ** -38 * 2
    for i in (0, 100, batch - 1):
        close(got[i:i + 1], r["out"], bound, "cache attention")
