"""The operators of an attention layer in float64 on the host, and bounds on what rounding to the result's type, and of the
probabilities and their gradients to the type of the operands, can change. `u` is half a step of a type relative to the
value: torch.finfo(t).eps / 2."""
import math

import torch

F = torch.float64
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def half_step(dtype):
    return torch.finfo(TYPES[dtype]).eps / 2


def heads_of(x, layout):
    """[batch, heads, sequence, channels] in float64."""
    x = x.to(F)
    return x if layout == "BNSD" else x.transpose(1, 2)


def back(x, layout):
    return x if layout == "BNSD" else x.transpose(1, 2)


def allowed(batch, sq, sk, causal, qlens, klens):
    """[batch, 1, sq, sk]: the pairs that the lengths and the causal order leave."""
    ql = torch.tensor([sq] * batch if qlens is None else [min(max(int(n), 0), sq) for n in qlens]).view(-1, 1, 1, 1)
    kl = torch.tensor([sk] * batch if klens is None else [min(max(int(n), 0), sk) for n in klens]).view(-1, 1, 1, 1)
    i, j = torch.arange(sq).view(1, 1, -1, 1), torch.arange(sk).view(1, 1, 1, -1)
    ok = (i < ql) & (j < kl)
    return ok & (j <= i + kl - ql) if causal else ok


def probabilities(q, k, scale, causal, mask, qlens, klens):
    """(p, lse, largest |score|) from q, k [batch, heads, sequence, channels]; k already has the heads of q."""
    s = q @ k.transpose(2, 3) * scale
    ok = allowed(q.shape[0], q.shape[2], k.shape[2], causal, qlens, klens)
    if mask is not None:
        if mask.dtype == torch.bool:
            ok = ok & mask
        else:
            s = s + torch.where(ok, mask.to(F), torch.zeros((), dtype=F))
    size = torch.where(ok & torch.isfinite(s), s.abs(), torch.zeros((), dtype=F)).amax()
    s = s.masked_fill(~ok, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None])
    return p, lse, float(size)


def used_keys(x, klens):
    """Keys or values [batch, heads, sequence, channels] with zeros behind the lengths (nothing there may count)."""
    if klens is None:
        return x
    x = x.clone()
    for b, n in enumerate(klens):
        x[b, :, max(int(n), 0):] = 0
    return x


def forward(q, k, v, layout="BSND", causal=False, scale=None, mask=None, qlens=None, klens=None):
    """dict of out, lse, and `spread` = sum_j p |v_j|, all in the layouts of the operator."""
    q, k, v = heads_of(q, layout), used_keys(heads_of(k, layout), klens), used_keys(heads_of(v, layout), klens)
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    scale = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    p, lse, size = probabilities(q, k, scale, causal, mask, qlens, klens)
    return {"out": back(p @ v, layout), "lse": lse, "spread": back(p @ v.abs(), layout), "size": size, "channels": q.shape[3]}


def forward_bound(r, dtype):
    """|computed - r["out"]|: probabilities rounded (u each), the result rounded (u), and what float32 does to the scores: a
    score is a float32 sum of `channels` products and an exponent of 2, both off by 2^-24 of at most (channels + 4) terms'
    size: 2^-24 (channels + 4) (size + 1) relative in every probability, twice (in the sum too)."""
    u = half_step(dtype)
    noise = 2.0 ** -23 * (r["channels"] + 4) * (r["size"] + 1)
    tiny = 2.0 ** -24 if dtype == "float16" else 0.0   # the steps of the smallest float16, in probabilities and result
    return (u + noise) * 1.01 * r["spread"] + u * r["out"].abs() * 1.01 + tiny * (1 + r["spread"]) * 64 + 1e-30


def lse_bound(r):
    return 2.0 ** -23 * (r["channels"] + 8) * (r["size"] + 1)


def gradient(dout, q, k, v, out, lse, layout="BSND", causal=False, scale=None, mask=None, qlens=None, klens=None):
    """dq, dk, dv from the result and its lse as given (rounded), with bounds' sums: for each gradient sum |p or ds| |other|."""
    dout, q, out = (heads_of(x, layout) for x in (dout, q, out))
    k, v = used_keys(heads_of(k, layout), klens), used_keys(heads_of(v, layout), klens)
    hkv = k.shape[1]
    group = q.shape[1] // hkv
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    scale = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    p, _, size = probabilities(q, k, scale, causal, mask, qlens, klens)
    if qlens is not None:   # rows behind the lengths are not read
        dout, q, out = dout.clone(), q.clone(), out.clone()
        for b, n in enumerate(qlens):
            dout[b, :, max(int(n), 0):] = 0
            out[b, :, max(int(n), 0):] = 0
            q[b, :, max(int(n), 0):] = 0
    dp = dout @ v.transpose(2, 3)
    delta = (dout * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    rough = p * (dout.abs() @ v.abs().transpose(2, 3) + (dout * out).abs().sum(-1, keepdim=True))   # sizes before cancelling

    def shared(x):
        return x.view(x.shape[0], hkv, group, x.shape[2], x.shape[3]).sum(2)

    t = lambda x: x.transpose(2, 3)   # noqa: E731
    grads = {"dq": ds @ k * scale, "dk": shared(t(ds) @ q * scale), "dv": shared(t(p) @ dout)}
    sums = {"dq": ds.abs() @ k.abs() * scale, "dk": shared(t(ds.abs()) @ q.abs() * scale), "dv": shared(t(p) @ dout.abs())}
    roughs = {"dq": rough @ k.abs() * scale, "dk": shared(t(rough) @ q.abs() * scale), "dv": sums["dv"]}
    # absolute steps of the smallest float16: of p (2^-25 each), and of ds lifted so that the largest |dout| is at least 1/2
    # (per row for dq, over the rows of a key head for dk)
    seen = (p > 0).to(F)
    top = dout.abs().amax()
    steps = {"dq": seen @ k.abs() * scale * dout.abs().amax(-1, keepdim=True).clamp(max=1) * 2,
             "dk": shared(t(seen) @ q.abs() * scale) * top.clamp(max=1) * 2, "dv": shared(t(seen) @ dout.abs())}
    return {n: {"exact": back(grads[n], layout), "sum": back(sums[n], layout), "rough": back(roughs[n], layout), "steps": back(steps[n], layout)}
            for n in grads}, size


def gradient_bound(r, dtype, size, channels):
    """Rounded probabilities or their gradients (u each), the rounded result (u), float32 in scores, products and delta."""
    u = half_step(dtype)
    noise = 2.0 ** -23 * (channels + 8) * (size + 2)
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0
    result = 2.0 ** -25 if dtype == "float16" else 0.0
    return 1.01 * (u * r["sum"] + noise * r["rough"] + u * r["exact"].abs() + tiny * r["steps"]) + result + 1e-30


def rotary(x, positions, layout="BSND", base=10000.0, rotary_dims=0, interleaved=False, inverse=False, scaling=None, magnitude=1.0):
    x = x.to(F) if layout == "BSND" else x.to(F).transpose(1, 2)
    r = rotary_dims or x.shape[3]
    w = base ** (-2.0 * torch.arange(r // 2, dtype=F) / r)
    if scaling and scaling["kind"] == "linear":
        w = w / scaling["factor"]
    elif scaling:
        out = []
        for rate in w.tolist():
            turns = scaling["original_length"] * rate / (2 * math.pi)
            share = min(1.0, max(0.0, (turns - scaling["low"]) / (scaling["high"] - scaling["low"])))
            out.append((1 - share) * rate / scaling["factor"] + share * rate)
        w = torch.tensor(out, dtype=F)
    angle = (positions.to(F)[..., None] * w)[..., None, :]
    if positions.dim() == 1:
        angle = angle[None]
    cos, sin = torch.cos(angle) * magnitude, torch.sin(angle) * (-magnitude if inverse else magnitude)
    y = x.clone()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    c, d = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = c, d
    else:
        y[..., :r // 2], y[..., r // 2:r] = c, d
    return y if layout == "BSND" else y.transpose(1, 2)


def dense_cache(cache, scale, table, length, page):
    """[key heads, tokens, channels] of one sequence; tokens of entries outside the pool are None in the second result."""
    parts, live = [], []
    for p in table[:-(-length // page)].tolist():
        inside = 0 <= p < cache.shape[0]
        parts.append(cache[p].to(F) * scale[p].to(F)[:, None, None] if inside else torch.zeros(cache.shape[1:], dtype=F))
        live += [inside] * page
    if not parts:
        return torch.zeros((cache.shape[1], 0, cache.shape[3]), dtype=F), torch.zeros(0, dtype=torch.bool)
    return torch.cat(parts, 1)[:, :length], torch.tensor(live)[:length]


def cache_attention(q, key_cache, value_cache, key_scale, value_scale, table, lengths, scale=None):
    batch, sq, h, dim = q.shape
    hkv, page = key_cache.shape[1], key_cache.shape[2]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out, spread, size = torch.zeros(q.shape, dtype=F), torch.zeros(q.shape, dtype=F), 0.0
    top = torch.zeros(q.shape, dtype=F)
    for b in range(batch):
        n = min(max(int(lengths[b]), 0), table.shape[1] * page)
        k, live = dense_cache(key_cache, key_scale, table[b], n, page)
        v, _ = dense_cache(value_cache, value_scale, table[b], n, page)
        k, v = k.repeat_interleave(h // hkv, 0), v.repeat_interleave(h // hkv, 0)
        for i in range(sq):
            seen = min(max(n - sq + 1 + i, 0), n)
            ok = live[:seen]
            if not bool(ok.any()):
                continue
            s = (k[:, :seen] @ q[b, i].to(F)[..., None])[..., 0] * scale
            size = max(size, float(s.abs().amax()))
            p = torch.softmax(s.masked_fill(~ok, -math.inf), -1)[:, None]
            out[b, i], spread[b, i] = (p @ v[:, :seen])[:, 0], (p @ v[:, :seen].abs())[:, 0]
            top[b, i] = v[:, :seen].abs().amax(1).amax(-1, keepdim=True)
    return {"out": out, "spread": spread, "size": size, "channels": dim, "top": top}


def cache_bound(r, dtype):
    """As forward_bound, with probabilities in float16 whatever the type of the queries: 2^-11 each, and relative to the
    largest scale of the values steps of 2^-25 (`top` is the largest value of the row); bfloat16 queries are exact in float16
    down to 2^-14 of the row's largest, below that off by 2^-25 of it: channels 2^-25 of the largest possible score."""
    u = half_step(dtype)
    noise = 2.0 ** -23 * (r["channels"] + 4) * (r["size"] + 1)
    return (2.0 ** -11 + noise) * 1.01 * r["spread"] + u * r["out"].abs() * 1.01 + 2.0 ** -24 * r["top"] * 4096 + (2.0 ** -25 if dtype == "float16" else 1e-30)
