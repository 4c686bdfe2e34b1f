"""The operators of an attention layer whose time is measured: rotary positions, attention that keeps no probabilities,
its gradient, and attention over a cache held in 8 bits.

`listed()` names calls from the smallest to the largest, `draw(rng)` gives more of the same ranges, `prepare` builds what
a program holds before the call (compiled kernel, inputs, output tensors), `run` is one pass: where `own` is true the
launch of the compiled description, else the same mathematics in elementary torch operations in 32 bits. `work` counts
every input read once and every output written once, and the products that the allowed pairs of query and key need.
`exact` is the definition in 64 bits.
"""
import json
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
SIZES = {"bfloat16": 2, "float16": 2, "float32": 4}


def listed():
    return [
        # one decoding step of 16 sequences far into a long context: queries and shared keys, frequencies scaled by wavelength
        {"name": "rotary_step", "kind": "rotary", "batch": 16, "seq": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "inverse": False, "scaling": "wavelength", "far": 100000, "dtype": "bfloat16"},
        # the gradient in float32 of adjacent pairs in the front part of every head, an odd number of tokens
        {"name": "rotary_part_grad", "kind": "rotary", "batch": 2, "seq": 1021, "heads": 12, "kv_heads": 0, "dim": 96, "rotary": 64,
         "interleaved": True, "inverse": True, "scaling": "linear", "far": 0, "dtype": "float32"},
        # a training batch: 16384 tokens
        {"name": "rotary_train", "kind": "rotary", "batch": 4, "seq": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "inverse": False, "scaling": "none", "far": 0, "dtype": "bfloat16"},
        # an encoder over a padded batch of short texts, no causal order
        {"name": "attention_short", "kind": "attention", "batch": 8, "q": 77, "k": 77, "heads": 12, "kv_heads": 12, "dim": 64,
         "causal": False, "mask": False, "lengths": True, "dtype": "float16"},
        # one token of each of 8 sequences over a cache of ordinary precision (the work is split along the keys)
        {"name": "attention_token", "kind": "attention", "batch": 8, "q": 1, "k": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "causal": True, "mask": False, "lengths": True, "dtype": "bfloat16"},
        # scores with an additive bias, as the attention probabilities of this repository take them, odd lengths
        {"name": "attention_bias", "kind": "attention", "batch": 4, "q": 1000, "k": 1003, "heads": 16, "kv_heads": 16, "dim": 64,
         "causal": False, "mask": True, "lengths": False, "dtype": "float16"},
        # a training or prefill layer, heads that share keys
        {"name": "attention_train", "kind": "attention", "batch": 2, "q": 4096, "k": 4096, "heads": 32, "kv_heads": 8, "dim": 128,
         "causal": True, "mask": False, "lengths": False, "dtype": "bfloat16"},
        # its gradient for a padded batch of short texts
        {"name": "grad_short", "kind": "grad", "batch": 8, "q": 200, "k": 200, "heads": 12, "kv_heads": 12, "dim": 64,
         "causal": True, "mask": False, "lengths": True, "dtype": "float16"},
        # and for the training layer
        {"name": "grad_train", "kind": "grad", "batch": 2, "q": 4096, "k": 4096, "heads": 32, "kv_heads": 8, "dim": 128,
         "causal": True, "mask": False, "lengths": False, "dtype": "bfloat16"},
        # one conversation of a few hundred tokens
        {"name": "cache_short", "kind": "cache", "batch": 1, "q": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "pages": 8,
         "dtype": "bfloat16"},
        # four drafted tokens at once for each of 16 sequences, small pages
        {"name": "cache_draft", "kind": "cache", "batch": 16, "q": 4, "heads": 16, "kv_heads": 4, "dim": 64, "page": 16, "pages": 125,
         "dtype": "float16"},
        # a serving batch of long conversations
        {"name": "cache_long", "kind": "cache", "batch": 32, "q": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "pages": 256,
         "dtype": "bfloat16"},
    ]


def _between(rng, low, high):
    """A whole number in [low, high], spread over the logarithm."""
    return int(min(max(round(math.exp(rng.uniform(math.log(low), math.log(high)))), low), high))


def draw(rng):
    kind = rng.choice(["rotary", "attention", "grad", "cache"])
    dtype = rng.choice(["bfloat16", "float16"])
    if kind == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        heads = rng.choice([1, 4, 8, 12, 16, 32])
        batch = _between(rng, 1, 16)
        return {"kind": kind, "batch": batch, "seq": _between(rng, 1, max(1, 16384 * 32 * 128 // (batch * heads * dim * 4))), "heads": heads,
                "kv_heads": rng.choice([0, 1, heads]), "dim": dim, "rotary": rng.choice([dim, dim // 2]), "interleaved": rng.random() < 0.5,
                "inverse": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "wavelength"]),
                "far": rng.choice([0, 10000, 1000000]), "dtype": rng.choice(["bfloat16", "float16", "float32"])}
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 8])
    if kind == "cache":
        page = rng.choice([16, 32, 64, 128])
        batch = _between(rng, 1, 32)
        return {"kind": kind, "batch": batch, "q": rng.choice([1, 1, 2, 4]), "heads": kv_heads * group, "kv_heads": kv_heads,
                "dim": rng.choice([64, 80, 96, 128]), "page": page, "pages": max(1, _between(rng, 64, 8192) // page), "dtype": dtype}
    most = 2 * 32 * 4096 * 4096 * 128 // 4   # a quarter of the largest listed pairs times channels
    dim = rng.choice([40, 64, 80, 96, 128])
    batch = _between(rng, 1, 8)
    k = _between(rng, 16, 8192)
    q = rng.choice([1, k, _between(rng, 2, 1024)]) if kind == "attention" else k
    q = max(1, min(q, most // (batch * kv_heads * group * dim * k)))
    if kind == "grad":
        q = k = max(1, min(k, int(math.sqrt(most / (batch * kv_heads * group * dim)))))
    mask = rng.random() < 0.25 and q * k * kv_heads * group <= 1 << 25
    return {"kind": kind, "batch": batch, "q": q, "k": k, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "causal": q <= k and rng.random() < 0.6, "mask": mask, "lengths": rng.random() < 0.4, "dtype": dtype}


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------
def _spread(low, high, count):
    """`count` whole numbers over [low, high], the last one `high`: the lengths of a batch."""
    return [low + int((high - low) * ((i + 1) * 0.6180339887 % 1.0)) for i in range(count - 1)] + [high]


def _lengths(case):
    """(query lengths, key lengths) of an attention case; a text that is padded is so on both sides."""
    q, k, batch = case["q"], case["k"], case["batch"]
    if not case["lengths"]:
        return [q] * batch, [k] * batch
    keys = _spread((k + 1) // 2, k, batch)
    return ([q] * batch if q != k else keys), keys


def _cache_lengths(case):
    capacity = case["page"] * case["pages"]
    return _spread(max(case["q"], capacity // 2), capacity, case["batch"])


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, factor=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * factor).to(DTYPES[dtype])


def _inputs(case, seed):
    """The input tensors of a case, by name."""
    g = _generator(seed)
    kind, dtype = case["kind"], case["dtype"]
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")   # noqa: E731
    if kind == "rotary":
        batch, seq, dim = case["batch"], case["seq"], case["dim"]
        first = torch.randint(0, case["far"] + 1, (batch, 1), generator=g, device="cuda", dtype=torch.int32)
        t = {"q": _normal(g, (batch, seq, case["heads"], dim), dtype)}
        if case["kv_heads"]:
            t["k"] = _normal(g, (batch, seq, case["kv_heads"], dim), dtype)
        t["positions"] = first + torch.arange(seq, device="cuda", dtype=torch.int32)
        return t
    if kind == "cache":
        batch, hkv, dim, page, pages = case["batch"], case["kv_heads"], case["dim"], case["page"], case["pages"]
        total = batch * pages
        shape = (total, hkv, page, dim)
        t = {"q": _normal(g, (batch, case["q"], case["heads"], dim), dtype)}
        for name in ("key", "value"):
            # what a block's quantisation leaves: a scale of its largest magnitude / 127
            t[name + "_cache"] = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
            t[name + "_scale"] = (torch.rand((total, hkv), generator=g, device="cuda") * 0.5 + 0.75) * (3.0 / 127.0)
        t["block_table"] = torch.randperm(total, generator=g, device="cuda").to(torch.int32).view(batch, pages)
        t["lengths"] = ints(_cache_lengths(case))
        return t
    batch, sq, sk, h, hkv, dim = (case[n] for n in ("batch", "q", "k", "heads", "kv_heads", "dim"))
    t = {"q": _normal(g, (batch, sq, h, dim), dtype, 2.0), "k": _normal(g, (batch, sk, hkv, dim), dtype),
         "v": _normal(g, (batch, sk, hkv, dim), dtype)}
    if case["mask"]:
        t["mask"] = torch.randn((1, h, sq, sk), generator=g, device="cuda")
        t["mask"][torch.rand((1, h, sq, sk), generator=g, device="cuda") < 0.1] = -math.inf
    if case["lengths"]:
        t["query_lengths"], t["key_lengths"] = (ints(v) for v in _lengths(case))
    if kind == "grad":
        t["dout"] = _normal(g, (batch, sq, h, dim), dtype)
    return t


# ---------------------------------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------------------------------
BASE = 500000.0
FACTOR = 8.0
BANDS = {"original_length": 8192, "low": 1.0, "high": 4.0}


def _description(case, t):
    """(text of the description, names of its inputs in order)."""
    from akg_amd import op_desc
    b = op_desc.DescBuilder("Layer_%s" % case["kind"])
    names = {torch.bfloat16: "bfloat16", torch.float16: "float16", torch.float32: "float32", torch.int32: "int32", torch.int8: "int8"}
    order, by_name = [], {}

    def given(name):
        if name not in t:
            return None
        if name not in by_name:
            by_name[name] = b.input(list(t[name].shape), names[t[name].dtype])
            order.append(name)
        return by_name[name]

    if case["kind"] == "rotary":
        scaling = {"none": None, "linear": {"kind": "linear", "factor": FACTOR},
                   "wavelength": dict(BANDS, kind="wavelength", factor=FACTOR)}[case["scaling"]]
        xs = [given(n) for n in ("q", "k") if n in t]
        outs = op_desc.rotary_embedding(b, xs, given("positions"), base=BASE, rotary_dims=case["rotary"],
                                        interleaved=case["interleaved"], inverse=case["inverse"], scaling=scaling)
    elif case["kind"] == "cache":
        outs = [op_desc.cache_attention(b, *[given(n) for n in ("q", "key_cache", "value_cache", "key_scale", "value_scale", "block_table",
                                                                 "lengths")])]
    elif case["kind"] == "attention":
        q, k, v = given("q"), given("k"), given("v")
        outs = op_desc.attention(b, q, k, v, mask=given("mask"), query_lengths=given("query_lengths"), key_lengths=given("key_lengths"),
                                 causal=case["causal"])
    else:
        dout, q, k, v, out, lse = (given(n) for n in ("dout", "q", "k", "v", "out", "lse"))
        outs = op_desc.attention_grad(b, dout, q, k, v, out, lse, mask=given("mask"), query_lengths=given("query_lengths"),
                                      key_lengths=given("key_lengths"), causal=case["causal"])
    return b.dumps(list(outs)), order


def prepare(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "grad":
        # what the forward pass left
        out, lse = _attention(case, t)
        t["out"], t["lse"] = out, lse
    state = {"case": case, "t": t}
    if own:
        from akg_amd import driver
        text, order = _description(case, t)
        kernel = driver.HipKernel(text)
        kernel.prepare()
        dtypes = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
        state["kernel"] = kernel
        state["inputs"] = [t[n] for n in order]
        state["outputs"] = [torch.empty(d.shape, dtype=dtypes[d.dtype], device="cuda") for d in kernel.outputs]
        state["arguments"] = state["inputs"] + state["outputs"]
    return state


def run(state):
    if own:
        state["kernel"].launch(state["arguments"])
        return state["outputs"]
    case, t = state["case"], state["t"]
    if case["kind"] == "rotary":
        return _rotary(case, t)
    if case["kind"] == "attention":
        return list(_attention(case, t))
    if case["kind"] == "grad":
        return _gradient(case, t)
    return [_cache(case, t)]


# ---------------------------------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _rotary(case, t):
    half = case["rotary"] // 2
    # angles in 64 bits: a position of a million turns a float32 angle by several hundredths
    w = BASE ** (-2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / case["rotary"])
    if case["scaling"] == "linear":
        w = w / FACTOR
    elif case["scaling"] == "wavelength":
        turns = BANDS["original_length"] * w / (2.0 * math.pi)
        ramp = ((turns - BANDS["low"]) / (BANDS["high"] - BANDS["low"])).clamp(0.0, 1.0)
        w = (1.0 - ramp) * w / FACTOR + ramp * w
    angle = t["positions"].to(torch.float64)[:, :, None, None] * w
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if case["inverse"]:
        sin = -sin
    outs = []
    for name in ("q", "k"):
        if name not in t:
            continue
        x = t[name].float()
        front, rest = x[..., :case["rotary"]], x[..., case["rotary"]:]
        if case["interleaved"]:
            a, b = front[..., 0::2], front[..., 1::2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        else:
            a, b = front[..., :half], front[..., half:]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        outs.append(torch.cat((turned, rest), dim=-1).to(t[name].dtype))
    return outs


def _hidden(case, t, i):
    """True where item i's queries may not see its keys, [q, k]."""
    sq, sk = case["q"], case["k"]
    rows = torch.arange(sq, device="cuda")[:, None]
    cols = torch.arange(sk, device="cuda")[None, :]
    if case["lengths"]:
        ql, kl = t["query_lengths"][i], t["key_lengths"][i]
    else:
        ql, kl = sq, sk
    hidden = (rows >= ql) | (cols >= kl)
    if case["causal"]:
        hidden = hidden | (cols > rows + (kl - ql))
    return hidden


def _scores(case, t, i):
    """Scores of item i in float32, [heads, q, k], -inf where hidden."""
    group = case["heads"] // case["kv_heads"]
    q = t["q"][i].float().transpose(0, 1).contiguous()
    k = t["k"][i].float().transpose(0, 1).repeat_interleave(group, 0).transpose(1, 2).contiguous()
    s = torch.matmul(q, k) * (1.0 / math.sqrt(case["dim"]))
    if case["mask"]:
        s = s + t["mask"][0]
    return s.masked_fill(_hidden(case, t, i), -math.inf)


def _attention(case, t):
    group = case["heads"] // case["kv_heads"]
    outs, sums = [], []
    for i in range(case["batch"]):
        s = _scores(case, t, i)
        top = s.amax(dim=-1, keepdim=True)
        e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = e.sum(dim=-1, keepdim=True)
        v = t["v"][i].float().transpose(0, 1).repeat_interleave(group, 0).contiguous()
        o = torch.matmul(e, v) / torch.where(total == 0, torch.ones_like(total), total)
        outs.append(o.transpose(0, 1).to(t["q"].dtype))
        sums.append((top + torch.log(total))[..., 0])
    return torch.stack(outs), torch.stack(sums)


def _gradient(case, t):
    h, hkv, dim = case["heads"], case["kv_heads"], case["dim"]
    group = h // hkv
    scale = 1.0 / math.sqrt(dim)
    grads = ([], [], [])
    for i in range(case["batch"]):
        lse = t["lse"][i][..., None]
        p = torch.exp(_scores(case, t, i) - torch.where(lse == -math.inf, torch.zeros_like(lse), lse))
        head = lambda x: x[i].float().transpose(0, 1)   # noqa: E731
        q, dout, out = head(t["q"]).contiguous(), head(t["dout"]).contiguous(), head(t["out"])
        k, v = head(t["k"]).repeat_interleave(group, 0).contiguous(), head(t["v"]).repeat_interleave(group, 0)
        dv = torch.matmul(p.transpose(1, 2).contiguous(), dout)
        dp = torch.matmul(dout, v.transpose(1, 2).contiguous())
        ds = p * (dp - (dout * out).sum(dim=-1, keepdim=True)) * scale
        dq = torch.matmul(ds, k)
        dk = torch.matmul(ds.transpose(1, 2).contiguous(), q)
        for kept, x in zip(grads, (dq, dk.view(hkv, group, -1, dim).sum(1), dv.view(hkv, group, -1, dim).sum(1))):
            kept.append(x.transpose(0, 1).to(t["q"].dtype))
    return [torch.stack(x) for x in grads]


def _cache(case, t):
    batch, sq, h, hkv, dim, page, pages = (case[n] for n in ("batch", "q", "heads", "kv_heads", "dim", "page", "pages"))
    group, tokens = h // hkv, page * pages
    table = t["block_table"].long()

    def dense(name):   # [batch, kv heads, tokens, dim]
        x = t[name + "_cache"][table].float() * t[name + "_scale"][table][..., None, None]
        return x.transpose(1, 2).reshape(batch, hkv, tokens, dim)

    q = t["q"].float().view(batch, sq, hkv, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, hkv, sq * group, dim).contiguous()
    s = torch.matmul(q, dense("key").transpose(2, 3).contiguous()) * (1.0 / math.sqrt(dim))
    last = t["lengths"][:, None] - sq + torch.arange(sq, device="cuda")            # the last key each query sees
    hidden = torch.arange(tokens, device="cuda") > last.repeat_interleave(group, 1)[..., None]
    s = s.masked_fill(hidden[:, None], -math.inf)
    e = torch.exp(s - s.amax(dim=-1, keepdim=True))
    o = torch.matmul(e, dense("value")) / e.sum(dim=-1, keepdim=True)
    return o.view(batch, hkv, sq, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, sq, h, dim).to(t["q"].dtype)


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def _pairs(case):
    """Pairs of query and key that see each other, over the batch, for one head."""
    total = 0
    for ql, kl in zip(*_lengths(case)):
        if not case["causal"]:
            total += ql * kl
            continue
        # query i sees the first kl - ql + i + 1 keys
        first = kl - ql + 1
        low = max(0, 1 - first)
        n = max(0, ql - low)
        total += n * (first + low) + n * (n - 1) // 2
    return total


def work(case):
    kind, e = case["kind"], SIZES[case["dtype"]]
    if kind == "rotary":
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["dim"] * e + 4 * tokens, "flops": 3 * n * case["rotary"]}
    if kind == "cache":
        h, hkv, dim = case["heads"], case["kv_heads"], case["dim"]
        lengths = _cache_lengths(case)
        blocks = sum(-(-n // case["page"]) for n in lengths)
        q = case["batch"] * case["q"] * h * dim
        return {"bytes": 2 * sum(lengths) * hkv * dim + 2 * blocks * hkv * 4 + 4 * blocks + 4 * case["batch"] + 2 * q * e,
                "flops": 4 * dim * h * sum(case["q"] * n - case["q"] * (case["q"] - 1) // 2 for n in lengths)}
    h, hkv, dim = case["heads"], case["kv_heads"], case["dim"]
    ql, kl = _lengths(case)
    q = sum(ql) * h * dim
    kv = sum(kl) * hkv * dim
    rows = case["batch"] * case["q"] * h
    mask = 4 * h * case["q"] * case["k"] if case["mask"] else 0
    lengths = 8 * case["batch"] if case["lengths"] else 0
    full = rows * dim
    if kind == "attention":
        return {"bytes": (q + 2 * kv + full) * e + 4 * rows + mask + lengths, "flops": 4 * dim * h * _pairs(case)}
    full_kv = case["batch"] * case["k"] * hkv * dim
    return {"bytes": (3 * q + 2 * kv + full + 2 * full_kv) * e + 4 * rows + mask + lengths, "flops": 10 * dim * h * _pairs(case)}


# ---------------------------------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    t = _inputs(case, seed)
    f = torch.float64
    kind = case["kind"]
    if kind == "rotary":
        r = case["rotary"]
        rates = []
        for i in range(r // 2):
            w = BASE ** (-2.0 * i / r)
            if case["scaling"] == "linear":
                w /= FACTOR
            elif case["scaling"] == "wavelength":
                length = 2.0 * math.pi / w
                if length > BANDS["original_length"] / BANDS["low"]:
                    w /= FACTOR
                elif length >= BANDS["original_length"] / BANDS["high"]:
                    share = (BANDS["original_length"] / length - BANDS["low"]) / (BANDS["high"] - BANDS["low"])
                    w = (1.0 - share) * (w / FACTOR) + share * w
            rates.append(-w if case["inverse"] else w)
        turn = torch.polar(torch.ones((), dtype=f, device="cuda"),
                           t["positions"].to(f).unsqueeze(-1) * torch.tensor(rates, dtype=f, device="cuda")).unsqueeze(2)
        outs = []
        for name in [n for n in ("q", "k") if n in t]:
            y = t[name].to(f).clone()
            pair = (y[..., 0:r:2], y[..., 1:r:2]) if case["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
            z = torch.complex(pair[0].contiguous(), pair[1].contiguous()) * turn
            pair[0].copy_(z.real)
            pair[1].copy_(z.imag)
            outs.append(y)
        return outs
    if kind == "cache":
        out = torch.zeros_like(t["q"], dtype=f)
        group = case["heads"] // case["kv_heads"]
        table = t["block_table"].tolist()
        for i, n in enumerate(_cache_lengths(case)):
            pages = torch.tensor(table[i][:-(-n // case["page"])], device="cuda")
            for j in range(case["kv_heads"]):
                k, v = ((t[x + "_cache"][pages, j].to(f) * t[x + "_scale"][pages, j].to(f)[:, None, None]).flatten(0, 1) for x in ("key", "value"))
                for row in range(case["q"]):
                    seen = n - case["q"] + row + 1
                    q = t["q"][i, row, j * group:(j + 1) * group].to(f)
                    p = torch.softmax(q @ k[:seen].T.contiguous() / math.sqrt(case["dim"]), dim=-1)
                    out[i, row, j * group:(j + 1) * group] = p @ v[:seen]
        return [out]
    group = case["heads"] // case["kv_heads"]
    out, lse = torch.zeros_like(t["q"], dtype=f), torch.full((case["batch"], case["heads"], case["q"]), -math.inf, dtype=f, device="cuda")
    dq, dk, dv = (torch.zeros_like(t[n], dtype=f) for n in ("q", "k", "v"))
    scale = case["dim"] ** -0.5
    for i, (ql, kl) in enumerate(zip(*_lengths(case))):
        for j in range(case["heads"]):
            q, k, v = t["q"][i, :ql, j].to(f), t["k"][i, :kl, j // group].to(f), t["v"][i, :kl, j // group].to(f)
            s = q @ k.T.contiguous() * scale
            if case["mask"]:
                s += t["mask"][0, j, :ql, :kl]
            if case["causal"]:
                s[torch.ones_like(s, dtype=torch.bool).triu(kl - ql + 1)] = -math.inf
            sums = torch.logsumexp(s, dim=-1)
            p = torch.exp(s - sums.clamp(min=-1e300)[:, None])
            o = p @ v
            out[i, :ql, j], lse[i, j, :ql] = o, sums
            if kind == "grad":
                do = t["dout"][i, :ql, j].to(f)
                dv[i, :kl, j // group] += p.T.contiguous() @ do
                ds = p * (do @ v.T.contiguous() - (do * o).sum(-1, keepdim=True))
                dq[i, :ql, j] = ds @ k * scale
                dk[i, :kl, j // group] += ds.T.contiguous() @ q * scale
    return [dq, dk, dv] if kind == "grad" else [out, lse]
