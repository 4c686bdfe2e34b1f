"""The operators of a layer of linear attention whose time is measured: rotary positions of several axes, linear attention with
a decay for each head over prompts, the same over single tokens, and its gradient.

`listed()` names calls from the smallest to the largest, `draw(rng)` gives more of the same ranges, `prepare` builds what
a program holds before the call (compiled kernel, inputs, output tensors), `run` is one pass: where `own` is true the
launch of the compiled description, else the same mathematics in elementary torch operations in 32 bits. `work` counts
every input read once and every output written once, and the products of the recurrence. `exact` is the definition in 64
bits, token by token.
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
SIZES = {"bfloat16": 2, "float16": 2, "float32": 4}


def listed():
    return [
        # one decoding step of 16 sequences that hold images: time, height and width, axes dealt pair by pair
        {"name": "axes_step", "kind": "axes", "batch": 16, "seq": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "axes": 3,
         "order": "cycle", "rates": "shared", "interleaved": False, "inverse": False, "dtype": "bfloat16"},
        # a training batch of video: 16384 tokens, a block of pairs for every axis
        {"name": "axes_train", "kind": "axes", "batch": 4, "seq": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "axes": 3,
         "order": "blocks", "rates": "shared", "interleaved": False, "inverse": False, "dtype": "bfloat16"},
        # one token of one conversation
        {"name": "token_one", "kind": "linear", "batch": 1, "seq": 1, "heads": 16, "kv_heads": 16, "dim": 128, "value_dim": 128,
         "state": True, "lengths": False, "dtype": "bfloat16"},
        # four drafted tokens for each of 16 sequences, heads that share keys
        {"name": "token_draft", "kind": "linear", "batch": 16, "seq": 4, "heads": 16, "kv_heads": 4, "dim": 64, "value_dim": 64,
         "state": True, "lengths": False, "dtype": "float16"},
        # one token for each sequence of a large serving batch: 64 x 32 states
        {"name": "token_batch", "kind": "linear", "batch": 64, "seq": 1, "heads": 32, "kv_heads": 32, "dim": 128, "value_dim": 128,
         "state": True, "lengths": False, "dtype": "bfloat16"},
        # an encoder's padded batch of short texts
        {"name": "linear_short", "kind": "linear", "batch": 8, "seq": 77, "heads": 12, "kv_heads": 12, "dim": 64, "value_dim": 64,
         "state": False, "lengths": True, "dtype": "float16"},
        # a prompt that continues a conversation, odd sizes, heads that share keys
        {"name": "linear_odd", "kind": "linear", "batch": 4, "seq": 1003, "heads": 16, "kv_heads": 4, "dim": 96, "value_dim": 80,
         "state": True, "lengths": True, "dtype": "bfloat16"},
        # one long prompt (the work is split along its tokens), its last state kept
        {"name": "linear_prompt", "kind": "linear", "batch": 1, "seq": 16384, "heads": 16, "kv_heads": 16, "dim": 128, "value_dim": 128,
         "state": True, "lengths": False, "dtype": "bfloat16"},
        # a training layer
        {"name": "linear_train", "kind": "linear", "batch": 4, "seq": 4096, "heads": 32, "kv_heads": 32, "dim": 128, "value_dim": 128,
         "state": False, "lengths": False, "dtype": "bfloat16"},
        # the gradient for a padded batch of short texts
        {"name": "grad_short", "kind": "grad", "batch": 8, "seq": 200, "heads": 12, "kv_heads": 12, "dim": 64, "value_dim": 64,
         "state": False, "lengths": True, "dtype": "float16"},
        # one piece of a long text whose state goes on, heads that share keys, odd lengths
        {"name": "grad_shared", "kind": "grad", "batch": 2, "seq": 1021, "heads": 16, "kv_heads": 4, "dim": 128, "value_dim": 128,
         "state": True, "lengths": True, "dtype": "bfloat16"},
        # the training layer's gradient
        {"name": "grad_train", "kind": "grad", "batch": 4, "seq": 4096, "heads": 32, "kv_heads": 32, "dim": 128, "value_dim": 128,
         "state": False, "lengths": False, "dtype": "bfloat16"},
    ]


def _between(rng, low, high):
    """A whole number in [low, high], spread over the logarithm."""
    return int(min(max(round(math.exp(rng.uniform(math.log(low), math.log(high)))), low), high))


def draw(rng):
    kind = rng.choice(["axes", "token", "linear", "linear", "grad"])
    dtype = rng.choice(["bfloat16", "float16"])
    if kind == "axes":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        heads = rng.choice([1, 4, 8, 12, 16, 32])
        batch = _between(rng, 1, 16)
        return {"kind": kind, "batch": batch, "seq": _between(rng, 1, max(1, 16384 * 32 * 128 // (batch * heads * dim * 4))), "heads": heads,
                "kv_heads": rng.choice([0, 1, heads]), "dim": dim, "rotary": rng.choice([dim, dim // 2]), "axes": rng.choice([2, 3]),
                "order": rng.choice(["blocks", "cycle"]), "rates": rng.choice(["shared", "own"]), "interleaved": rng.random() < 0.5,
                "inverse": rng.random() < 0.5, "dtype": rng.choice(["bfloat16", "float16", "float32"])}
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    dim = rng.choice([32, 40, 64, 80, 96, 128, 192, 256])
    value_dim = rng.choice([dim, dim, dim, 64, 128])
    state = rng.random() < 0.5
    if kind == "token":
        return {"kind": "linear", "batch": max(1, min(_between(rng, 1, 256), 64 * 32 * 128 * 128 // (heads * dim * value_dim))),
                "seq": rng.choice([1, 1, 1, 2, 3, 5]), "heads": heads, "kv_heads": kv_heads, "dim": dim, "value_dim": value_dim, "state": True,
                "lengths": False, "dtype": dtype}
    batch = _between(rng, 1, 8)
    most = 4 * 4096 * 32 * 128 * 128 // (4 if kind == "grad" else 2)
    seq = max(1, min(_between(rng, 16, 16384), most // (batch * heads * dim * value_dim), 4 * 4096 * 32 * 128 // (2 * batch * heads * max(dim, value_dim))))
    return {"kind": kind, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim, "value_dim": value_dim, "state": state,
            "lengths": rng.random() < 0.4, "dtype": dtype}


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------
BASE = 10000.0


def _sections(case):
    """Pairs of every axis: a quarter for time, the rest for height and width, or two halves."""
    pairs = case["rotary"] // 2
    first = pairs // 4 if case["axes"] == 3 else pairs - pairs // 2
    rest = pairs - first
    return [first, rest] if case["axes"] == 2 else [first, rest - rest // 2, rest // 2]


def _lengths(case):
    """Lengths spread over [half, whole], the last one whole."""
    seq, batch = case["seq"], case["batch"]
    if not case["lengths"]:
        return [seq] * batch
    return [seq // 2 + int((seq - seq // 2) * ((i + 1) * 0.6180339887 % 1.0)) for i in range(batch - 1)] + [seq]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, factor=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * factor).to(DTYPES[dtype])


def _inputs(case, seed):
    """The input tensors of a case, by name."""
    g = _generator(seed)
    dtype = case["dtype"]
    batch, seq, h, hkv, dim = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    if case["kind"] == "axes":
        t = {"q": _normal(g, (batch, seq, h, dim), dtype)}
        if hkv:
            t["k"] = _normal(g, (batch, seq, hkv, dim), dtype)
        # frames of 32 x 32 patches, from some frame on; with two axes the rows and columns of one picture
        at = torch.arange(seq, device="cuda") + torch.randint(0, 100000, (batch, 1), generator=g, device="cuda")
        axes = [at // 1024, at // 32 % 32, at % 32] if case["axes"] == 3 else [at // 32, at % 32]
        t["positions"] = torch.stack(axes).to(torch.int32)
        return t
    value_dim = case["value_dim"]
    t = {"q": _normal(g, (batch, seq, h, dim), dtype), "k": _normal(g, (batch, seq, hkv, dim), dtype),
         "v": _normal(g, (batch, seq, hkv, value_dim), dtype)}
    # heads that remember from some 30 to some 4000 tokens
    reach = 5.0 + 7.0 * (torch.arange(h, device="cuda") + torch.rand((h,), generator=g, device="cuda")) / h
    t["log_decay"] = torch.log1p(-torch.exp2(-reach))
    if case["state"]:
        # as some hundred tokens leave it
        t["state"] = torch.randn((batch, h, dim, value_dim), generator=g, device="cuda") * 8.0
    if case["lengths"]:
        t["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    if case["kind"] == "grad":
        t["dout"] = _normal(g, (batch, seq, h, value_dim), dtype)
        if case["state"]:
            t["dstate"] = torch.randn((batch, h, dim, value_dim), generator=g, device="cuda")
    return t


# ---------------------------------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------------------------------
def _description(case, t):
    """(text of the description, names of its inputs in order)."""
    from akg_amd import op_desc
    b = op_desc.DescBuilder("Layer_%s" % case["kind"])
    names = {v: k for k, v in DTYPES.items()}
    names[torch.int32] = "int32"
    order, by_name = [], {}

    def given(name):
        if name not in t:
            return None
        if name not in by_name:
            by_name[name] = b.input(list(t[name].shape), names[t[name].dtype])
            order.append(name)
        return by_name[name]

    if case["kind"] == "axes":
        xs = [given(n) for n in ("q", "k") if n in t]
        outs = op_desc.rotary_embedding(b, xs, given("positions"), base=BASE, rotary_dims=case["rotary"], interleaved=case["interleaved"],
                                        inverse=case["inverse"], sections=_sections(case), axis_order=case["order"], axis_rates=case["rates"])
    elif case["kind"] == "linear":
        outs = op_desc.linear_attention(b, given("q"), given("k"), given("v"), given("log_decay"), state=given("state"),
                                        lengths=given("lengths"), last_state=case["state"])
    else:
        outs = op_desc.linear_attention_grad(b, given("dout"), given("q"), given("k"), given("v"), given("log_decay"), state=given("state"),
                                             dstate=given("dstate"), lengths=given("lengths"))
    return b.dumps(list(outs)), order


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "t": t}
    if own:
        from akg_amd import driver
        text, order = _description(case, t)
        kernel = driver.HipKernel(text)
        kernel.prepare()
        state["kernel"] = kernel
        state["outputs"] = [torch.empty(d.shape, dtype=DTYPES[d.dtype], device="cuda") for d in kernel.outputs]
        state["arguments"] = [t[n] for n in order] + state["outputs"]
    return state


def run(state):
    if own:
        state["kernel"].launch(state["arguments"])
        return state["outputs"]
    case, t = state["case"], state["t"]
    if case["kind"] == "axes":
        return _axes(case, t)
    if case["kind"] == "grad":
        return _gradient(case, t)
    return _linear(case, t)


# ---------------------------------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _axes(case, t):
    r, sections = case["rotary"], _sections(case)
    half = r // 2
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    if case["order"] == "cycle":
        # the j-th pair of every axis before the (j + 1)-th of any
        turn = torch.cat([torch.arange(n) for n in sections])
        axis = axis[torch.argsort(turn * len(sections) + axis)]
    index = torch.arange(half, dtype=torch.float64)
    if case["rates"] == "own":
        nth = torch.stack([(axis == a).cumsum(0) - 1 for a in range(len(sections))])[axis, torch.arange(half)]
        rate = BASE ** (-nth.to(torch.float64) / torch.tensor(sections, dtype=torch.float64)[axis])
    else:
        rate = BASE ** (-2.0 * index / r)
    # angles in 64 bits: a position of a hundred thousand turns a float32 angle by some thousandths
    angle = t["positions"][axis.cuda()].permute(1, 2, 0).to(torch.float64)[:, :, None, :] * rate.cuda()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if case["inverse"]:
        sin = -sin
    outs = []
    for name in ("q", "k"):
        if name not in t:
            continue
        x = t[name].float()
        front, rest = x[..., :r], x[..., r:]
        if case["interleaved"]:
            a, b = front[..., 0::2], front[..., 1::2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        else:
            a, b = front[..., :half], front[..., half:]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        outs.append(torch.cat((turned, rest), dim=-1).to(t[name].dtype))
    return outs


CHUNK = 64


def _walk(case, a, b, c, log_decay, lengths, start):
    """out[i] = a[i] . S[i], S[i] = decay S[i-1] + b[i] c[i]^T from S[-1] = `start`, for a, b, c [batch, heads, tokens,
    channels] with zeros behind the lengths; and S after the last token. Chunks of tokens, all at once: inside a chunk as
    masked products, before it from the states that the chunks in front of it add up to."""
    batch, h, seq, _ = a.shape
    size = min(CHUNK, seq)
    n = -(-seq // size)
    pad = lambda x: torch.nn.functional.pad(x, (0, 0, 0, n * size - seq)).view(batch, h, n, size, x.shape[-1])   # noqa: E731
    a, b, c = pad(a), pad(b), pad(c)
    g = log_decay[:, None, None]
    steps = torch.arange(size, device="cuda")
    back = (steps[:, None] - steps).float()
    weight = torch.where(back >= 0, torch.exp(g * back.clamp(min=0)), torch.zeros_like(back))          # [h, i, j]
    scores = torch.matmul(a, b.transpose(-1, -2).contiguous()) * weight[:, None]
    inside = torch.matmul(scores, c)
    fade = torch.exp(log_decay[:, None] * (size - 1 - steps))[:, None, :, None]
    added = torch.matmul((b * fade).transpose(-1, -2).contiguous(), c)                                  # [batch, h, n, D, E]
    chunks = torch.arange(n, device="cuda")
    gap = (chunks[:, None] - 1 - chunks).float()
    across = torch.where(gap >= 0, torch.exp(g * size * gap.clamp(min=0)), torch.zeros_like(gap))      # [h, n, n]
    before = torch.matmul(across, added.flatten(-2)).view_as(added)
    if start is not None:
        before = before + torch.exp(log_decay[:, None] * size * chunks)[:, :, None, None] * start[:, :, None]
    grown = torch.exp(log_decay[:, None] * (steps + 1))[:, None, :, None]
    out = (inside + torch.matmul(a, before) * grown).view(batch, h, n * size, -1)[:, :, :seq]
    # the state after the last token: that before its chunk, and the chunk's tokens up to it
    last = (lengths.clamp(min=1) - 1) // size
    one = torch.arange(batch, device="cuda")
    left = lengths - last * size                                                                       # [batch]
    age = (left[:, None] - 1 - steps)[:, None]                                                          # [batch, 1, size]
    fade = torch.where(age >= 0, torch.exp(log_decay[:, None] * age.clamp(min=0)), torch.zeros((), device="cuda"))
    state = torch.matmul((b[one, :, last] * fade[..., None]).transpose(-1, -2).contiguous(), c[one, :, last])
    state = state + torch.exp(log_decay * left[:, None])[..., None, None] * before[one, :, last]
    return out, state


def _heads(x, case, live):
    """[batch, tokens, heads, channels] as float32 [batch, all heads, tokens, channels], zeros behind the lengths."""
    x = x.float().transpose(1, 2)
    if x.shape[1] != case["heads"]:
        x = x.repeat_interleave(case["heads"] // x.shape[1], 1)
    return torch.where(live, x, torch.zeros((), device="cuda")).contiguous()


def _alive(case, t):
    lengths = t["lengths"].long() if case["lengths"] else torch.full((case["batch"],), case["seq"], device="cuda")
    return lengths, (torch.arange(case["seq"], device="cuda") < lengths[:, None])[:, None, :, None]


def _linear(case, t):
    if case["seq"] == 1 and case["state"] and not case["lengths"]:
        # a single token: the recurrence
        group = case["heads"] // case["kv_heads"]
        q, k, v = (t[n][:, 0].float() for n in ("q", "k", "v"))
        k, v = (x.repeat_interleave(group, 1) if group > 1 else x for x in (k, v))
        state = t["state"] * torch.exp(t["log_decay"])[:, None, None] + k[..., :, None] * v[..., None, :]
        out = (q[..., :, None] * state).sum(-2) * case["dim"] ** -0.5
        return [out[:, None].to(t["q"].dtype), state]
    lengths, live = _alive(case, t)
    q, k, v = (_heads(t[n], case, live) for n in ("q", "k", "v"))
    out, state = _walk(case, q * case["dim"] ** -0.5, k, v, t["log_decay"], lengths, t.get("state"))
    out = out.transpose(1, 2).contiguous().to(t["q"].dtype)
    return [out, state] if case["state"] else [out]


def _gradient(case, t):
    batch, seq, h, hkv = (case[n] for n in ("batch", "seq", "heads", "kv_heads"))
    lengths, live = _alive(case, t)
    q, k, v, dout = (_heads(t[n], case, live) for n in ("q", "k", "v", "dout"))
    q = q * case["dim"] ** -0.5
    turned = t["state"].transpose(-1, -2) if case["state"] else None
    dq = _walk(case, dout * case["dim"] ** -0.5, v, k, t["log_decay"], lengths, turned)[0]
    # backward in time: every sequence from its last token
    at = torch.arange(seq, device="cuda")
    at = torch.where(at < lengths[:, None], lengths[:, None] - 1 - at, at)[:, None, :, None]
    turn = lambda x: torch.gather(x, 2, at.expand(batch, h, seq, x.shape[-1]))   # noqa: E731
    q, k, v, dout = turn(q), turn(k), turn(v), turn(dout)
    # the last token's state is read by the last token itself and handed on as it is: one step of decay less than a walk's start
    last = t["dstate"] * torch.exp(-t["log_decay"])[:, None, None] if case["state"] else None
    dv, first = _walk(case, k, q, dout, t["log_decay"], lengths, last)
    dk = _walk(case, v, dout, q, t["log_decay"], lengths, last.transpose(-1, -2) if case["state"] else None)[0]
    give = lambda x, heads: x.view(batch, heads, -1, seq, x.shape[-1]).sum(2).transpose(1, 2).contiguous().to(t["q"].dtype)   # noqa: E731
    grads = [give(dq, h), give(turn(dk), hkv), give(turn(dv), hkv)]
    if case["state"]:
        grads.append(first * torch.exp(t["log_decay"])[:, None, None])
    return grads


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    e = SIZES[case["dtype"]]
    batch, seq, h, hkv, dim = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    if case["kind"] == "axes":
        n = batch * seq * (h + hkv)
        return {"bytes": 2 * n * dim * e + 4 * case["axes"] * batch * seq, "flops": 3 * n * case["rotary"]}
    value_dim = case["value_dim"]
    tokens, rows = sum(_lengths(case)), batch * seq
    states = 4 * batch * h * dim * value_dim if case["state"] else 0
    small = 4 * h + (4 * batch if case["lengths"] else 0)
    read = tokens * (h * dim + hkv * (dim + value_dim)) * e
    if case["kind"] == "linear":
        return {"bytes": read + rows * h * value_dim * e + 2 * states + small, "flops": 4 * tokens * h * dim * value_dim}
    write = rows * (h * dim + hkv * (dim + value_dim)) * e
    return {"bytes": read + tokens * h * value_dim * e + write + 3 * states + small, "flops": 10 * tokens * h * dim * value_dim}


# ---------------------------------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    t = _inputs(case, seed)
    f = torch.float64
    if case["kind"] == "axes":
        r, left = case["rotary"], list(_sections(case))
        pairs, used = [], [0] * len(left)
        a = 0
        for i in range(r // 2):
            # the next axis that has a pair left: the same one as long as it has, or the one behind it
            if case["order"] == "cycle" and i:
                a = (a + 1) % len(left)
            while left[a] == 0:
                a = (a + 1) % len(left)
            left[a] -= 1
            exponent = used[a] / _sections(case)[a] if case["rates"] == "own" else 2.0 * i / r
            pairs.append((a, math.exp(-math.log(BASE) * exponent)))
            used[a] += 1
        outs = []
        for name in [n for n in ("q", "k") if n in t]:
            y = t[name].to(f).clone()
            for i, (a, rate) in enumerate(pairs):
                u, v = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
                angle = t["positions"][a].to(f)[..., None] * (-rate if case["inverse"] else rate)
                x1, x2 = y[..., u].clone(), y[..., v].clone()
                y[..., u] = x1 * torch.cos(angle) - x2 * torch.sin(angle)
                y[..., v] = x2 * torch.cos(angle) + x1 * torch.sin(angle)
            outs.append(y)
        return outs
    batch, seq, h, hkv, dim, value_dim = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim", "value_dim"))
    grad = case["kind"] == "grad"
    group, scale = h // hkv, 1.0 / math.sqrt(dim)
    lengths = torch.tensor(_lengths(case), device="cuda")
    wide = lambda x: x.to(f).repeat_interleave(group, 2)   # noqa: E731
    q, k, v = t["q"].to(f) * scale, wide(t["k"]), wide(t["v"])
    decay = torch.exp(t["log_decay"].to(f))[None, :, None, None]
    zero = torch.zeros((batch, h, dim, value_dim), dtype=f, device="cuda")
    s = t["state"].to(f) if case["state"] else zero
    out, dq = torch.zeros((batch, seq, h, value_dim), dtype=f, device="cuda"), torch.zeros_like(q)
    dout = t["dout"].to(f) if grad else None
    for i in range(seq):
        live = (i < lengths)[:, None, None, None]
        s = torch.where(live, decay * s + k[:, i, :, :, None] * v[:, i, :, None, :], s)
        if grad:
            dq[:, i] = torch.where(live[..., 0], (s * dout[:, i, :, None, :]).sum(-1) * scale, 0.0)
        else:
            out[:, i] = torch.where(live[..., 0], (q[:, i, :, :, None] * s).sum(-2), 0.0)
    if not grad:
        return [out, s] if case["state"] else [out]
    ds = t["dstate"].to(f) if case["state"] else zero   # of the state after token i
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for i in reversed(range(seq)):
        live = (i < lengths)[:, None, None, None]
        here = ds + q[:, i, :, :, None] * dout[:, i, :, None, :]
        dk[:, i] = torch.where(live[..., 0], (here * v[:, i, :, None, :]).sum(-1), 0.0)
        dv[:, i] = torch.where(live[..., 0], (here * k[:, i, :, :, None]).sum(-2), 0.0)
        ds = torch.where(live, decay * here, ds)
    share = lambda x: x.view(batch, seq, hkv, group, -1).sum(3)   # noqa: E731
    return [dq, share(dk), share(dv)] + ([ds] if case["state"] else [])
