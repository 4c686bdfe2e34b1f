"""Linear attention with a decay for each head, its gradient and rotary positions of several axes in float64 on the host, and
bounds on what roundings can change. `u` is half a step of a type relative to the value: torch.finfo(t).eps / 2."""
import math

import torch

from attention_reference import back, half_step, heads_of

F = torch.float64
CHUNK = 64


def powers(g, n):
    """exp(g n) for every head, [heads, *n.shape]: 1 where n is 0, also for g = -inf; 0 where n is negative."""
    g = g.to(F).view([-1] + [1] * n.dim())
    n = n.to(F)[None]
    return torch.where(n < 0, torch.zeros((), dtype=F), torch.where(n == 0, torch.ones((), dtype=F), torch.exp(torch.where(n == 0, torch.zeros((), dtype=F), g * n))))


def recurrence(a, b, c, g, scale, length, start):
    """The definition, token by token, for one sequence: a, b, c [heads, tokens, channels]. (out, last state)."""
    s = start.clone()
    lam = torch.exp(g.to(F))[:, None, None]
    out = torch.zeros((a.shape[0], a.shape[1], c.shape[2]), dtype=F)
    for t in range(length):
        s = torch.where(lam == 0, torch.zeros((), dtype=F), lam * s) + b[:, t, :, None] * c[:, t, None, :]
        out[:, t] = scale * (a[:, t, :, None] * s).sum(1)
    return out, s


def walk(a, b, c, g, scale, length, start, backward=False):
    """(out, state, rough, state_rough) of one sequence, in chunks; a backward walk starts at the last token, with a state that
    is that token's already, and leaves the one in front of the first. `rough`: [2, ...] sums of the sizes of what is rounded
    where it is contracted (masked products times |c|, |a| times the state in front of the chunk), and the same with the sizes of
    the terms of the masked products; `state_rough`: of the terms of a state."""
    heads, tokens = a.shape[:2]
    order = torch.arange(length - 1, -1, -1) if backward else torch.arange(length)
    a, b, c = a[:, order], b[:, order], c[:, order]
    z = 1 if backward else 0
    grow, show = (scale, 1.0) if backward else (1.0, scale)
    out, rough = torch.zeros((heads, tokens, c.shape[2]), dtype=F), torch.zeros((2, heads, tokens, c.shape[2]), dtype=F)
    s, size = start.clone(), start.abs()
    for r0 in range(0, length, CHUNK):
        x, y, w = (t[:, r0:r0 + CHUNK] for t in (a, b, c))
        n = x.shape[1]
        i = torch.arange(n)
        p = (x @ y.transpose(1, 2)) * powers(g, i[:, None] - i) * scale
        seen = powers(g, i + 1 - z)[..., None] * show
        out[:, order[r0:r0 + n]] = p @ w + seen * (x @ s)
        terms = (x.abs() @ y.abs().transpose(1, 2)) * powers(g, i[:, None] - i) * scale
        for k, sizes in enumerate((p.abs(), terms)):
            rough[k, :, order[r0:r0 + n]] = sizes @ w.abs() + seen * (x.abs() @ size)
        fade = powers(g, torch.tensor([n]))[..., None]
        left = powers(g, n - 1 - i + z)[..., None] * grow
        s = torch.where(fade == 0, torch.zeros((), dtype=F), fade * s) + (y * left).transpose(1, 2) @ w
        size = torch.where(fade == 0, torch.zeros((), dtype=F), fade * size) + (y * left).abs().transpose(1, 2) @ w.abs()
    return out, s, rough, size


def lengths_of(lengths, batch, seq):
    return [seq] * batch if lengths is None else [min(max(int(n), 0), seq) for n in lengths]


def start_of(state, slots, b, shape):
    if state is None:
        return torch.zeros(shape, dtype=F)
    if slots is None:
        return state[b].to(F)
    n = int(slots[b])
    return state[n].to(F) if 0 <= n < state.shape[0] else torch.zeros(shape, dtype=F)


def wide(x, heads):
    return x.repeat_interleave(heads // x.shape[1], 1)


def forward(q, k, v, log_decay, state=None, slots=None, lengths=None, layout="BSND", scale=None):
    """dict of out, rough (layout of the operator), last and last_rough ([batch, heads, channels, channels])."""
    q, k, v = (heads_of(x, layout) for x in (q, k, v))
    batch, h, seq, dim = q.shape
    scale = 1 / math.sqrt(dim) if scale is None else scale
    k, v = wide(k, h), wide(v, h)
    parts = [walk(q[b], k[b], v[b], log_decay, scale, n, start_of(state, slots, b, (h, dim, v.shape[3])))
             for b, n in enumerate(lengths_of(lengths, batch, seq))]
    out, last, rough, size = (torch.stack(x) for x in zip(*parts))
    return {"out": back(out, layout), "rough": [back(rough[:, k], layout) for k in range(2)], "last": last, "last_rough": size, "channels": dim, "seq": seq}


def gradient(dout, q, k, v, log_decay, state=None, dstate=None, lengths=None, layout="BSND", scale=None):
    """dict of dq, dk, dv, dstate: (exact, rough) each."""
    dout, q, k, v = (heads_of(x, layout) for x in (dout, q, k, v))
    batch, h, seq, dim = q.shape
    hkv, e = v.shape[1], v.shape[3]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    k, v = wide(k, h), wide(v, h)
    got = {n: ([], []) for n in ("dq", "dk", "dv", "dstate")}

    def keep(name, exact, rough):
        got[name][0].append(exact)
        got[name][1].append(rough)
    t = lambda x: x.transpose(1, 2)   # noqa: E731
    for b, n in enumerate(lengths_of(lengths, batch, seq)):
        first, last = start_of(state, None, b, (h, dim, e)), start_of(dstate, None, b, (h, dim, e))
        dq = walk(dout[b], v[b], k[b], log_decay, scale, n, t(first))
        dk = walk(v[b], dout[b], q[b], log_decay, scale, n, t(last), backward=True)
        dv = walk(k[b], q[b], dout[b], log_decay, scale, n, last, backward=True)
        keep("dq", dq[0], dq[2])
        for name, x in (("dk", dk), ("dv", dv)):
            keep(name, x[0].view(hkv, h // hkv, seq, -1).sum(1), x[2].view(2, hkv, h // hkv, seq, -1).sum(2))
        keep("dstate", dv[1], dv[3])
    stacked = {n: tuple(torch.stack(x) for x in pair) for n, pair in got.items()}
    return {n: (x, y) if n == "dstate" else (back(x, layout), [back(y[:, k], layout) for k in range(2)]) for n, (x, y) in stacked.items()}


def bound(exact, rough, dtype, channels, seq):
    """|computed - exact| of a result in `dtype`. bfloat16: masked products and the state are rounded where they are contracted
    again (u of each term, on a state off by 2^-16 of its terms). float16: every operand goes as two bfloat16 parts, which
    leave 2^-16 of it (of the operands given: nothing, 11 digits fit 16), and the product of two rests is left out, at most 2^-8
    2^-8 of a term: 2^-16 of the terms of the masked products (`rough[1]`), and of what they and the state are contracted with.
    float32: sums of at most `channels` + 64 terms a chunk (2^-24 a step of each term, twice), the weights, whose exponents are
    off by 2^-23 of themselves where a weight is not below 2^-30 (2^-18), the state once a chunk. The result rounded."""
    u = half_step(dtype)
    operands = u + 2.0 ** -15 if dtype == "bfloat16" else 4 * 2.0 ** -16
    noise = 2.0 ** -23 * (channels + 64 + seq / 64) + 2.0 ** -18 + (2.0 ** -16 if dtype == "float16" else 0)
    return 1.02 * (operands * rough[0] + noise * rough[1] + u * exact.abs()) + (2.0 ** -25 if dtype == "float16" else 0) + 1e-30


def state_bound(rough, channels, seq, rounded=True):
    """|computed - exact| of a state: its terms go as two bfloat16 parts (2^-16; float16: of both operands, 3 2^-16), or as they
    are (token after token); float32 in weights and sums."""
    return ((3 * 2.0 ** -16 if rounded else 0) + 2.0 ** -23 * (64 + seq / 64) + 2.0 ** -20) * rough + 1e-30


def rotary_axes(x, positions, sections, order, rates, base, rotary_dims=0, interleaved=False, inverse=False, layout="BSND", magnitude=1.0):
    """`positions` [axes, batch or 1, sequence]."""
    x = x.to(F) if layout == "BSND" else x.to(F).transpose(1, 2)
    r = rotary_dims or x.shape[3]
    axes = [a for a, n in enumerate(sections) for _ in range(n)]
    if order == "cycle":
        axes = [a for j in range(max(sections)) for a, n in enumerate(sections) if j < n]
    y = x.clone()
    used = [0] * len(sections)
    for i, a in enumerate(axes):
        rate = base ** (-used[a] / sections[a]) if rates == "own" else base ** (-2.0 * i / r)
        used[a] += 1
        angle = positions[a].to(F)[..., None] * rate
        c, s = torch.cos(angle) * magnitude, torch.sin(angle) * (-magnitude if inverse else magnitude)
        u, v = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        y[..., u], y[..., v] = x[..., u] * c - x[..., v] * s, x[..., v] * c + x[..., u] * s
    return y if layout == "BSND" else y.transpose(1, 2)
