"""Plain 64-bit forms of the operators on packed documents, and how far a
correct kernel can be from them.

Rounding is half a step: 2^-24 of a value in 32 bits, 2^-8 in bfloat16."""
import numpy as np

E32, E16 = 2.0 ** -24, 2.0 ** -8


def positions(segments):
    """Token by token."""
    out, doc, at = [], None, 0
    for d, kind, frames, rows, cols, step in segments:
        if d != doc:
            doc, at = d, 0
        if kind == 0:
            out += [(at + i,) * 3 for i in range(frames)]
            at += frames
        elif frames * rows * cols > 0:
            out += [(at + step * f, at + r, at + c) for f in range(frames) for r in range(rows)
                    for c in range(cols)]
            at += max(step * (frames - 1) + 1, rows, cols)
    return np.array(out, np.int32).reshape(-1, 3)


def columns(axis, layout):
    """Both columns of each pair."""
    n = len(axis)
    if layout == "half":
        return [(j, j + n) for j in range(n)]
    if layout == "adjacent":
        return [(2 * j, 2 * j + 1) for j in range(n)]
    out, j = [], 0
    while j < n:
        run = 1
        while j + run < n and axis[j + run] == axis[j]:
            run += 1
        out += [(2 * j + i, 2 * j + run + i) for i in range(run)]
        j += run
    return out


def rope(x, pos, freq, axis, layout):
    x = x.astype(np.float64)
    y = x.copy()
    for j, (a, b) in enumerate(columns(axis, layout)):
        t = pos[:, axis[j]].astype(np.float64) * float(freq[j])
        c, s = np.cos(t)[:, None], np.sin(t)[:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def rope_bound(x, y, axis, layout, bf16):
    """cos and sin: the turn's fraction, below 1/2, in 32 bits (2^-25 turns, 2 pi of them an
    angle: 3.2 units of 2^-24) and two steps (4 units) of the functions: 8 units; each product
    and their sum half a step more: 3 units. The output's own rounding on top."""
    pair = np.abs(x.astype(np.float64))
    total = pair.copy()
    for a, b in columns(axis, layout):
        total[..., a] = total[..., b] = pair[..., a] + pair[..., b]
    return 11 * E32 * total + (E16 if bf16 else E32) * np.abs(y)


def visible(ql, kl, causal, window, prefix):
    p = np.arange(ql)[:, None] + (kl - ql)
    j = np.arange(kl)[None]
    seen = np.ones((ql, kl), bool)
    if causal:
        seen &= j <= p
    if window is not None:
        seen &= np.abs(p - j) <= window
    return seen | (j < prefix), np.abs(p - j)


def attention(q, k, v, q_off, k_off, *, causal=False, window=None, prefix=None, scale=1.0,
              cap=0.0, slopes=None, bf16=False):
    """out, lse and their bounds, [query rows, heads, ...]; rows outside every document NaN.

    A score's error: products summed in 32 bits, (hd + 8) half steps of sum |q| |k| (a step per
    addition; 4 for operands held in three parts; 2 for the scale; 2 spare); the cap's tanh, 8
    half steps of the cap; the bias, 3 half steps of its size; 4 half steps of the score for base
    2 and the maximum. A weight then errs by twice the largest score error (its own and the
    sum's), by 8 half steps in the exponential and the sum's own (kl / 64 + 16) half steps; the
    weighted sum adds as many. Weights of bfloat16 products are rounded to it."""
    rows, nh, hd = q.shape
    nkv = k.shape[1]
    out = np.full(q.shape, np.nan)
    lse = np.full((rows, nh), np.nan)
    ob, lb = np.full(q.shape, np.nan), np.full((rows, nh), np.nan)
    for d in range(len(q_off) - 1):
        a, b, c, e = q_off[d], q_off[d + 1], k_off[d], k_off[d + 1]
        if b == a:
            continue
        seen, gap = visible(b - a, e - c, causal, window, prefix[d] if prefix is not None else 0)
        for h in range(nh):
            qq = q[a:b, h].astype(np.float64)
            kk = np.where(seen.any(0)[:, None], k[c:e, h // (nh // nkv)].astype(np.float64), 0)
            vv = np.where(seen.any(0)[:, None], v[c:e, h // (nh // nkv)].astype(np.float64), 0)
            s = qq @ kk.T * scale
            err = (hd + 8) * E32 * (np.abs(qq) @ np.abs(kk).T) * abs(scale) + 4 * E32 * np.abs(s)
            if cap:
                s = cap * np.tanh(s / cap)
                err = err + 8 * E32 * cap
            if slopes is not None:
                bias = float(slopes[h]) * gap
                s = s - bias
                err = err + 3 * E32 * np.abs(bias)
            s = np.where(seen, s, -np.inf)
            top = s.max(1, initial=-np.inf)
            some = top > -np.inf
            w = np.exp(s - np.where(some, top, 0)[:, None])
            total = w.sum(1)
            w = w / np.where(some, total, 1)[:, None]
            # scores far below the maximum have no weight: their error does not count
            heavy = np.where(seen & (w > 2.0 ** -40), err, 0).max(1, initial=0)
            length = (e - c) / 64 + 16
            rel = np.expm1(2 * heavy) + (8 + 2 * length) * E32 + 2.0 ** -38 * (e - c)
            mass = w @ np.abs(vv)
            out[a:b, h] = w @ vv
            ob[a:b, h] = rel[:, None] * mass + E32 * np.abs(out[a:b, h])
            if bf16:
                ob[a:b, h] += E16 * (mass + np.abs(out[a:b, h])) * (1 + E16)
            with np.errstate(divide="ignore"):
                lse[a:b, h] = np.where(some, top + np.log(total), -np.inf)
            lb[a:b, h] = rel + 4 * E32 * np.abs(np.where(some, lse[a:b, h], 0)) + 4 * E32
    return out, lse, ob, lb
