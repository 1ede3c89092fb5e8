"""Plain 64-bit forms of the operators over grouped rows (CPU tensors), and bounds on a kernel's error.

Bounds: a sum of n terms held in 32 bits is off by at most n * 2^-23 of the sum of the terms' magnitudes (a
step of 2^-23 for each addition, so that truncated additions count too), and an output of 16 bits by half a
step more (2^-8 of its value in bf16, 2^-11 in fp16, and 2^-25 where fp16 has no more digits)."""
from __future__ import annotations

import torch

STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25, torch.float32: 2.0**-126}


def d(t):
    return None if t is None else t.detach().cpu().double()


def close(got, want, magnitude, terms, dtype, what=""):
    """Every |got - want| within terms * 2^-23 * magnitude and the output's own rounding."""
    assert got.dtype == dtype, what
    sums = terms * 2.0**-23 * magnitude
    bound = sums + STEP[dtype] * (want.abs() + sums) + TINY[dtype]
    off = (got.cpu().double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound)[bad].max()):.3g} times the bound"


def sort_pairs(ids, groups):
    """(offsets, order, pos) of a stable sort of the pairs by group, one pair at a time."""
    flat = ids.reshape(-1).tolist()
    rows = [[i for i, g in enumerate(flat) if g == want] for want in range(groups)] if groups <= 64 else None
    if rows is None:
        rows = [[] for _ in range(groups)]
        for i, g in enumerate(flat):
            if 0 <= g < groups:
                rows[g].append(i)
    order = [i for r in rows for i in r]
    offsets = [0]
    for r in rows:
        offsets.append(offsets[-1] + len(r))
    pos = [-1] * len(flat)
    for p, i in enumerate(order):
        pos[i] = p
    order += [-1] * (len(flat) - len(order))
    return (torch.tensor(offsets, dtype=torch.int32), torch.tensor(order, dtype=torch.int32),
            torch.tensor(pos, dtype=torch.int32).reshape(ids.shape))


def combine(pos, ys, w):
    """y, and the sum of magnitudes."""
    tokens, topk = pos.shape
    y = torch.zeros((tokens, ys.shape[1]), dtype=torch.float64)
    mag = torch.zeros_like(y)
    for t in range(tokens):
        for j in range(topk):
            p = int(pos[t, j])
            if p >= 0:
                f = 1.0 if w is None else float(w[t, j])
                y[t] += f * d(ys[p])
                mag[t] += abs(f) * d(ys[p]).abs()
    return y, mag


def grouped(offsets, x, w):
    at = offsets.tolist()
    y = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64)
    mag = torch.zeros_like(y)
    for g, (i, j) in enumerate(zip(at, at[1:])):
        y[i:j] = d(x[i:j]) @ d(w[g]).T
        mag[i:j] = d(x[i:j]).abs() @ d(w[g]).abs().T
    return y, mag


def grouped_dx(offsets, dy, w):
    return grouped(offsets, dy, w.transpose(1, 2))


def grouped_dw(offsets, dy, x):
    at = offsets.tolist()
    dw = torch.zeros((len(at) - 1, dy.shape[1], x.shape[1]), dtype=torch.float64)
    mag = torch.zeros_like(dw)
    for g, (i, j) in enumerate(zip(at, at[1:])):
        dw[g] = d(dy[i:j]).T @ d(x[i:j])
        mag[g] = d(dy[i:j]).abs().T @ d(x[i:j]).abs()
    return dw, mag


def lora(offsets, adapter, x, a, b, base, scale):
    """out (rows of no request: zero), the mask of rows that belong to one, and a bound on the error before the last rounding.

    The intermediate u = a x may be kept as two 16-bit terms: half a step of a half step, 2^-16 in bf16, 2^-22 in fp16
    (and 2^-25 at its smallest numbers), and comes in up to 8 parts of the sum over K, each kept so."""
    rows, rank, K = x.shape[0], a.shape[1], x.shape[1]
    out = torch.zeros((rows, b.shape[1]), dtype=torch.float64)
    err = torch.zeros_like(out)
    real = torch.zeros(rows, dtype=torch.bool)
    at = list(range(rows + 1)) if offsets is None else offsets.tolist()
    two = STEP[x.dtype] ** 2
    tiny = TINY[x.dtype]
    for r, (i, j) in enumerate(zip(at, at[1:])):
        real[i:j] = True
        if base is not None:
            out[i:j] = d(base[i:j])
        e = int(adapter[r])
        if e < 0 or e >= a.shape[0] or i == j:
            continue
        s = 1.0 if scale is None else float(scale[e])
        u, um = d(x[i:j]) @ d(a[e]).T, d(x[i:j]).abs() @ d(a[e]).abs().T
        delta, bm = s * (u @ d(b[e]).T), d(b[e]).abs().T
        err[i:j] = abs(s) * ((um * (two + K * 2.0**-23) + 8 * tiny) @ bm + 16 * rank * 2.0**-23 * (um @ bm)) + 2.0**-22 * (out[i:j].abs() + delta.abs())
        out[i:j] += delta
    return out, real, err
