"""The cache in 8 bits in plain float64: rows to codes and back, and attention over the rows that the codes stand for."""
import math

import numpy as np
import torch

PAGE = 64
LIMIT = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
SMALLEST = 2.0 ** -96


def to_grid(y, dtype):
    """y (float64) rounded half to even to the numbers of the codes' type."""
    if dtype == torch.int8:
        return np.rint(y)
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -40))), -6)
    step = np.exp2(e - 3)
    return np.rint(y / step) * step


def store_rows(x, dtype):
    """Codes (as numbers) and scales of rows x [..., entries]."""
    x = np.asarray(x, dtype=np.float64)
    top = np.abs(x).max(-1, keepdims=True)
    bad = ~np.isfinite(top)
    empty = top < SMALLEST
    with np.errstate(invalid="ignore", divide="ignore"):
        y = np.where(empty | bad, 0.0, x / np.where(empty | bad, 1.0, top) * LIMIT[dtype])
    scale = np.where(bad, np.nan, np.where(empty, 0.0, top / LIMIT[dtype]))
    return to_grid(np.where(np.isfinite(y), y, 0.0), dtype), scale[..., 0]


def random_store(gen, pages, heads, size, dtype, spread=0.5, device="cuda"):
    """A store of 8-bit pages on the device: (codes, scales), rows of unequal sizes."""
    x = torch.randn(pages, heads, PAGE, size, generator=gen, device=device)
    x = x * torch.exp(spread * torch.randn(heads, 1, size, generator=gen, device=device))
    x = x * torch.exp(0.5 * torch.randn(pages, heads, PAGE, 1, generator=gen, device=device))
    top = x.abs().amax(-1, keepdim=True)
    y = x * (LIMIT[dtype] / top)
    codes = y.to(dtype) if dtype == torch.float8_e4m3fn else y.round().to(dtype)
    return codes.contiguous(), (top[..., 0] / LIMIT[dtype]).contiguous()


def numbers(codes):
    """Codes as float64 numbers on the host."""
    return codes.float().double().cpu().numpy()


def attend(q, k, v, position, *, scale, group, maps=1, window=None, chunk=None, keep_first=0, slopes=None, sinks=None, softcap=None):
    """One token's attention in float64: q [heads, dim], k [kv_heads, keys, dim], v [v_heads, keys, vdim] (the sequence's rows from key 0
    on).  Returns out [heads, vdim] (each map's own), the same with |v|, the largest weight times value of every head, the largest
    sum |q k| scale, and the largest |q| times the largest sum |k| times scale: what bounds on the error are made of."""
    keys = np.arange(position + 1)
    lo = max(0, position - window + 1) if window else 0
    if chunk:
        lo = max(lo, position // chunk * chunk)
    seen = keys[(keys >= lo) | (keys < keep_first)]
    heads, vdim = q.shape[0], v.shape[-1]
    out, size, top, reach, span = np.zeros((heads, vdim)), np.zeros((heads, vdim)), np.zeros(heads), np.zeros(heads), np.zeros(heads)
    for h in range(heads):
        kv = h // group
        s = k[kv][seen] @ q[h] * scale
        reach[h] = (np.abs(k[kv][seen]) @ np.abs(q[h])).max() * scale
        span[h] = np.abs(q[h]).max() * np.abs(k[kv][seen]).sum(-1).max() * scale
        if softcap:
            s = softcap * np.tanh(s / softcap)
        if slopes is not None:
            s = s - slopes[h] * (position - seen)
        m = s.max() if sinks is None else max(s.max(), sinks[h])
        p = np.exp(s - m)
        total = p.sum() + (math.exp(sinks[h] - m) if sinks is not None else 0.0)
        rows = v[kv // maps][seen]
        out[h], size[h] = p @ rows / total, p @ np.abs(rows) / total
        top[h] = (p * np.abs(rows).max(-1)).max() / total
    return out, size, top, reach, span


def difference(out, lam, heads, kv_heads, eps, factor):
    """Two maps' outputs [query heads as (value head, map, group), vdim] to normed differences [heads, vdim]."""
    o = out.reshape(kv_heads, 2, heads // kv_heads, -1)
    o = (o[:, 0] - lam * o[:, 1]).reshape(heads, -1)
    return o / np.sqrt((o * o).mean(-1, keepdims=True) + eps) * factor


def output_bound(want, size, top, reach, span, position, *, dim, group, codes, maps=1, softcap=None, slopes=None, lam=None, eps=None, factor=None,
                 rounding=2.0 ** -11):
    """What one token's output (bfloat16) may be off by, and the value itself with two maps' difference taken; ``rounding``: of a weight.

    Scores: exact products added in float32 (or integers), up to 2^-23 of the terms' size a step, and a few roundings of the score itself, of a
    slope's product and of a cap; twice that is the relative error of a weight over the sum.  With ``codes`` (the type, for single
    tokens) the queries are rounded: int8 to 16 bits, half a unit of 1/32512 of the head's largest entry; float8_e4m3fn to float16, half of
    whose smallest step is 2^-25 in units in which the largest entry is 2^14 or more.
    Weights: their rounding, the hardware's exponential, sums of position + 1 terms in float32; a weight below 2^-22 of the largest has an
    absolute error instead.  Then the output's own rounding."""
    rounded = {None: 0.0, torch.int8: 0.5 / 32512, torch.float8_e4m3fn: 2.0 ** -39}[codes]
    score = 2.0 ** -23 * (dim + 16) * reach + rounded * 1.001 * span + (2.0 ** -20 * softcap if softcap else 0.0)
    if slopes is not None:
        score = score + 2.0 ** -22 * slopes * position
    weight = rounding + 2.0 ** -16 + (position + 1) * 2.0 ** -26 + 4 * score[:, None]
    bound = weight * size + (position + 1) * 2.0 ** -31 * top[:, None]
    if maps == 2:
        heads = want.shape[0] // 2
        kv_heads = heads // group
        raw = want.reshape(kv_heads, 2, group, -1)
        raw = (raw[:, 0] - lam * raw[:, 1]).reshape(heads, -1)
        b = bound.reshape(kv_heads, 2, group, -1)
        b = (b[:, 0] + abs(lam) * b[:, 1]).reshape(heads, -1)
        want = difference(want, lam, heads, kv_heads, eps, factor)
        # the norm's factor is off by at most the largest relative error of the row
        rms = np.sqrt((raw * raw).mean(-1, keepdims=True) + eps)
        shift = np.sqrt((b * b).mean(-1, keepdims=True)) / rms
        bound = factor * b / rms * (1 + 2 * shift) + 2 * shift * np.abs(want) + 2.0 ** -18 * np.abs(want)
    return want, bound + 2.0 ** -8 * (np.abs(want) + bound) + 1e-37
