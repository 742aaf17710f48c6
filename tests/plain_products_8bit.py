"""Products in 8-bit integers in 64 bits on the host or the device, with bounds on how far a kernel in 32 bits may be off.

A number in float32 is off by at most 2^-24 of itself after each rounding (U below), one rounded to bfloat16 by 2^-8."""
import math

import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}
SMALLEST = 2.0 ** -96


def up(n, step):
    return -(-n // step) * step


def codes_of(x):
    """Codes and scales of rows of any finite numbers."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    held = top >= SMALLEST
    safe = torch.where(held, top, 1.0)
    return torch.where(held, torch.round(x * 127.0 / safe), 0.0), torch.where(held, top / 127.0, 0.0)


def laid_out(codes, scales):
    """Codes [experts, parts, features, inner] and scales in the kernels' layout."""
    e, p, f, k = codes.shape
    big = torch.zeros((e, p, up(f, 16), up(k, 128)), dtype=torch.int8, device=codes.device)
    big[:, :, :f, :k] = codes.to(torch.int8)
    s = torch.zeros((e, p, up(f, 16)), dtype=torch.float32, device=codes.device)
    s[:, :, :f] = scales.float()
    return big, s


def random_weight(gen, experts, parts, features, inner, device):
    w = torch.randn((experts, parts, features, inner), generator=gen, device=device) / math.sqrt(inner)
    codes, scales = codes_of(w)
    return codes, scales.squeeze(-1).float(), *laid_out(codes, scales.squeeze(-1))


def product(x, codes, scales):
    """The exact result and a bound of a float32 kernel's error: the token's scale, the sum as float32 and two products are a rounding each."""
    q, step = codes_of(x)
    exact = (q @ codes.double().T) * step * scales.double()
    return exact, 4.01 * U * exact.abs()


def gate(g, u, activation, limit):
    """The unit's value and a bound of its error in float32 for g and u that are off by 4.01 U each: an error of g moves silu(g) by at most
    (1 + |g|) as much of itself, and exp, tanh, the division and the products add a handful of roundings (16 leaves room for errors of
    exp and tanh of two units in the last place); 1 + tanh loses what the sum cancels, so gelu is bounded by |g| instead."""
    if limit > 0:
        gc, uc = g.clamp(max=limit), u.clamp(-limit, limit)
        unit = gc * torch.sigmoid(1.702 * gc)
        return unit * (uc + 1), 16 * U * (1 + 1.702 * gc.abs()) * unit.abs() * (uc.abs() + 1)
    if activation == "gelu_tanh":
        value = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
        slope = 1 + math.sqrt(2 / math.pi) * (g.abs() + 3 * 0.044715 * g.abs() ** 3).clamp(max=20)
        return value * u, 16 * U * slope * g.abs() * u.abs()
    value = g * torch.sigmoid(g)
    return value * u, 16 * U * (1 + g.abs()) * (value * u).abs()


def block(x, in_codes, in_scales, down_codes, down_scales, activation="silu", limit=0.0):
    """A gated block and a bound of its error: beside the second product's roundings, an entry of h that is nearer to the middle of two codes
    than its own error (and the scale's) may go to either of them."""
    g, _ = product(x, in_codes[0], in_scales[0])
    u, _ = product(x, in_codes[1], in_scales[1])
    h, off = gate(g, u, activation, limit)
    top = h.abs().amax(-1, keepdim=True)
    q, step = codes_of(h)
    v = h * 127 / top.clamp_min(1e-300)
    # the largest entry's own error moves every code of its row
    largest = off.gather(-1, h.abs().argmax(-1, keepdim=True)) / top.clamp_min(1e-300)
    near = ((v - v.floor() - 0.5).abs() <= 127 * off / top.clamp_min(1e-300) + v.abs() * (largest + 4 * U)).double()
    w = down_codes.double()
    exact = (q @ w.T) * step * down_scales.double()
    flipped = (near @ w.abs().T) * step * down_scales.double().abs()
    return exact, flipped + (4.01 * U + largest) * (exact.abs() + flipped)


def agree(got, exact, bound, what=""):
    """got within the bound of its type: the bound and the last rounding's."""
    bound = bound + HALF_STEP[got.dtype] * (exact.abs() + bound) + 1e-37
    off = (got.double() - exact).abs()
    worst = (off / bound).nan_to_num(nan=float("inf")).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times its bound"
