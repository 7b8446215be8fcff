"""The linear layers of a feed-forward block in 64 bits, and how far a result in fewer may be from them."""

import math

import numpy as np
import torch

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # half a step, relative: torch.finfo(t).eps / 2 (bf16: eps is 2^-7)
TINY = {torch.float32: 1e-37, torch.float16: 2.0**-24, torch.bfloat16: 1e-37}  # half a step of the subnormals, with room

ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


def act(g, name):
    s = torch.sigmoid(g)
    if name == "silu":
        return g * s
    if name == "gelu":
        return 0.5 * g * torch.erfc(-g / math.sqrt(2))
    if name == "gelu_tanh":
        return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g**3))  # (1 + tanh z) / 2, which cancels below -18
    if name == "relu":
        return torch.where(g <= 0, torch.zeros_like(g), g)
    return s


def slope(g, name):
    """d act / dg by its formula (not by autograd: the tests hold it against differences, too)."""
    s = torch.sigmoid(g)
    if name == "silu":
        return s * (1 + g * (1 - s))
    if name == "gelu":
        return 0.5 * torch.erfc(-g / math.sqrt(2)) + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        z = 2 * c * (g + 0.044715 * g**3)
        return torch.sigmoid(z) + g * torch.sigmoid(z) * torch.sigmoid(-z) * 2 * c * (1 + 3 * 0.044715 * g * g)
    if name == "relu":
        return torch.where(g <= 0, torch.zeros_like(g), torch.ones_like(g))
    return s * (1 - s)


def sum_error(k, dtype):
    """Relative to the sum of magnitudes: 16-bit products go into the tensor cores' fp32 sums 16 at a time, each addition off by at most
    a whole step of fp32 (they truncate), with as much again inside a group; fp32 ones one by one, half a step each, plus what
    three bf16 planes leave out (2^-24 or so)."""
    return (k / 16 + 2) * 2.0**-22 if dtype != torch.float32 else (k / 2 + 8) * 2.0**-23


def act_error(g, name, dtype):
    """Of the activation, relative to it: 2^-18 (fp32: 2^-21) for the quotient and the functions, and what its exponential e^-y adds. y
    is off by 6 half steps of fp32 where it is computed (gelu_tanh: four products, a sum, a rounded constant), which changes e^-y by
    the factor 1 + 6 |y| 2^-24; the fast exponential of 16-bit results is good to 2 + 1.173 |y| units in the last place, 2^-23 each."""
    y = {"gelu_tanh": 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g**3)}.get(name, g).abs().clamp(max=104)  # beyond, e^-y is 0 or infinite in fp32
    err = 6 * 2.0**-24 * y if name == "gelu_tanh" else torch.zeros_like(y)
    return 2.0**-21 + err if dtype == torch.float32 else 2.0**-18 + err + 1.2 * 2.0**-23 * y


def gated(x, w, name, dtype):
    """(h, tolerance of h, projections, their tolerance) for 2-D x, w of any float type, in 64 bits."""
    x, w = x.double(), w.double()
    F = w.shape[0] // 2
    p, mag = x @ w.t(), x.abs() @ w.abs().t()
    err = sum_error(x.shape[1], dtype) * mag
    g, u = p[:, :F], p[:, F:]
    a = act(g, name)
    h = a * u
    fn = act_error(g, name, dtype)  # and |act'| <= 1.13
    tol = U[dtype] * h.abs() + (1.13 * err[:, :F] + fn * a.abs()) * (u.abs() + err[:, F:]) + a.abs() * err[:, F:]
    return h, 1.001 * tol + TINY[dtype], p, 1.001 * err + 1e-37  # (the projections are fp32 sums)


def gated_grads(dh, x, w, p, name, dtype):
    """(dx, tolerance, dw, tolerance) for the projections `p` that the backward pass is given."""
    dh, x, w, p = dh.double(), x.double(), w.double(), p.double()
    F = w.shape[0] // 2
    g, u = p[:, :F], p[:, F:]
    a, s = act(g, name), slope(g, name)
    dp = torch.cat([dh * u * s, dh * a], 1)
    fn = 2.0**-18 if dtype != torch.float32 else 2.0**-20
    # dP is rounded to the operands' type; a slope is a sum of terms up to 1 + |g| (beyond 30 it is 0 or 1)
    ddp = U[dtype] * dp.abs() + TINY[dtype] + torch.cat([fn * dh.abs() * u.abs() * (1 + g.abs().clamp(max=30)), act_error(g, name, dtype) * dh.abs() * a.abs()], 1)
    dx, dw = dp @ w, dp.t() @ x
    tx = U[dtype] * dx.abs() + ddp @ w.abs() + sum_error(2 * F, dtype) * (dp.abs() @ w.abs())
    tw = U[dtype] * dw.abs() + ddp.t() @ x.abs() + sum_error(x.shape[0], dtype) * (dp.abs().t() @ x.abs())
    return dx, 1.001 * tx + TINY[dtype], dw, 1.001 * tw + TINY[dtype]


def words(n, seed, offset, subsequence=0):
    """n 32-bit words of Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011) on the host."""
    draws, m = (n + 3) // 4, np.uint64(0xFFFFFFFF)
    seed, offset, subsequence = seed % 2**64, offset % 2**64, subsequence % 2**64
    with np.errstate(over="ignore"):
        count = np.arange(draws, dtype=np.uint64) + np.uint64(offset)
    a, b = count & m, count >> np.uint64(32)
    c, d = np.full(draws, subsequence & 0xFFFFFFFF, np.uint64), np.full(draws, subsequence >> 32, np.uint64)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p, q = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (q >> np.uint64(32)) ^ b ^ np.uint64(k0), q & m, (p >> np.uint64(32)) ^ d ^ np.uint64(k1), p & m
        k0, k1 = (k0 + 0x9E3779B9) % 2**32, (k1 + 0xBB67AE85) % 2**32
    return np.stack([a, b, c, d], 1).reshape(-1)[:n]


def kept(shape, p, seed, offset, subsequence=0):
    n = int(np.prod(shape))
    return torch.from_numpy(words(n, seed, offset, subsequence) >= np.uint64(round(p * 2**32))).view(*shape)


def assert_within(got, ref, tol, what=""):
    ref, tol = ref.to(got.device), tol.to(got.device)
    off = (got.double() - ref).abs()
    bad = ~((off <= tol) | (got.double() == ref))
    if bool(bad.any()):
        i = int((off / tol).nan_to_num(nan=math.inf).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst {got.flatten()[i].item()} for {ref.flatten()[i].item()}, tolerance {tol.flatten()[i].item()}")
