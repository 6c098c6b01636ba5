"""Plain 64-bit definitions of the operators of residual networks, and how far a kernel that sums in fp32 and rounds once may be from them."""
import math

import numpy as np
import torch

U32 = 2.0 ** -24                     # a rounding to fp32 is off by at most this, relative to the value


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the spacing of the type's subnormal numbers: what a rounding may be off by near 0."""
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2


def act64(name, v):
    return {"identity": lambda: v, "relu": lambda: torch.clamp(v, min=0), "tanh": lambda: torch.tanh(v), "sigmoid": lambda: torch.sigmoid(v),
            "fast_tanh": lambda: (lambda c: c * (27 + c * c) / (27 + 9 * c * c))(torch.clamp(v, -3, 3)),
            "gelu": lambda: v * 0.5 * torch.erfc(-v / math.sqrt(2)), "silu": lambda: v * torch.sigmoid(v)}[name]()


def slope64(name, v):
    if name == "fast_tanh":          # the framework's slope of this activation: 1 - a^2
        return 1 - act64(name, v) ** 2
    v = v.detach().clone().requires_grad_(True)
    act64(name, v).sum().backward()
    g = v.grad
    return torch.where(v == 0, torch.zeros_like(g), g).detach() if name == "relu" else g.detach()


def product_error(a, b):
    """Bound on the error of a b^T summed in fp32 in any order, by an adder that truncates: one step of 2^-23 of the sum of magnitudes per addition."""
    return (a.shape[1] + 2) * 2 * U32 * (a.abs() @ b.abs().t())


def activation_error(v):
    """fp32 evaluation of an activation or its slope: sixteen roundings of numbers no larger than 1 + |v| (v^2 where the slope multiplies by v)."""
    return 16 * U32 * (1 + v.abs())


def norm64(kind, v, weight, bias, epsilon):
    if kind == "none":
        return v
    c = v - v.mean(1, keepdim=True) if kind == "layer" else v
    hat = c / torch.sqrt((c * c).mean(1, keepdim=True) + epsilon)
    hat = hat if weight is None else hat * weight
    return hat if bias is None else hat + bias


def norm_residual64(branch, residual, post, post_weight, post_bias, gate, gate_rows, scale, pre, pre_weight, pre_bias, epsilon):
    out = torch.zeros_like(branch if residual is None else residual) if residual is None else residual
    if branch is not None:
        u = norm64(post, branch, post_weight, post_bias, epsilon)
        if gate is not None:
            u = u * gate[torch.arange(u.shape[0], device=u.device) // gate_rows]
        out = out + scale * u
    return out, norm64(pre, out, pre_weight, pre_bias, epsilon) if pre != "none" else None


def philox_halves(n, seed, stream_id, call):
    """The 16 random bits of elements 0 .. n-1."""
    m = 0xFFFFFFFF
    out = np.zeros(((n + 7) // 8, 4), np.uint64)
    for b in range(out.shape[0]):
        c = [b & m, call & m, (call >> 32) & m, (0x80000000 + ((b >> 32) << 16) + stream_id) & m]
        k0, k1 = seed & m, (seed >> 32) & m
        for _ in range(10):
            p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(p1 >> 32) ^ c[1] ^ k0, p1 & m, (p0 >> 32) ^ c[3] ^ k1, p0 & m]
            k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
        out[b] = c
    return out.astype("<u4").reshape(-1).view("<u2")[:n].astype(np.int64)


def dropout64(x, p, seed, stream_id, call, residual=None):
    T = int(math.floor(p * 65536 + 0.5))
    keep = torch.from_numpy(philox_halves(x.numel(), seed, stream_id, call) >= T).view(x.shape).to(x.device)
    y = torch.where(keep, x / (1 - T / 65536) if T < 65536 else x, torch.zeros_like(x))
    return (y if residual is None else y + residual), keep


def assert_within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    if bad.any():
        i = tuple(int(j) for j in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values, first at {i}: got {got[i].item()}, want {want[i].item()}, bound {torch.as_tensor(bound).expand_as(want)[i].item()}")
