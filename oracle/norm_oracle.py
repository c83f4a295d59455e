"""Dropout and group norm with an activation, from their definitions, in numpy / torch float64 on the CPU.

Activations are (B, H, W, C) float64 tensors without padding.  The generator is Philox4x32-10 as published (Salmon,
Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC11); its known answers are in the tests."""
import math

import numpy as np
import torch


def philox4x32(counter, key, rounds=10):
    """counter: four arrays of 32-bit values (as uint64), key: two.  Returns four arrays."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [np.uint64(v) for v in key]
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(rounds):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> sh) ^ c[1] ^ k[0], q & low, (p >> sh) ^ c[3] ^ k[1], p & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return c


def pad_ch(c):
    return 32 if c <= 32 else (c + 15) // 16 * 16


def kept_count(p):
    return math.floor((1.0 - p) * 65536 + 0.5)


def units_kept(units, p, seed, offset):
    """Whether each of these unit numbers survives."""
    e = np.asarray(units, dtype=np.uint64)
    n = e >> np.uint64(3)
    z = np.zeros_like(n)
    w = philox4x32([n & np.uint64(0xFFFFFFFF), n >> np.uint64(32), z + np.uint64(offset & 0xFFFFFFFF), z + np.uint64(offset >> 32)],
                   [seed & 0xFFFFFFFF, seed >> 32])
    j = (e & np.uint64(7)).astype(np.int64)
    word = np.choose(j >> 1, w)
    half = (word >> (np.uint64(16) * (e & np.uint64(1)))) & np.uint64(0xFFFF)
    return half < np.uint64(kept_count(p))


def drop_factor(shape, p, seed, offset=0, per_channel=False):
    """What each element is multiplied by, (B, H, W, C) float64: 0 or 65536 / K."""
    B, H, W, C = shape
    pitch = pad_ch(C)
    rows = np.arange(B if per_channel else B * H * W, dtype=np.uint64)
    units = rows[:, None] * np.uint64(pitch) + np.arange(C, dtype=np.uint64)[None]
    K = kept_count(p)
    f = np.where(units_kept(units, p, seed, offset), 65536.0 / max(K, 1), 0.0)
    f = f.reshape(B, 1, 1, C) if per_channel else f.reshape(B, H, W, C)
    return torch.from_numpy(np.broadcast_to(f, shape).copy())


def act(z, kind):
    return {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, torch.where(z <= 0, torch.zeros_like(z), z)),
            "silu": lambda: z * torch.sigmoid(z), "gelu": lambda: 0.5 * z * torch.erfc(-z * math.sqrt(0.5))}[kind]()


def act_slope(z, kind):
    if kind == "none":
        return torch.ones_like(z)
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * torch.sigmoid(-z))
    return 0.5 * torch.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _per_channel(t, cg):
    """(B, G) -> (B, 1, 1, C)"""
    return t.repeat_interleave(cg, 1)[:, None, None]


def _group_mean(t, groups):
    B, H, W, C = t.shape
    return t.reshape(B, H * W, groups, C // groups).mean((1, 3))


def group_norm_act_fwd(x, groups, gamma, beta, kind, eps, factor=None):
    """(y, mean, rstd, z) of a float64 x."""
    cg = x.shape[3] // groups
    mean = _group_mean(x, groups)
    d = x - _per_channel(mean, cg)
    rstd = (_group_mean(d * d, groups) + eps) ** -0.5
    z = d * _per_channel(rstd, cg) * gamma + beta
    y = act(z, kind)
    return (y if factor is None else torch.where(factor > 0, y * factor, torch.zeros_like(y))), mean, rstd, z


def group_norm_act_bwd(x, dy, mean, rstd, groups, gamma, beta, kind, factor=None):
    """(dx, dgamma, dbeta, parts) from given statistics; parts are the terms a rounding bound is made of."""
    cg = x.shape[3] // groups
    r = _per_channel(rstd, cg)
    h = (x - _per_channel(mean, cg)) * r
    z = h * gamma + beta
    da = dy if factor is None else torch.where(factor > 0, dy * factor, torch.zeros_like(dy))
    dz = da * act_slope(z, kind)
    t = dz * gamma
    m1, m2 = _per_channel(_group_mean(t, groups), cg), _per_channel(_group_mean(t * h, groups), cg)
    dx = r * (t - m1 - h * m2)
    parts = dict(r=r, h=h, z=z, da=da, dz=dz, t=t, m1=m1, m2=m2, a1=_per_channel(_group_mean(t.abs(), groups), cg),
                 a2=_per_channel(_group_mean((t * h).abs(), groups), cg))
    return dx, (dz * h).sum((0, 1, 2)), dz.sum((0, 1, 2)), parts
