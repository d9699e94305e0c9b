"""float64 oracle of group normalisation with an activation and of counter-based dropout, channels last (numpy, formula by formula)."""
import numpy as np
from scipy.special import ndtr


def philox4x32(counter, key, rounds=7):
    """Philox4x32 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): counter [..., 4], key [2] of
    32-bit words -> [..., 4] of 32-bit words (uint64 arrays)."""
    c = [np.asarray(counter, np.uint64)[..., k] for k in range(4)]
    k0, k1 = (int(k) for k in key)
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> sh) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> sh) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, -1)


def drop_numbers(first, count, seed, offset):
    """The 16-bit numbers of elements first .. first + count - 1."""
    b = np.arange(first // 8, (first + count + 7) // 8, dtype=np.uint64)
    ctr = np.stack([b & np.uint64(0xFFFFFFFF), b >> np.uint64(32), np.full_like(b, offset & 0xFFFFFFFF), np.full_like(b, offset >> 32)], -1)
    w = philox4x32(ctr, (seed & 0xFFFFFFFF, seed >> 32))
    n = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], -1).reshape(-1)
    return n[first % 8:first % 8 + count].astype(np.int64)


def drop_factor(shape, p, seed, offset, first=0):
    """0 where an element is dropped, 65536 / (65536 - t) where it is kept, t = round(65536 p)."""
    t = int(np.rint(p * 65536))
    if t == 65536:
        return np.zeros(shape)
    n = drop_numbers(first, int(np.prod(shape)), seed, offset)
    return np.where(n >= t, 65536.0 / (65536 - t), 0.0).reshape(shape)


def act(z, name):
    if name == "relu":
        return np.where(z < 0, 0.0, z)
    if name == "silu":
        return z / (1 + np.exp(-z))
    return z * ndtr(z) if name == "gelu" else z


def act_grad(z, name):
    if name == "relu":
        return np.where(z <= 0, 0.0, 1.0)
    if name == "silu":
        s = 1 / (1 + np.exp(-z))
        return s + z * s * (1 - s)
    return ndtr(z) + z * np.exp(-z * z / 2) / np.sqrt(2 * np.pi) if name == "gelu" else np.ones_like(z)


def stats(x, groups, eps):
    """[N, G] mean and rstd of x [N, H, W, C]."""
    n, h, w, c = x.shape
    v = x.reshape(n, h * w, groups, c // groups)
    mean = v.mean(axis=(1, 3))
    return mean, 1 / np.sqrt(((v - mean[:, None, :, None]) ** 2).mean(axis=(1, 3)) + eps)


def per_channel(s, c):
    """[N, G] -> [N, 1, 1, C]."""
    return np.repeat(s, c // s.shape[1], axis=1)[:, None, None, :]


def forward(x, groups, gamma, beta, eps, name, factor=1.0):
    """y, mean, rstd and the pre-activations z, xh."""
    c = x.shape[3]
    mean, rstd = stats(x, groups, eps)
    xh = (x - per_channel(mean, c)) * per_channel(rstd, c)
    z = xh * gamma + beta
    return act(z, name) * factor, mean, rstd, z, xh


def backward(dy, x, groups, gamma, beta, eps, name, factor=1.0):
    """dx, dgamma, dbeta."""
    n, h, w, c = x.shape
    _, mean, rstd, z, xh = forward(x, groups, gamma, beta, eps, name)
    dz = dy * factor * act_grad(z, name)
    a, b = dz.sum(axis=(1, 2)), (dz * xh).sum(axis=(1, 2))
    m = h * w * (c // groups)
    s1, s2 = ((v * gamma).reshape(n, groups, -1).sum(2) / m for v in (a, b))
    dx = per_channel(rstd, c) * (dz * gamma - per_channel(s1, c) - xh * per_channel(s2, c))
    return dx, b.sum(0), a.sum(0)
