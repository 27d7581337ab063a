"""ORACLE (test infrastructure).  The per-image layers in 64 bits on the CPU: group normalisation + activation (+ dropout)
(+ shortcut) with its gradient from the written-out formulas, and dropout's mask from the generator's definition.

Channels-last arrays [N, HW, C]; statistics over one image's pixels and one group's channels (biased variance)."""
import numpy as np
import torch

SLOPE = 0.1


def philox4x32(ctr, key, rounds=10):
    """Philox-4x32 (Salmon, Moraes, Dror, Shaw, SC 2011): ctr uint32 [..., 4], key uint32 [2] -> uint32 [..., 4]."""
    c = [np.asarray(ctr[..., i], dtype=np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    m32 = np.uint64(0xFFFFFFFF)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m32]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack([v.astype(np.uint32) for v in c], -1)


def keep_mask(n, q, seed, step, layer, first=0):
    """bool [n]: elements first ... first + n - 1 of the dense tensor; ``first`` is a multiple of 8."""
    assert first % 8 == 0
    blocks = np.arange(first // 8, (first + n + 7) // 8, dtype=np.uint64)
    ctr = np.stack([blocks & np.uint64(0xFFFFFFFF), blocks >> np.uint64(32), np.full_like(blocks, step & 0xFFFFFFFF),
                    np.full_like(blocks, layer & 0xFFFFFFFF)], -1)
    w = philox4x32(ctr, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    half = np.stack([w & np.uint32(0xFFFF), w >> np.uint32(16)], -1).reshape(-1)[:n]
    return torch.from_numpy(half.astype(np.int64) >= q)


def drop_factor(shape, q, seed, step, layer):
    """float64: 65536 / (65536 - q) where an element is kept, else 0."""
    keep = keep_mask(int(np.prod(shape)), q, seed, step, layer).view(shape)
    return keep.double() * (65536.0 / (65536 - q) if q < 65536 else 0.0)


def act(z, kind):
    if kind == 2:
        return z * torch.tanh(torch.nn.functional.softplus(z, threshold=1e9))
    return torch.where(z > 0, z, SLOPE * z) if kind == 1 else z


def act_grad(z, kind):
    if kind == 2:
        t = torch.tanh(torch.nn.functional.softplus(z, threshold=1e9))
        return t + z * (1 - t * t) * torch.sigmoid(z)
    return torch.where(z > 0, torch.ones_like(z), torch.full_like(z, SLOPE)) if kind == 1 else torch.ones_like(z)


def group_norm(x, gamma, beta, groups, eps):
    """-> dict(mean, rstd [N, G]; xh, z [N, HW, C]) in float64."""
    N, HW, C = x.shape
    v = x.double().reshape(N, HW, groups, C // groups)
    mean = v.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((v - mean).pow(2).mean((1, 3), keepdim=True) + eps)
    xh = ((v - mean) * rstd).reshape(N, HW, C)
    return dict(mean=mean[:, 0, :, 0], rstd=rstd[:, 0, :, 0], xh=xh, z=xh * gamma.double() + beta.double())


def gn_act(x, gamma, beta, groups, eps, kind, factor=1.0, res=None):
    n = group_norm(x, gamma, beta, groups, eps)
    y = act(n['z'], kind) * factor
    return (y if res is None else y + res.double()), n


def gn_act_grad(x, dy, gamma, beta, groups, eps, kind, factor=1.0):
    """-> dict(dx, ggamma, gbeta, dz, h, plus what group_norm gives)."""
    n = group_norm(x, gamma, beta, groups, eps)
    N, HW, C = x.shape
    cg = C // groups
    dz = dy.double() * factor * act_grad(n['z'], kind)
    h = dz * gamma.double()
    grp = lambda t: t.reshape(N, HW, groups, cg)      # noqa: E731
    s1 = grp(h).mean((1, 3), keepdim=True)
    s2 = grp(h * n['xh']).mean((1, 3), keepdim=True)
    dx = n['rstd'][:, None, :, None] * (grp(h) - s1 - grp(n['xh']) * s2)
    return dict(n, dx=dx.reshape(N, HW, C), gbeta=dz.sum((0, 1)), ggamma=(dz * n['xh']).sum((0, 1)), dz=dz, h=h,
                s1=s1[:, 0, :, 0], s2=s2[:, 0, :, 0])
