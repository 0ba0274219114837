"""Test-only: the channel-last row operators in 64 bits, written from their formulas (CPU, numpy / torch double)."""
import math

import numpy as np
import torch


def philox(counter, key):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011) of (..., 4) 32-bit counters under a key of two words."""
    c = [np.asarray(counter[..., i], dtype=np.uint64) for i in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, -1)


def keep_mask(n, p, seed, call):
    q = int(p * 65536 + 0.5)
    blocks = np.arange((n + 7) // 8, dtype=np.uint64)
    c = np.zeros((blocks.size, 4), np.uint64)
    low = np.uint64(0xFFFFFFFF)
    c[:, 0], c[:, 1] = blocks & low, blocks >> np.uint64(32)
    call &= (1 << 64) - 1
    seed &= (1 << 64) - 1
    c[:, 2], c[:, 3] = call & 0xFFFFFFFF, call >> 32
    w = philox(c, (seed & 0xFFFFFFFF, seed >> 32))
    h = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], -1).reshape(-1)[:n]
    return torch.from_numpy(h >= q), (65536.0 / (65536 - q) if q < 65536 else 0.0)


def act(z, name, slope):
    if name == "relu":
        return torch.relu(z)
    if name == "leaky_relu":
        return torch.where(z > 0, z, slope * z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    return z


def act_grad(z, name, slope):
    if name == "relu":
        return (z > 0).double()
    if name == "leaky_relu":
        return torch.where(z > 0, 1.0, slope).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def group_norm(x, groups, weight, bias, eps, name, slope, residual, cuts, factor, dy):
    """Rows x (R, C) in double; cuts: sample borders; factor: keep / (1 - p) or None.  -> dict of y, dx, dres, dw, db and of
    what the bounds of the tests are made of."""
    R, C = x.shape
    out = {k: torch.zeros(R, C, dtype=torch.float64) for k in ("y", "dx", "dres", "z", "xh", "offset", "spread1", "spread2",
                                                               "rstd")}
    dw, db, aw, ab = (torch.zeros(C, dtype=torch.float64) for _ in range(4))
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias
    for lo, hi in zip(cuts[:-1], cuts[1:]):
        if hi <= lo:
            continue
        p = x[lo:hi].reshape(hi - lo, groups, C // groups)
        mean = p.mean((0, 2), keepdim=True)
        rstd = 1 / torch.sqrt(((p - mean) ** 2).mean((0, 2), keepdim=True) + eps)
        full = lambda t: t.expand(hi - lo, groups, C // groups).reshape(hi - lo, C)   # noqa: E731
        xh = ((p - mean) * rstd).reshape(hi - lo, C)
        z = xh * w + b + (0 if residual is None else residual[lo:hi])
        f = 1.0 if factor is None else factor[lo:hi]
        out["y"][lo:hi] = act(z, name, slope) * f
        out["z"][lo:hi], out["xh"][lo:hi] = z, xh
        out["offset"][lo:hi], out["rstd"][lo:hi] = full((mean * rstd).abs()), full(rstd)
        if dy is None:
            continue
        g = dy[lo:hi] * f * act_grad(z, name, slope)
        h, v = (g * w).reshape(p.shape), xh.reshape(p.shape)
        out["dx"][lo:hi] = ((h - h.mean((0, 2), keepdim=True) - v * (h * v).mean((0, 2), keepdim=True)) * rstd).reshape(hi - lo, C)
        out["spread1"][lo:hi] = full(h.abs().mean((0, 2), keepdim=True))
        out["spread2"][lo:hi] = full((h * v).abs().mean((0, 2), keepdim=True))
        out["dres"][lo:hi] = g
        dw += (g * xh).sum(0)
        db += g.sum(0)
        aw += (g * xh).abs().sum(0)
        ab += g.abs().sum(0)
    out.update(dw=dw, db=db, aw=aw, ab=ab)
    return out


def in_8_bits(x, block_rows):
    """x (double) rounded to e4m3 under one power of two per block of block_rows x 128: the values."""
    rows, cols = x.shape
    out = torch.zeros(-(-rows // block_rows) * block_rows, -(-cols // 128) * 128, dtype=torch.float64)
    out[:rows, :cols] = x
    b = out.view(-1, block_rows, out.shape[1] // 128, 128)
    top = b.abs().amax((1, 3), keepdim=True).numpy()
    m, e = np.frexp(top)                                   # top = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = np.maximum(np.where(m <= 0.875, e - 9, e - 8), -126)
    scale = torch.from_numpy(np.where(top == 0, 1.0, np.ldexp(1.0, e)))
    v = (b / scale).numpy()
    place = np.ldexp(1.0, np.maximum(np.frexp(v)[1] - 1, -6) - 3)      # the last of four significant bits, >= 2^-9
    return (torch.from_numpy(np.rint(v / place) * place) * scale).reshape(out.shape)[:rows, :cols].clone()
