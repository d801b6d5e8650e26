"""The token operators (yolopoint_amd/utils/token_ops.py) from their definitions, in 64 bits on the CPU: test infrastructure only.  No reference
counterpart.  Rounding to a storage type happens where the definition has it (the stored sum z) and nowhere else."""
import numpy as np
import torch


def philox4x32_10(counter, key):
    """Philox4x32-10 (Salmon et al., SC 2011): counter uint64 arrays (low, high words of 64 bits), key a 64-bit number -> uint32 [n, 4]."""
    u = np.uint64
    low = u(0xFFFFFFFF)
    lo, hi = (np.asarray(c, dtype=u) for c in counter)
    c = [lo & low, lo >> u(32), hi & low, hi >> u(32)]
    k0, k1 = key & 0xFFFFFFFF, key >> 32
    for _ in range(10):
        p0, p1 = u(0xD2511F53) * c[0], u(0xCD9E8D57) * c[2]
        c = [(p1 >> u(32)) ^ c[1] ^ u(k0), p1 & low, (p0 >> u(32)) ^ c[3] ^ u(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, axis=-1).astype(np.uint32)


def keep_mask(n, p, seed, offset, start=0):
    """Which of the elements start .. start + n - 1 are kept (bool [n])."""
    g = np.arange(start // 8, (start + n + 7) // 8, dtype=np.uint64)
    words = philox4x32_10((g, np.full_like(g, offset)), seed)
    halves = np.ascontiguousarray(words).view("<u2").reshape(-1).astype(np.int64)
    first = start - start // 8 * 8
    return torch.from_numpy(halves[first:first + n] >= threshold(p))


def threshold(p):
    return int(np.floor(p * 65536.0 + 0.5))


def drop_scale(p):
    t = threshold(p)
    return float(np.float32(65536.0 / (65536 - t))) if t < 65536 else 0.0


def dropout(x, p, seed, offset, residual=None):
    keep = keep_mask(x.numel(), p, seed, offset).view(x.shape)
    y = torch.where(keep, x.double() * drop_scale(p), torch.zeros((), dtype=torch.float64))
    return y if residual is None else y + residual.double()


def layer_norm(x, w, b, eps):
    """-> y, mean, rstd, xhat"""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xhat = (x - mean) * rstd
    y = xhat * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double())
    return y, mean, rstd, xhat


def layer_norm_backward(x, w, dy, eps):
    """-> dx, dweight, dbias"""
    _, _, rstd, xhat = layer_norm(x, None, None, eps)
    dy = dy.double()
    h = dy if w is None else dy * w.double()
    dx = rstd * (h - h.mean(-1, keepdim=True) - xhat * (h * xhat).mean(-1, keepdim=True))
    D = x.shape[-1]
    return dx, (dy * xhat).reshape(-1, D).sum(0), dy.reshape(-1, D).sum(0)


def stored_sum(x, residual, p, seed, offset):
    return dropout(x, p, seed, offset, residual).float().to(x.dtype)          # (by way of fp32, as the definition has it)


def rotary(x, positions, inv_freq, interleaved, layout, scale, inverse=False):
    """x [B, T, H, D] or [B, H, T, D]; positions [T], [B, T], [T, 2] or [B, T, 2] as `token_ops.rotary` reads them."""
    B, T = (x.shape[0], x.shape[1]) if layout == "bthd" else (x.shape[0], x.shape[2])
    pos, half = positions.double(), inv_freq.numel()
    R = 2 * half
    if tuple(pos.shape) in ((T,), (1, T), (B, T)):
        angle = pos.reshape(-1, T, 1) * inv_freq
    else:
        pos = pos.reshape(-1, T, 2)
        angle = torch.cat([pos[..., :1] * inv_freq[:half // 2], pos[..., 1:] * inv_freq[half // 2:]], -1)
    angle = angle.unsqueeze(2 if layout == "bthd" else 1)
    c, s = angle.cos() * scale, angle.sin() * scale * (-1.0 if inverse else 1.0)
    out = x.double().clone()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, half), slice(half, R))
    u, v = x[..., a].double(), x[..., b].double()
    out[..., a], out[..., b] = u * c - v * s, v * c + u * s
    return out
