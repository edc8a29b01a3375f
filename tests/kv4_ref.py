"""The 4-bit cache's format and the attention over it, restated in 64 bits (numpy)."""
import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def near(x):
    """What blocks of 32 along the last axis (a multiple of 32) stand for."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = np.abs(b).max(-1, keepdims=True)
    s = np.full(top.shape, -120.0)
    while True:  # the smallest s of [-120, 125] with top <= 7 2^s
        over = (top > 7 * 2.0 ** s) & (s < 125)
        if not over.any():
            break
        s = s + over
    y = np.abs(b) / 2.0 ** s
    dist = np.abs(y[..., None] - VALUES)
    best = dist.min(-1, keepdims=True)
    # of two equally near ones the even code (a step apart: one of them is even)
    code = np.where(dist == best, np.arange(8), -1)
    hi = code.max(-1)
    lo = np.where(code >= 0, code, 99).min(-1)
    code = np.where(hi % 2 == 0, hi, lo)
    return (np.sign(b) * VALUES[code] * 2.0 ** s).reshape(x.shape)


def near_kv(k, v):
    """k, v [B,H,P,128]: keys blocked along dimensions, values along 32 keys."""
    p = k.shape[2]
    vt = np.pad(np.swapaxes(np.asarray(v, np.float64), 2, 3), ((0, 0), (0, 0), (0, 0), (0, -p % 32)))
    return near(k), np.swapaxes(near(vt)[..., :p], 2, 3)


def attention(q, k, v, scale, valid=None):
    """(out, sum p |v|) [B,Sq,H,128]; valid [B, keys]."""
    s = np.einsum("bhqd,bhkd->bhqk", np.asarray(q, np.float64), k) * scale
    if valid is not None:
        s = np.where(valid[:, None, None, :] != 0, s, -np.inf)
        v = np.where(valid[:, None, :, None] != 0, v, 0.0)  # a hidden key's value does not count
    with np.errstate(invalid="ignore"):
        e = np.exp(s - s.max(-1, keepdims=True))
        p = e / e.sum(-1, keepdims=True)
    return np.einsum("bhqk,bhkd->bqhd", p, v), np.einsum("bhqk,bhkd->bqhd", p, np.abs(v))
