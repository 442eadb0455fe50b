"""numpy restatement of the training operators (test infrastructure: what the tests compare with, never the product):
LayerNorm with its backward pass, dropout drawn from Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
numbers: as easy as 1, 2, 3", SC 2011) and the residual update z + dropout(y) with its LayerNorm. Rows are the last axis.

Parity status: the reference runs inference only, so there are no outputs of its own to compare with. Pinned by
tests/test_oracle_training.py: the generator against the paper's known answers, the gradients against torch's float64
autograd and against differences.
"""

from __future__ import annotations

import numpy as np

__all__ = ["philox", "dropped", "dropout", "ln", "ln_grads", "residual", "residual_grads"]

LOW = np.uint64(0xFFFFFFFF)
HALF = np.uint64(32)


def philox(c0, c1, c2, c3, k0: int, k1: int):
    """The four 32-bit words of Philox4x32-10 for counters c0..c3 and key k0, k1 (uint64 arrays of 32-bit values)."""
    c = [np.asarray(v, dtype=np.uint64) for v in np.broadcast_arrays(c0, c1, c2, c3)]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> HALF) ^ c[1] ^ np.uint64(k0), b & LOW, (a >> HALF) ^ c[3] ^ np.uint64(k1), a & LOW]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def _words(n, seed: int, offset: int, site: int):
    """Word n % 4 of block n // 4 for an array of draw numbers n."""
    n = np.asarray(n, dtype=np.uint64)
    block, word = n >> np.uint64(2), (n & np.uint64(3)).astype(np.int64)
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    w = philox(block & LOW, (block >> HALF) | np.uint64(site << 16), np.uint64(offset & 0xFFFFFFFF),
               np.uint64(offset >> 32), seed & 0xFFFFFFFF, seed >> 32)
    return np.choose(word, w)


def dropped(shape, p: float, seed: int, offset: int = 0, site: int = 0, shared=None, first_row: int = 0, rows=None):
    """Truth values: which elements of a tensor of this shape (rows first_row .. of its [rows, D] form) are dropped."""
    D = shape[-1]
    total = int(np.prod(shape[:-1], dtype=np.int64))
    r = np.arange(first_row, total if rows is None else first_row + rows, dtype=np.int64)
    limit = np.uint64(round(p * 2 ** 32))
    if shared is None:
        per = (D + 3) // 4
        n = r[:, None] * (4 * per) + np.arange(D)
        return _words(n, seed, offset, site) < limit
    I, J = shape[-3], shape[-2]
    g = r // J if shared == "row" else r // (I * J) * J + r % J
    return np.broadcast_to((_words(g, seed, offset, site) < limit)[:, None], (len(r), D))


def dropout(x, p: float, drop):
    return np.where(drop, 0.0, x / (1.0 - p) if p < 1 else 0.0)


def _centred(x, eps):
    c = x - x.mean(-1, keepdims=True)
    return c, 1.0 / np.sqrt((c * c).mean(-1, keepdims=True) + eps)


def ln(x, w=None, b=None, eps: float = 1e-5):
    c, rstd = _centred(x, eps)
    y = c * rstd
    return y * (1.0 if w is None else w) + (0.0 if b is None else b)


def ln_grads(dy, x, w=None, eps: float = 1e-5):
    """(dx, dw, db) of ln over rows [R, D]."""
    c, rstd = _centred(x, eps)
    xh = c * rstd
    g = dy if w is None else dy * w
    dx = rstd * (g - g.mean(-1, keepdims=True) - xh * (g * xh).mean(-1, keepdims=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def residual(z, y, p, drop, w=None, b=None, eps: float = 1e-5):
    z_new = z + dropout(y, p, drop)
    return z_new, ln(z_new, w, b, eps)


def residual_grads(dz_new, dln, z_new, p, drop, w=None, eps: float = 1e-5):
    dx, dw, db = ln_grads(dln, z_new, w, eps)
    dz = dx if dz_new is None else dz_new + dx
    return dz, dropout(dz, p, drop), dw, db
