"""numpy restatement of the sequence attention's training form (test infrastructure: what the tests compare with, never the
product): the relative position bias by buckets, the norms of queries and keys with the position rotation, the attention with
pair bias, mask and gate, and their gradients, in the precision of the inputs (float64 in the tests).

Parity status: the reference has none of the three (its attention, boltz_mlx/layers/attentionv2.py:59-83, is the forward pass
without positions, which tests/test_oracle_attention.py compares with oracle.pairformer's). The gradients are pinned by
differences of the forward passes and by torch's float64 autograd.
"""

from __future__ import annotations

import numpy as np

__all__ = ["buckets", "rel_bias", "rel_bias_grad", "qk_norm_rope", "qk_norm_rope_grads", "attention", "attention_grads"]


def buckets(edges, pos_q, pos_k, group_q=None, group_k=None):
    """[.., N, M] bucket numbers: edges at or below the distance; len(edges) + 1 for pairs of different groups."""
    d = np.asarray(pos_q)[..., :, None] - np.asarray(pos_k)[..., None, :]
    at = np.zeros(d.shape, dtype=np.int64)
    for e in edges:
        at += d >= e
    if group_q is not None:
        at[np.asarray(group_q)[..., :, None] != np.asarray(group_k)[..., None, :]] = len(edges) + 1
    return at


def rel_bias(table, at, add=None):
    """[.., H, N, M] from table [buckets, H] and bucket numbers [.., N, M]."""
    y = np.moveaxis(table[at], -1, -3)
    return y if add is None else y + add


def rel_bias_grad(dy, at, count):
    """[buckets, H] from dy [.., H, N, M] and bucket numbers [.., N, M] (shared by the batch where they have none)."""
    H = dy.shape[-3]
    at = np.broadcast_to(at, dy.shape[:-3] + dy.shape[-2:]).reshape(-1)
    rows = np.moveaxis(dy, -3, -1).reshape(-1, H)
    out = np.zeros((count, H))
    for k in range(count):
        out[k] = rows[at == k].sum(0)
    return out


def _rotate(x, pos, base, rotary, interleaved, sign):
    """x [rows, heads, C] with its first channels turned by sign * pos."""
    if not rotary or pos is None:
        return x
    angle = sign * np.asarray(pos, dtype=np.float64)[:, None] * base ** (-2.0 * np.arange(rotary // 2) / rotary)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    out = x.copy()
    first = np.arange(0, rotary, 2) if interleaved else np.arange(rotary // 2)
    second = first + (1 if interleaved else rotary // 2)
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., first] * s + x[..., second] * c
    return out


def qk_norm_rope(x, w, H, pos, eps=1e-5, base=10000.0, rotary=None, interleaved=False):
    """x [rows, H C] -> its normed and rotated heads; w [C] or None."""
    C = x.shape[1] // H
    h = x.reshape(-1, H, C)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * (1.0 if w is None else w)
    return _rotate(y, pos, base, C if rotary is None else rotary, interleaved, 1).reshape(x.shape)


def qk_norm_rope_grads(dy, x, w, H, pos, eps=1e-5, base=10000.0, rotary=None, interleaved=False):
    """(dx, dw) for dy [rows, H C]."""
    C = x.shape[1] // H
    h = x.reshape(-1, H, C)
    size = np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    xh = h / size
    g = _rotate(dy.reshape(-1, H, C), pos, base, C if rotary is None else rotary, interleaved, -1)
    dw = (g * xh).sum((0, 1))
    g = g * (1.0 if w is None else w)
    return ((g - xh * (g * xh).mean(-1, keepdims=True)) / size).reshape(x.shape), dw


def _heads(x, H):
    return x.reshape(*x.shape[:-1], H, -1).swapaxes(-2, -3)  # [S, H, n, C]


def _rows(x):
    return x.swapaxes(-2, -3).reshape(*x.shape[:-3], x.shape[-2], -1)


def attention(q, k, v, H, g=None, bias=None, mask=None, mult=1):
    """(out [S, N, H C], stats [S, H, N, 2], p [S, H, N, M]) for q, g [S, N, H C], k, v [S, M, H C], bias [S / mult, H, N, M],
    mask [S, M]. Keys that the mask leaves out take no part, whatever they hold; a row without any logit gives 0."""
    S, M = k.shape[:2]
    on = np.ones((S, M), dtype=bool) if mask is None else np.asarray(mask) != 0
    on = on | ~on.any(1, keepdims=True)
    k, v = np.where(on[..., None], k, 0.0), np.where(on[..., None], v, 0.0)
    x = _heads(q, H) @ _heads(k, H).swapaxes(-1, -2) / np.sqrt(q.shape[-1] // H)
    if bias is not None:
        x = x + np.repeat(bias, mult, 0)
    x = np.where(on[:, None, None], x, -np.inf)
    top = x.max(-1, keepdims=True)
    e = np.exp(x - np.where(np.isneginf(top), 0.0, top))
    total = e.sum(-1, keepdims=True)
    p = e / np.where(total == 0, 1.0, total)
    o = _rows(p @ _heads(v, H))
    return o if g is None else o / (1 + np.exp(-g)), np.concatenate([top, total], -1), p


def attention_grads(dout, q, k, v, H, g=None, bias=None, mask=None, mult=1):
    """{"q", "k", "v"[, "g"][, "bias"]}: the gradients of attention's output."""
    scale = 1 / np.sqrt(q.shape[-1] // H)
    o, _, p = attention(q, k, v, H, None, bias, mask, mult)
    if mask is not None:
        on = np.asarray(mask) != 0
        on = on | ~on.any(1, keepdims=True)
        k, v = np.where(on[..., None], k, 0.0), np.where(on[..., None], v, 0.0)
    d, out = dout, {}
    if g is not None:
        s = 1 / (1 + np.exp(-g))
        out["g"] = dout * o * s * (1 - s)
        d = dout * s
    d = _heads(d, H)
    dp = d @ _heads(v, H).swapaxes(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdims=True))
    out["v"] = _rows(p.swapaxes(-1, -2) @ d)
    out["q"] = _rows(ds @ _heads(k, H)) * scale
    out["k"] = _rows(ds.swapaxes(-1, -2) @ _heads(q, H)) * scale
    if bias is not None:
        out["bias"] = ds.reshape(-1, mult, *ds.shape[1:]).sum(1)
    return out
