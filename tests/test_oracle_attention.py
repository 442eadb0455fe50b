"""The attention oracle against what it restates: torch's float64 autograd, differences of the forward passes, and the single
track's attention of the reference's formulas."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention as T


def rand(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape)


def tt(x):
    return None if x is None else torch.tensor(x, dtype=torch.float64, requires_grad=True)


def difference(f, x, d, h=1e-6):
    """The derivative of f at x in direction d."""
    return (f(x + h * d) - f(x - h * d)) / (2 * h)


@pytest.mark.parametrize("gate, biased, masked, mult", [(True, True, True, 2), (False, True, False, 1), (True, False, True, 1),
                                                        (False, False, False, 2)])
def test_attention_gradients(gate, biased, masked, mult):
    S, N, M, H, C = 4, 5, 7, 3, 8
    q, k, v, dout = rand(1, S, N, H * C), rand(2, S, M, H * C), rand(3, S, M, H * C), rand(4, S, N, H * C)
    g = rand(5, S, N, H * C) if gate else None
    bias = rand(6, S // mult, H, N, M) if biased else None
    mask = None
    if masked:
        mask = (rand(7, S, M) > -0.5).astype(np.float64)
        mask[1] = 0
    out, stats, p = T.attention(q, k, v, H, g, bias, mask, mult)
    grads = T.attention_grads(dout, q, k, v, H, g, bias, mask, mult)
    ts = {n: tt(x) for n, x in dict(q=q, k=k, v=v, g=g, bias=bias).items()}
    x = torch.einsum("snhc,smhc->shnm", ts["q"].view(S, N, H, C), ts["k"].view(S, M, H, C)) / C ** 0.5
    if biased:
        x = x + ts["bias"].repeat_interleave(mult, 0)
    if masked:
        off = torch.tensor(mask) == 0
        off = off & ~off.all(1, keepdim=True)
        x = x.masked_fill(off[:, None, None], -torch.inf)
    y = torch.einsum("shnm,smhc->snhc", x.softmax(-1), ts["v"].view(S, M, H, C)).reshape(S, N, H * C)
    if gate:
        y = y * torch.sigmoid(ts["g"])
    assert np.allclose(out, y.detach().numpy(), rtol=1e-12, atol=1e-12)
    assert np.allclose(stats[..., 0] + np.log(stats[..., 1]), torch.logsumexp(x, -1).detach().numpy(), rtol=1e-12)
    assert np.allclose(p.sum(-1), 1)
    y.backward(torch.tensor(dout))
    for n, d in grads.items():
        assert np.allclose(d, ts[n].grad.numpy(), rtol=1e-10, atol=1e-12), n
    args = dict(q=q, k=k, v=v, g=g, bias=bias)
    for n in grads:
        d = rand(8, *args[n].shape)
        f = lambda x: (T.attention(**{**args, n: x}, H=H, mask=mask, mult=mult)[0] * dout).sum()  # noqa: E731, B023
        assert np.isclose(difference(f, args[n], d), (grads[n] * d).sum(), rtol=1e-6, atol=1e-8), n


def test_attention_is_the_single_tracks():
    """As the reference's formulas have it where every sample has a key: the mask as an addition of -inf's stand-in, 1e6."""
    N, H, C = 9, 2, 8
    q, k, v, g, bias = rand(1, 1, N, H * C), rand(2, 1, N, H * C), rand(3, 1, N, H * C), rand(4, 1, N, H * C), rand(5, 1, H, N, N)
    mask = np.ones((1, N))
    mask[0, 6:] = 0
    x = np.einsum("ihc,jhc->hij", q[0].reshape(N, H, C), k[0].reshape(N, H, C)) / C ** 0.5 + bias[0] + (1 - mask[0]) * -1e6
    e = np.exp(x - x.max(-1, keepdims=True))
    p = e / e.sum(-1, keepdims=True)
    want = np.einsum("hij,jhc->ihc", p, v[0].reshape(N, H, C)).reshape(N, H * C) / (1 + np.exp(-g[0]))
    assert np.allclose(T.attention(q, k, v, H, g, bias, mask)[0][0], want, rtol=1e-12, atol=1e-12)


def test_rows_and_keys_that_take_no_part():
    S, N, M, H, C = 1, 4, 6, 1, 8
    q, k, v, bias = rand(1, S, N, C), rand(2, S, M, C), rand(3, S, M, C), rand(4, 1, H, N, M)
    mask = np.array([[1.0, 0, 1, 1, 0, 1]])
    kb, vb, bb = k.copy(), v.copy(), bias.copy()
    kb[0, 1], vb[0, 4], bb[..., 1] = np.nan, np.inf, np.nan
    for a, b in zip(T.attention(q, k, v, H, None, bias, mask), T.attention(q, kb, vb, H, None, bb, mask)):
        assert np.array_equal(a, b)
    bias[0, 0, 2] = -np.inf
    out, stats, p = T.attention(q, k, v, H, None, bias, mask)
    assert (out[0, 2] == 0).all() and stats[0, 0, 2, 1] == 0 and np.isneginf(stats[0, 0, 2, 0]) and (p[0, 0, 2] == 0).all()
    grads = T.attention_grads(rand(5, S, N, C), q, k, v, H, None, bias, mask)
    assert (grads["q"][0, 2] == 0).all() and (grads["bias"][0, 0, 2] == 0).all() and (grads["k"][0, 1] == 0).all()
    bias[0, 0, 2] = np.finfo(np.float64).min  # the type's lowest value everywhere is a softmax over equals
    assert np.allclose(T.attention(q, k, v, H, None, bias, mask)[2][0, 0, 2], mask[0] / 4)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [0, 4, 10])
def test_norms(interleaved, rotary):
    rows, H, C = 5, 3, 10
    x, w, dy, pos = rand(1, rows, H * C), 1 + 0.2 * rand(2, C), rand(3, rows, H * C), np.array([0, 1, 7, 1000, 123456])
    kw = dict(rotary=rotary, interleaved=interleaved)
    dx, dw = T.qk_norm_rope_grads(dy, x, w, H, pos, **kw)
    f = lambda x, w: (T.qk_norm_rope(x, w, H, pos, **kw) * dy).sum()  # noqa: E731
    d = rand(4, rows, H * C)
    assert np.isclose(difference(lambda a: f(a, w), x, d), (dx * d).sum(), rtol=1e-6)
    d = rand(5, C)
    assert np.isclose(difference(lambda a: f(x, a), w, d), (dw * d).sum(), rtol=1e-6)
    y = T.qk_norm_rope(x, None, H, pos, **kw).reshape(rows, H, C)
    assert np.allclose((y * y).mean(-1), 1, atol=1e-3)  # a rotation keeps the norm
    # products of queries and keys depend on the positions' difference alone
    a, b = rand(6, 1, C), rand(7, 1, C)
    dots = [(T.qk_norm_rope(a, None, 1, [p + 11], **kw) * T.qk_norm_rope(b, None, 1, [p], **kw)).sum() for p in (0, 5, 3000)]
    assert np.allclose(dots, dots[0])


def test_buckets_and_bias():
    pos = np.array([1, 2, 3, 7, 1, 2])
    chain = np.array([0, 0, 0, 0, 1, 1])
    at = T.buckets([-1, 0, 1, 2], pos, pos, chain, chain)
    assert (at[0, 1], at[1, 0], at[0, 0], at[3, 0], at[0, 3], at[0, 4], at[4, 5]) == (1, 3, 2, 4, 0, 5, 1)
    table, dy = rand(1, 6, 3), rand(2, 2, 3, 6, 6)
    d = rand(3, 6, 3)
    grad = T.rel_bias_grad(dy, at, 6)
    assert np.isclose(((T.rel_bias(table + d, at) - T.rel_bias(table, at)) * dy).sum(), (grad * d).sum())
    assert T.rel_bias(table, at)[2, 0, 3] == table[0, 2]


def test_rel_buckets():
    from boltz_mlx_amd import kernels as K

    for edges in ([], [0], [-3, -1, 0, 4, 9], K.clipped_edges(1), K.clipped_edges(32), list(range(-100, 154))):
        for other in (False, True):
            b = K.rel_buckets(edges, other, device="cpu")
            d = np.arange(-400, 400)
            want = T.buckets(edges, d, np.zeros(1, dtype=np.int64))[:, 0]
            got = b.lut.numpy()[np.clip(d - b.lo, 0, len(b.lut) - 1)]
            assert np.array_equal(got, want) and b.count == len(edges) + 1 + other and b.other == other
    assert len(K.clipped_edges(32)) == 64
    for bad in ([1, 1], [3, 2], list(range(256)), [0, 16384]):
        with pytest.raises(ValueError, match="rel_buckets"):
            K.rel_buckets(bad, device="cpu")
    with pytest.raises(ValueError, match="rel_buckets"):
        K.rel_buckets(list(range(255)), True, device="cpu")
