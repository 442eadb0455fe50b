"""The training oracle against what it restates: the generator's published known answers, torch's float64 autograd and
differences of the forward pass."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import training as T


@pytest.mark.parametrize("ctr, key, want", [
    # the known answers published with the paper
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_known_answers(ctr, key, want):
    assert tuple(int(w) for w in T.philox(*ctr, *key)) == want


def test_draws_are_apart_and_fair():
    shape, p = (3, 40, 50, 21), 0.3
    base = T.dropped(shape, p, 5, 7, 1)
    n = base.size
    # the share dropped is within six standard deviations of p, and another seed, offset or site draws independently
    assert abs(base.mean() - p) < 6 * (p * (1 - p) / n) ** 0.5
    agree = p * p + (1 - p) * (1 - p)
    for other in (T.dropped(shape, p, 6, 7, 1), T.dropped(shape, p, 5, 8, 1), T.dropped(shape, p, 5, 7, 2)):
        assert abs((base == other).mean() - agree) < 6 * (agree * (1 - agree) / n) ** 0.5
    row = T.dropped(shape, p, 5, 7, 1, "row").reshape(shape)
    col = T.dropped(shape, p, 5, 7, 1, "column").reshape(shape)
    assert (row == row[:, :, :1, :1]).all() and len(np.unique(row[:, :, 0, 0])) == 2
    assert (col == col[:, :1, :, :1]).all() and len(np.unique(col[:, 0, :, 0])) == 2


@pytest.mark.parametrize("affine", [True, False])
def test_gradients_against_autograd(affine):
    rng = np.random.default_rng(3)
    z, y, dz, dl = rng.standard_normal((4, 6, 11))
    w, b = (1 + 0.1 * rng.standard_normal(11), 0.1 * rng.standard_normal(11)) if affine else (None, None)
    drop = T.dropped((2, 3, 11), 0.4, 9, shared=None)
    t = [torch.tensor(v, requires_grad=True) for v in (z, y)]
    tw = [None if v is None else torch.tensor(v, requires_grad=True) for v in (w, b)]
    zn = t[0] + torch.where(torch.tensor(drop), 0.0, t[1] / 0.6)
    xn = torch.nn.functional.layer_norm(zn, (11,), *tw)
    ref = torch.autograd.grad((zn, xn), t + [v for v in tw if v is not None], (torch.tensor(dz), torch.tensor(dl)))
    gz, gl = T.residual(z, y, 0.4, drop, w, b)
    assert np.abs(gz - zn.detach().numpy()).max() < 1e-13 and np.abs(gl - xn.detach().numpy()).max() < 1e-12
    for got, want in zip(T.residual_grads(dz, dl, gz, 0.4, drop, w), ref):
        assert np.abs(got - want.numpy()).max() < 1e-12


def test_gradients_against_differences():
    rng = np.random.default_rng(4)
    x, dy = rng.standard_normal((2, 3, 9))
    w, b = 1 + 0.1 * rng.standard_normal(9), 0.1 * rng.standard_normal(9)
    dx, dw, db = T.ln_grads(dy, x, w)
    f = lambda x, w, b: (dy * T.ln(x, w, b)).sum()  # noqa: E731
    h = 1e-5
    for got, args in ((dx, 0), (dw, 1), (db, 2)):
        vals = [x, w, b]
        for i in np.ndindex(vals[args].shape):
            up, down = [v.copy() for v in vals], [v.copy() for v in vals]
            up[args][i] += h
            down[args][i] -= h
            assert abs((f(*up) - f(*down)) / (2 * h) - got[i]) < 1e-8
