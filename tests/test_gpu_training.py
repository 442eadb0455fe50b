"""The training operators on the GPU (LayerNorm at any width with its backward pass, dropout, the residual update) against
the float64 oracle.

Tolerances, from the kernels' arithmetic: u = 2^-24 is fp32's half step. A row's sum of D <= 8192 terms passes at most 15
additions (3 inside a chunk, 4 chunks, 6 steps over a wave, 2 over the waves), so it errs by 16u times the mean of the
terms' sizes after the division:
  mean: 16u M, M the row's largest |x|;  xh: (1 + |xh|) E with E = u (16 M rstd + 14);
  y: |w| (1 + |xh|) E + 2u (|xh w| + |b|);
  dx, with G the row's largest |dy w|: c1 errs by 17u G, c2 by G (18u + 2E) (the mean of |xh| is at most 1), so the whole by
  rstd G (1 + |xh|) (6E + 60u);
  dw: each term errs by |dy| (1 + |xh|) E, the sum by its depth (the rows of one thread, its wave, the workgroups) times u
  times the terms' sizes.
Outputs in fewer bits add their half step (fp16 2^-11, bf16 2^-8, relative) and fp16's smallest half step 2^-25."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import training as T  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
STEP = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 1e-37, F16: 2.0 ** -25, BF16: 1e-37}
TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]
# every row layout's first and last width, whole chunks and odd ones
WIDTHS = [8, 9, 15, 63, 64, 65, 77, 100, 128, 129, 250, 256, 257, 384, 511, 513, 768, 1000, 1021, 1025, 1536, 2048, 2049,
          2055, 4096, 4097, 8185, 8192]
ROWS = [1, 2, 3, 5, 31, 33, 70]


def K():
    from boltz_mlx_amd import kernels

    return kernels


def rand(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def acts(seed, rows, D, dtype):
    """Rows with a mean and a scale of their own."""
    return (rand(seed, rows, D) * (0.5 + rand(seed + 1, rows, 1).abs()) + rand(seed + 2, rows, 1)).to(dtype)


def np64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def close(got, ref, tol, dtype=None):
    dtype = dtype or got.dtype
    err = np.abs(np64(got) - ref)
    lim = tol + (STEP[dtype] * (np.abs(ref) + tol) + TINY[dtype] + U * np.abs(ref))
    bad = ~(err <= lim)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float((err / lim).max()))


def row_terms(x, eps=1e-5):
    """(xh, rstd, E) of the rows, as the docstring has them."""
    c = x - x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + eps)
    return c * rstd, rstd, U * (16 * np.abs(x).max(-1, keepdims=True) * rstd + 14)


def ln_tol(x, w, b, eps=1e-5):
    xh, _, E = row_terms(x, eps)
    w = 1.0 if w is None else w
    return np.abs(w) * (1 + np.abs(xh)) * E + 2 * U * (np.abs(xh * w) + (0 if b is None else np.abs(b)))


def dx_tol(dy, x, w, eps=1e-5):
    xh, rstd, E = row_terms(x, eps)
    G = np.abs(dy if w is None else dy * w).max(-1, keepdims=True)
    return rstd * G * (1 + np.abs(xh)) * (6 * E + 60 * U)


def dw_tol(dy, x):
    xh, _, E = row_terms(x)
    depth = len(x) // 256 + 128
    return (np.abs(dy) * (1 + np.abs(xh)) * E).sum(0) + depth * U * np.abs(dy * xh).sum(0), depth * U * np.abs(dy).sum(0)


def params(seed, D, affine=True):
    return (1 + rand(seed, D, scale=0.1), rand(seed + 1, D, scale=0.1)) if affine else (None, None)


def check_grads(dx, dw, db, dy, x, w):
    dy, x, w = np64(dy), np64(x), np64(w)
    rx, rw, rb = T.ln_grads(dy, x, w)
    close(dx, rx, dx_tol(dy, x, w))
    tw, tb = dw_tol(dy, x)
    if dw is not None:
        close(dw, rw, tw)
    if db is not None:
        close(db, rb, tb)


# -------------------------------------------------------------------------------------------------- LayerNorm

@pytest.mark.parametrize("D", WIDTHS)
def test_layer_norm_widths(D):
    for k, (tx, ty) in enumerate(TYPES):
        rows = ROWS[(k + D) % len(ROWS)]
        x, (w, b) = acts(D + k, rows, D, tx), params(D, D)
        y = K().layer_norm(x, w, b, 1e-5, out_dtype=ty)
        assert y.dtype == ty and y.shape == x.shape
        close(y, T.ln(np64(x), np64(w), np64(b)), ln_tol(np64(x), np64(w), np64(b)))


@pytest.mark.parametrize("D", WIDTHS)
def test_layer_norm_bwd_widths(D):
    for k, (tx, ty) in enumerate(TYPES):
        rows = ROWS[(k + D) % len(ROWS)]
        x, dy, (w, _) = acts(D + k, rows, D, tx), rand(D + k + 9, rows, D, dtype=ty), params(D, D)
        dx, dw, db = K().layer_norm_bwd(dy, x, w)
        assert dx.dtype == tx and dw.dtype == db.dtype == F32
        check_grads(dx, dw, db, dy, x, w)


@pytest.mark.parametrize("rows, D", [(257, 64), (4099, 128), (20011, 72), (1500, 384), (3001, 1021), (1100, 2100),
                                     (1030, 8192), (70001, 16)])
def test_layer_norm_bwd_many_rows(rows, D):
    """Several workgroups, each with several rows: the partial sums and their meeting."""
    x, dy, (w, _) = acts(1, rows, D, F32), rand(2, rows, D, dtype=F16), params(3, D)
    dx, dw, db = K().layer_norm_bwd(dy, x, w)
    check_grads(dx, dw, db, dy, x, w)
    again = K().layer_norm_bwd(dy, x, w)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))  # a fixed order of sums


def test_layer_norm_without_affine_and_needs():
    x, dy = acts(5, 300, 200, BF16), rand(6, 300, 200, dtype=BF16)
    close(K().layer_norm(x, None, None, out_dtype=BF16), T.ln(np64(x)), ln_tol(np64(x), None, None))
    dx, dw, db = K().layer_norm_bwd(dy, x, None, need_weight=False, need_bias=False)
    assert dw is None and db is None
    check_grads(dx, None, None, dy, x, None)
    w = 1 + rand(7, 200, scale=0.1)
    full = K().layer_norm_bwd(dy, x, w)
    for need in ((True, False), (False, True)):
        part = K().layer_norm_bwd(dy, x, w, need_weight=need[0], need_bias=need[1])
        assert torch.equal(part[0], full[0])
        for got, ref, n in zip(part[1:], full[1:], need):
            assert torch.equal(got, ref) if n else got is None


def test_layer_norm_hard_rows():
    """Rows with a large mean (the two-pass variance), constant rows (variance 0: eps alone), and rows with an infinity or
    a NaN, which spoil themselves and no other."""
    x = rand(8, 40, 96)
    x[0:8] += 300.0
    x[8:12] = 2.5
    x[13, 7], x[14, 95], x[15, 0] = float("inf"), float("nan"), float("-inf")
    dy, (w, b) = rand(9, 40, 96), params(10, 96)
    spoilt = [13, 14, 15]
    fine = [r for r in range(40) if r not in spoilt]
    y, (dx, _, _) = K().layer_norm(x, w, b), K().layer_norm_bwd(dy, x, w)
    assert torch.isnan(y[spoilt]).all() and torch.isnan(dx[spoilt]).all()
    xf, df = np64(x)[fine], np64(dy)[fine]
    close(y[fine], T.ln(xf, np64(w), np64(b)), ln_tol(xf, np64(w), np64(b)))
    rx, rw, rb = T.ln_grads(df, xf, np64(w))
    close(dx[fine], rx, dx_tol(df, xf, np64(w)))
    _, dw, db = K().layer_norm_bwd(dy[fine], x[fine], w)
    tw, tb = dw_tol(df, xf)
    close(dw, rw, tw)
    close(db, rb, tb)


def test_layer_norm_tiny_and_huge_rows():
    """Variances that are denormal in fp32 (eps 0) and squares near its largest value. A square of s errs by half a denormal
    step, 2^-150, and so does the mean of the squares: 2^-149 / s^2 of the variance at most, half of that of rstd and xh."""
    w, b = params(1, 130)
    for scale in (1e-19, 1e-20, 1e17):
        x, dy = rand(2, 20, 130, scale=scale), rand(3, 20, 130)
        y, (dx, _, _) = K().layer_norm(x, w, b, 0.0), K().layer_norm_bwd(dy, x, w, 0.0)
        xr, dr, wr = np64(x), np64(dy), np64(w)
        xh, rstd, _ = row_terms(xr, 0.0)
        rel = 2.0 ** -149 / xr.var(-1, keepdims=True)
        close(y, T.ln(xr, wr, np64(b), 0.0), ln_tol(xr, wr, np64(b), 0.0) + rel * np.abs(xh * wr))
        G = np.abs(dr * wr).max(-1, keepdims=True)
        close(dx, T.ln_grads(dr, xr, wr, 0.0)[0], dx_tol(dr, xr, wr, 0.0) + 4 * rel * rstd * G * (1 + np.abs(xh)))


@pytest.mark.parametrize("D", [64, 77, 128, 384, 2056, 8191])
def test_strides_offsets_and_neighbours(D):
    """Views at odd offsets (element alignment only), transposed inputs, and the memory around the outputs untouched."""
    from boltz_mlx_amd import _lib

    rows = 37
    base = acts(11, rows + 2, D, F16).flatten()
    x = base[3:3 + rows * D].view(rows, D)
    g = rand(12, D, rows, dtype=F16).t()
    w = (1 + rand(13, D + 1, scale=0.1))[1:]
    check_grads(*K().layer_norm_bwd(g, x, w), g, x, w)
    close(K().layer_norm(x, w, None, out_dtype=F16), T.ln(np64(x), np64(w)), ln_tol(np64(x), np64(w), None))
    # outputs inside larger buffers
    gc = g.contiguous()
    dx, dw = torch.full((rows * D + 40,), 7.0, dtype=F16, device="cuda"), torch.full((2 * D + 40,), 7.0, device="cuda")
    ws = torch.full((max(1, _lib.load().bzpf_layernorm_bwd_ws(rows, D) // 4) + 16,), 7.0, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    _lib.call("bzpf_layernorm_bwd", gc.data_ptr(), 1, x.data_ptr(), 1, w.data_ptr(), 1e-5, dx[11:].data_ptr(),
              dw[9:].data_ptr(), dw[20 + D:].data_ptr(), ws.data_ptr(), 4 * (ws.numel() - 16), rows, D, st)
    torch.cuda.synchronize()
    check_grads(dx[11:11 + rows * D].view(rows, D), dw[9:9 + D], dw[20 + D:20 + 2 * D], gc, x, w)
    for t in (dx[:11], dx[11 + rows * D:], dw[:9], dw[9 + D:20 + D], dw[20 + 2 * D:], ws[-16:]):
        assert (t == 7.0).all()


def test_no_rows():
    x, w, rng = torch.empty(0, 4, 32, device="cuda"), torch.ones(32, device="cuda"), K().dropout_rng(1)
    assert K().layer_norm(x, w, w).shape == x.shape
    dx, dw, db = K().layer_norm_bwd(x, x, w)
    assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all()
    assert K().dropout(x, 0.5, rng).shape == x.shape and K().dropout(x, 0.5, rng, shared="row").shape == x.shape
    zn, xn = K().dropout_add_ln(x, x, w, w, 1e-5, 0.5, rng)
    assert zn.shape == xn.shape == x.shape
    dz, dy, dw, db = K().dropout_add_ln_bwd(x, x, x, w, 1e-5, 0.5, rng)
    assert dz.shape == dy.shape == x.shape and (dw == 0).all() and (db == 0).all()


def test_earlier_widths_keep_their_results():
    """The widths and types that LayerNorm had before run the same kernel at any row count; a misaligned input takes the
    other one, which agrees to rounding."""
    x, (w, b) = acts(14, 130, 128, F32), params(15, 128)
    buf = torch.empty(130 * 128 + 1, device="cuda")
    buf[1:] = x.flatten()
    a, c = K().layer_norm(x, w, b), K().layer_norm(buf[1:].view(130, 128), w, b)
    ref, tol = T.ln(np64(x), np64(w), np64(b)), ln_tol(np64(x), np64(w), np64(b))
    close(a, ref, tol)
    close(c, ref, tol)


# -------------------------------------------------------------------------------------------------- dropout

def dropped_of(t, p, rng, site=0, shared=None, **rows):
    seed, off = (int(v) for v in rng.tolist())
    return T.dropped(tuple(t.shape), p, seed, off, site, shared, **rows).reshape(-1, t.shape[-1])


DEEP = [(2, 17, 5, 77), (3, 40, 31, 128), (2, 3, 4, 1025), (4, 3, 1)]


@pytest.mark.parametrize("shape, shared", [(s, None) for s in [(1,), (7,), (8,), (100003,), (3, 1), (5, 3), (4, 9),
                                                               (33, 64)] + DEEP] +
                         [(s, m) for s in DEEP for m in ("row", "column")])
def test_dropout(shape, shared):
    for k, (tx, ty) in enumerate(TYPES):
        rng = K().dropout_rng(2 ** 40 + 12345 * k, 2 ** 33 + k)
        p = (0.1, 0.25, 0.5, 0.9)[k % 4]
        x = rand(k, *shape, dtype=tx)
        x[x == 0] = 1
        y = K().dropout(x, p, rng, 7 * k, shared, out_dtype=ty)
        assert y.dtype == ty and y.shape == x.shape
        d = dropped_of(x, p, rng, 7 * k, shared).reshape(shape)
        assert np.array_equal(np64(y) == 0, d)  # the same draws, and no kept element lost
        close(y, T.dropout(np64(x), p, d), 2 * U * np.abs(np64(x)) / (1 - p))


def test_dropout_ends_and_special_values():
    x = rand(3, 20, 6, 50, dtype=F16)
    x[::2, ::3, ::7] = float("inf")
    x[1::2, ::3, ::5] = float("nan")
    rng = K().dropout_rng(-5, -1)  # any int64 is a seed
    assert torch.equal(K().dropout(x, 0.0, None), x) or torch.equal(torch.isnan(K().dropout(x, 0.0, None)), torch.isnan(x))
    for shared in (None, "row", "column"):
        assert (K().dropout(x, 1.0, rng, shared=shared) == 0).all()
        y, d = K().dropout(x, 0.5, rng, 65535, shared), dropped_of(x, 0.5, rng, 65535, shared).reshape(x.shape)
        assert (y[torch.tensor(d, device="cuda")] == 0).all()  # infinities and NaNs too
        keep = torch.tensor(~d, device="cuda")
        assert torch.equal(torch.isnan(y[keep]), torch.isnan(x[keep]))
        assert torch.equal(torch.isinf(y[keep]), torch.isinf(x[keep]))
    tiny = 2.0 ** -34  # rounds to no draw at all
    assert torch.equal(K().dropout(x[0].nan_to_num(), tiny, rng), x[0].nan_to_num())


def test_dropout_differs_by_seed_offset_and_site():
    x, r = torch.ones(1000, 64, device="cuda"), K().dropout_rng
    base = K().dropout(x, 0.5, r(1, 2), 3)
    assert torch.equal(base, K().dropout(x, 0.5, r(1, 2), 3))
    for other in (K().dropout(x, 0.5, r(2, 2), 3), K().dropout(x, 0.5, r(1, 3), 3), K().dropout(x, 0.5, r(1, 2), 4)):
        share = (base == other).float().mean().item()
        assert abs(share - 0.5) < 6 * 0.5 / 64000 ** 0.5  # independent fair draws agree in half of the places


# -------------------------------------------------------------------------------------------------- residual update

def check_residual(shape, ty, to, p, shared, seed, affine=True, zero_dz=False):
    D = shape[-1]
    z, y = acts(seed, int(np.prod(shape[:-1])), D, F32).view(shape), rand(seed + 3, *shape, dtype=ty)
    w, b = params(seed + 4, D, affine)
    rng, site = K().dropout_rng(seed * 77 + 2 ** 35, seed), seed % 9
    zn, xn = K().dropout_add_ln(z, y, w, b, 1e-5, p, rng, site, shared, out_dtype=to)
    assert zn.dtype == F32 and xn.dtype == to
    d = dropped_of(z, p, rng, site, shared) if p > 0 else np.zeros((z.numel() // D, D), bool)
    flat = lambda t: np64(t).reshape(-1, D)  # noqa: E731
    close(zn.view(-1, D), flat(z) + T.dropout(flat(y), p, d), 3 * U * np.abs(flat(y)) / (1 - p))
    zr = flat(zn)  # the LayerNorm of what the kernel wrote
    close(xn.view(-1, D), T.ln(zr, np64(w), np64(b)), ln_tol(zr, np64(w), np64(b)))
    dz_new, dln = None if zero_dz else rand(seed + 5, *shape), rand(seed + 6, *shape, dtype=to)
    dz, dy, dw, db = K().dropout_add_ln_bwd(dz_new, dln, zn, w, 1e-5, p, rng, site, shared, y_dtype=ty,
                                            need_weight=affine)
    assert dz.dtype == F32 and dy.dtype == ty
    rz, ry, rw, rb = T.residual_grads(None if zero_dz else flat(dz_new), flat(dln), zr, p, d, np64(w))
    tol = dx_tol(flat(dln), zr, np64(w)) + 2 * U * np.abs(rz)
    close(dz.view(-1, D), rz, tol)
    assert (flat(dy)[d] == 0).all()
    close(dy.view(-1, D), ry, (tol + 2 * U * np.abs(rz)) / (1 - p))
    tw, tb = dw_tol(flat(dln), zr)
    if affine:
        close(dw, rw, tw)
    else:
        assert dw is None
    close(db, rb, tb)


@pytest.mark.parametrize("D", WIDTHS)
def test_residual_widths(D):
    for k, (ty, to) in enumerate(TYPES):
        shared = (None, "row", "column")[(k + D) % 3]
        check_residual((2, 3, ROWS[k], D), ty, to, (0.25, 0.1, 0.0, 0.6)[(k + D // 8) % 4], shared, k + D)


@pytest.mark.parametrize("shape, shared", [((1, 65, 67, 128), "row"), ((1, 65, 67, 128), "column"), ((2, 50, 41, 77), None),
                                           ((3, 31, 33, 64), "column"), ((1, 1, 1300, 384), None),
                                           ((5, 1, 220, 1025), "row"), ((1, 3, 350, 4099), None)])
def test_residual_many_rows(shape, shared):
    check_residual(shape, BF16, BF16, 0.25, shared, 21)
    check_residual(shape, F16, F32, 0.15, shared, 22, affine=False, zero_dz=True)


def test_residual_keeps_the_stream_where_the_update_is_dropped():
    z, y = rand(1, 4, 5, 6, 96), rand(2, 4, 5, 6, 96)
    y[:, :, ::2] = float("nan")
    rng = K().dropout_rng(11)
    for shared in (None, "row", "column"):
        zn, _ = K().dropout_add_ln(z, y, None, None, 1e-5, 0.5, rng, 1, shared)
        d = torch.tensor(dropped_of(z, 0.5, rng, 1, shared).reshape(z.shape).copy(), device="cuda")
        assert torch.equal(zn[d], z[d])
        dz = torch.full_like(z, float("inf"))
        _, dy, _, _ = K().dropout_add_ln_bwd(dz, torch.zeros_like(z), z, None, 1e-5, 0.5, rng, 1, shared,
                                             need_weight=False)
        assert (dy[d] == 0).all() and torch.isinf(dy[~d]).all()


# -------------------------------------------------------------------------------------------------- sizes past 32 bits

def test_offsets_past_32_bits():
    """More than 2^31 elements (fp16): the last rows' values, gradients and draws."""
    D, rows = 2048, 2 ** 20 + 77
    x = torch.empty(rows, D, dtype=F16, device="cuda")
    x.view(-1)[:2 ** 31].view(2 ** 20, D).copy_(acts(1, 2 ** 10, D, F16).repeat(2 ** 10, 1))
    x[2 ** 20:] = acts(2, 77, D, F16)
    w, rng = 1 + rand(3, D, scale=0.1), K().dropout_rng(5, 6)
    tail = x[-80:]
    y = K().dropout(x, 0.5, rng, 9)
    d = dropped_of(x, 0.5, rng, 9, first_row=rows - 80, rows=80)
    close(y[-80:], T.dropout(np64(tail), 0.5, d), 2 * U * np.abs(np64(tail)) * 2)
    assert (np64(y[-80:])[d] == 0).all()
    del y
    dx, dw, db = K().layer_norm_bwd(x, x, w)  # the input as its own gradient
    ref = T.ln_grads(np64(tail), np64(tail), np64(w))[0]
    close(dx[-80:], ref, dx_tol(np64(tail), np64(tail), np64(w)))
    assert torch.isfinite(dw).all() and torch.isfinite(db).all()
    del dx
    close(K().layer_norm(x, w, None, out_dtype=F16)[-80:], T.ln(np64(tail), np64(w)), ln_tol(np64(tail), np64(w), None))


# -------------------------------------------------------------------------------------------------- autograd

def test_autograd_against_float64_and_differences():
    from boltz_mlx_amd import autograd as A

    shape, p = (2, 5, 6, 40), 0.3
    z, y = rand(1, *shape).requires_grad_(), rand(2, *shape).requires_grad_()
    w, b = (t.requires_grad_() for t in params(3, 40))
    rng = K().dropout_rng(17, 4)
    gz, gl = rand(5, *shape), rand(6, *shape)

    def f(z, y, w, b):
        zn, xn = A.dropout_add_ln(z, A.layer_norm(y, w, b), w, b, 1e-5, p, rng, 2, "row", out_dtype=F32)
        return zn, A.dropout(xn, p, rng, 3)

    got = torch.autograd.grad(f(z, y, w, b), (z, y, w, b), (gz, gl))
    leaves = [t.detach().double().cpu().requires_grad_() for t in (z, y, w, b)]
    z6, y6, w6, b6 = leaves
    d1 = torch.tensor(dropped_of(z, p, rng, 2, "row").reshape(shape).copy())
    d2 = torch.tensor(dropped_of(z, p, rng, 3).reshape(shape).copy())
    ln = torch.nn.functional.layer_norm
    zn = z6 + torch.where(d1, 0.0, ln(y6, (40,), w6, b6) / (1 - p))
    out = torch.where(d2, 0.0, ln(zn, (40,), w6, b6) / (1 - p))
    ref = torch.autograd.grad((zn, out), leaves, (gz.double().cpu(), gl.double().cpu()))
    for g, r in zip(got, ref):
        # two LayerNorms in a chain: each errs by some 100u of the largest gradient, times the weights' and scales' growth
        assert (g.double().cpu() - r).abs().max() <= 2000 * U * r.abs().max()
    # along a direction: central differences of the kernels' own forward pass. Its value, a sum of 2400 terms with a mean
    # size near 1, is formed in float64 from fp32 outputs that err by some 20u each: at h = 2^-6 the difference errs by
    # 20u sqrt(2400) / h = 4e-3 and by the third derivative's h^2 / 6 (1e-3 for terms of unit size over 2400 terms).
    v = [rand(7 + i, *t.shape) / t.numel() ** 0.5 for i, t in enumerate((z, y, w, b))]
    h = 2.0 ** -6

    def value(s):
        with torch.no_grad():
            a, c = f(*(t + s * h * dv for t, dv in zip((z, y, w, b), v)))
            return (a.double() * gz).sum() + (c.double() * gl).sum()

    slope = sum((g.double() * dv).sum() for g, dv in zip(got, v))
    assert abs((value(1) - value(-1)) / (2 * h) - slope) < 0.02 + 0.01 * abs(slope)


def test_autograd_needs_and_types():
    from boltz_mlx_amd import autograd as A
    from boltz_mlx_amd.layers.dropout import Dropout
    from boltz_mlx_amd.layers.norm import LayerNorm

    z, y, rng = rand(1, 3, 4, 64), rand(2, 3, 4, 64, dtype=BF16), K().dropout_rng(3)
    ln = LayerNorm(64).cuda()
    with torch.no_grad():
        ln.weight.add_(rand(4, 64, scale=0.1))
    drop = Dropout(0.25, "column", site=5).train()
    zn, xn = drop.add_ln(z.unsqueeze(0), y.unsqueeze(0), ln, rng)
    k_zn, k_xn = K().dropout_add_ln(z[None], y[None], ln.weight, ln.bias, ln.eps, 0.25, rng, 5, "column")
    assert torch.equal(zn, k_zn) and torch.equal(xn, k_xn) and xn.dtype == BF16
    zn.sum().backward()  # only the stream is used: the LayerNorm's parameters have no gradient
    assert ln.weight.grad is None
    yr = y.clone().requires_grad_()
    zn, xn = drop.add_ln(z[None], yr[None], ln, rng)
    (xn.float() ** 2).sum().backward()
    assert yr.grad.dtype == BF16 and ln.weight.grad.shape == (64,)
    zn, _ = drop.add_ln(z[None], yr[None], ln, rng)
    (g,) = torch.autograd.grad(zn, yr, torch.ones_like(zn))
    d = dropped_of(z[None], 0.25, rng, 5, "column").reshape(3, 4, 64)
    assert np.array_equal(np64(g) == 0, d)
    half = ln.weight.detach().half().requires_grad_()
    (gw,) = torch.autograd.grad(A.layer_norm(z, half, None).sum(), half)
    assert gw.dtype == F16
    with pytest.raises(RuntimeError):  # the generator may not change between the passes
        out = drop(yr[None], rng)
        rng[1] += 1
        out.sum().backward()
    drop.eval()
    assert drop(y, rng) is y
    a, c = drop.add_ln(z, y, ln, rng)
    assert torch.equal(a, z + y.float())
    close(ln.with_grad(z), np64(ln(z)), 0 * np64(z))


def test_half_parameters():
    """Parameters that are not fp32 are converted for the call and live until its launch."""
    x, z, y, g = acts(1, 50, 96, F32), acts(2, 50, 96, F32), rand(3, 50, 96), rand(4, 50, 96)
    for dt in (F16, BF16):
        w, b = (t.to(dt) for t in params(5, 96))
        wf, bf = w.float(), b.float()
        assert torch.equal(K().layer_norm(x, w, b), K().layer_norm(x, wf, bf))
        for got, want in ((K().layer_norm_bwd(g, x, w), K().layer_norm_bwd(g, x, wf)),
                          (K().dropout_add_ln(z, y, w, b, 1e-5, 0.0, None), K().dropout_add_ln(z, y, wf, bf, 1e-5, 0.0, None)),
                          (K().dropout_add_ln_bwd(g, y, z, w[::1], 1e-5, 0.0, None),
                           K().dropout_add_ln_bwd(g, y, z, wf, 1e-5, 0.0, None))):
            assert all(torch.equal(p, q) for p, q in zip(got, want))
    strided = torch.stack([wf, wf + 1], 1)[:, 0]
    assert torch.equal(K().layer_norm_bwd(g, x, strided)[0], K().layer_norm_bwd(g, x, wf)[0])


def test_autograd_layouts_and_repeats():
    """Transposed inputs, expanded gradients, a single row, one graph walked twice, and a saved tensor changed in place."""
    from boltz_mlx_amd import autograd as A

    w, b = (t.requires_grad_() for t in params(1, 48))
    base = rand(2, 48, 20).requires_grad_()
    y = A.layer_norm(base.t(), w, b)
    dx, dw, db = torch.autograd.grad(y.sum(), (base, w, b), retain_graph=True)
    check_grads(dx.t(), dw, db, torch.ones(20, 48), base.t(), w)
    again = torch.autograd.grad(y.sum(), (base, w, b))
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))
    with pytest.raises(RuntimeError):  # the graph is gone
        torch.autograd.grad(y.sum(), base)
    row = rand(3, 48).requires_grad_()
    y = A.layer_norm(row, w, b)
    assert y.shape == (48,)
    (dr,) = torch.autograd.grad(y, row, base[:, 0].detach())
    check_grads(dr[None], None, None, base[:, 0][None], row[None], w)
    z = rand(4, 6, 48).requires_grad_()
    zn, xn = A.dropout_add_ln(z, rand(5, 6, 48), w, b)
    zn.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        xn.sum().backward()
    x = rand(6, 30, 48).t().contiguous().t().requires_grad_()
    rng = K().dropout_rng(4)
    (g,) = torch.autograd.grad(A.dropout(x, 0.5, rng).sum(), x)
    d = dropped_of(x, 0.5, rng)
    assert np.array_equal(np64(g), np.where(d, 0.0, 2.0))


def test_a_saved_tensor_changed_by_the_packages_own_kernels():
    """The inference wrappers write through device pointers: a backward pass whose saved tensor one of them has changed
    raises, as after torch's own in-place operations."""
    from boltz_mlx_amd import autograd as A

    class LN:
        weight, bias, eps = torch.ones(128, device="cuda"), torch.zeros(128, device="cuda"), 1e-5

    w, b = (t.requires_grad_() for t in params(1, 128))
    z, y = rand(2, 6, 6, 128), rand(3, 6, 6, 128)
    outs = [A.layer_norm(z, w, b)]
    zn, xn = A.dropout_add_ln(y, z, w, b)
    outs.append(xn)
    K().add_ln(z, y, LN)
    K().transition(rand(4, 36, 128), rand(5, 512, 128), rand(6, 128, 256), zn.detach(), True)
    K().linear(rand(7, 36, 128), rand(8, 128, 128), out=zn.detach().view(36, 128), accumulate=True)
    for out in outs:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), w)


def test_threads():
    """Calls from several host threads at once, each on a stream of its own."""
    import threading

    xs = [acts(20 + k, 3000, 128, F32) for k in range(3)]
    dy, w, rng = rand(1, 3000, 128), 1 + rand(2, 128, scale=0.1), K().dropout_rng(3)
    ref = [K().layer_norm_bwd(dy, x, w) + (K().dropout(x, 0.3, rng, k),) for k, x in enumerate(xs)]
    torch.cuda.synchronize()
    got = [None] * 3

    def work(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got[k] = K().layer_norm_bwd(dy, xs[k], w) + (K().dropout(xs[k], 0.3, rng, k),)
        s.synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, r in zip(got, ref):
        assert all(torch.equal(a, c) for a, c in zip(g, r))


def test_gradients_of_gradients_are_refused():
    from boltz_mlx_amd import autograd as A

    x, w = rand(1, 4, 32).requires_grad_(), rand(2, 32).requires_grad_()
    for out in (A.layer_norm(x, w), A.dropout(x, 0.5, K().dropout_rng(1)), A.dropout_add_ln(x, x, w)[1]):
        with pytest.raises(RuntimeError, match="gradients of gradients"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_entry_points_refusals_are_the_packages_error(monkeypatch):
    """What a C entry point refuses raises BzpfError, through the torch binding as everywhere else."""
    from boltz_mlx_amd import _lib
    from boltz_mlx_amd import autograd as A

    x, rng = rand(1, 6, 32, dtype=F16), K().dropout_rng(1)
    calls = [lambda: K().layer_norm(x, None, None, out_dtype=BF16), lambda: K().layer_norm_bwd(x, x.bfloat16(), None),
             lambda: K().dropout(x, 0.5, rng, out_dtype=BF16),
             lambda: K().dropout_add_ln(x.float(), x, None, None, 1e-5, 0.5, rng, out_dtype=BF16),
             lambda: K().dropout_add_ln_bwd(None, x, x.float(), None, 1e-5, 0.5, rng, y_dtype=BF16),
             lambda: A.layer_norm(x.requires_grad_(), out_dtype=BF16)]
    for call in calls:
        with pytest.raises(_lib.BzpfError, match="failed .-1.: bzpf_.*bad dtype"):
            call()
    monkeypatch.setattr(_lib, "_train", None)
    monkeypatch.setattr(_lib, "_no_train", True)
    with pytest.raises(_lib.BzpfError, match="bad dtype"):
        calls[0]()


def test_launch_times_are_recorded():
    x, w, rng = rand(1, 40, 64), rand(2, 64), K().dropout_rng(1)
    K().start_timing()
    K().layer_norm(x, w, w)
    K().layer_norm_bwd(x, x, w)
    K().dropout(x, 0.5, rng)
    zn, _ = K().dropout_add_ln(x, x, w, w, 1e-5, 0.5, rng)
    K().dropout_add_ln_bwd(x, x, zn, w, 1e-5, 0.5, rng)
    times = K().stop_timing()
    assert set(times) == {"bzpf_layernorm", "bzpf_layernorm_bwd", "bzpf_dropout", "bzpf_dropout_add_ln",
                          "bzpf_dropout_add_ln_bwd"} and all(len(v) == 1 for v in times.values())


# -------------------------------------------------------------------------------------------------- streams and graphs

def test_side_stream_and_two_calls_at_once():
    x, dy, w = acts(1, 5000, 128, F32), rand(2, 5000, 128, dtype=F16), 1 + rand(3, 128, scale=0.1)
    x2 = acts(9, 5000, 128, F32)
    ref, ref2 = K().layer_norm_bwd(dy, x, w), K().layer_norm_bwd(dy, x2, w)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            a = K().layer_norm_bwd(dy, x, w)
        with torch.cuda.stream(s2):
            b = K().layer_norm_bwd(dy, x2, w)
        outs.append((a, b))
    torch.cuda.synchronize()
    for a, b in outs:
        assert all(torch.equal(p, q) for p, q in zip(a + b, ref + ref2))


def test_captured_step_replays_with_new_inputs_and_draws():
    """A whole update (forward and backward, autograd and kernels) in one graph: every replay, with new inputs and another
    offset written between, gives what the eager calls give."""
    from boltz_mlx_amd import autograd as A

    shape, p = (1, 37, 41, 128), 0.25
    z, y = rand(1, *shape), rand(2, *shape, dtype=F16)
    w, b = params(3, 128)
    rng, gz, gl = K().dropout_rng(8, 0), rand(4, *shape), rand(5, *shape, dtype=F16)

    def step(leaves):
        lz, ly, lw, lb = leaves
        zn, xn = A.dropout_add_ln(lz, ly, lw, lb, 1e-5, p, rng, 1, "row")
        t = A.dropout(A.layer_norm(zn, lw, lb, out_dtype=F16), p, rng, 2)
        return (zn.detach(), xn.detach(), t.detach()) + torch.autograd.grad((zn, xn, t), leaves, (gz, gl, gl))

    def fresh():
        return [t.detach().requires_grad_() for t in (z, y, w, b)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    leaves = fresh()
    with torch.cuda.graph(graph):
        outs = step(leaves)
    seen = []
    for k in range(4):
        z.copy_(rand(10 + k, *shape))
        y.copy_(rand(20 + k, *shape, dtype=F16))
        rng[1] = k
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = step(fresh())
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        seen.append(got[2] == 0)
    assert not torch.equal(seen[0], seen[1])


def test_two_graphs_keep_their_own_workspaces():
    x, dy, w = acts(1, 9000, 384, F32), rand(2, 9000, 384), 1 + rand(3, 384, scale=0.1)
    xs = [acts(4 + k, 9000, 384, F32) for k in range(2)]
    refs = [K().layer_norm_bwd(dy, t, w) for t in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K().layer_norm_bwd(dy, t, w))
        graphs.append(g)
    for order in ((0, 1), (1, 0), (0, 1)):
        for k in order:
            graphs[k].replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, refs):
            assert all(torch.equal(a, c) for a, c in zip(o, r))
        (x * 2).sum()
        torch.cuda.synchronize()


# -------------------------------------------------------------------------------------------------- all together

def test_a_block_of_updates_trains():
    """Three pair updates in a chain (dropout per row, per column and per element, each with the next LayerNorm), as a
    layer's training step has them: values and every parameter's gradient against float64 autograd."""
    from boltz_mlx_amd.layers.dropout import Dropout
    from boltz_mlx_amd.layers.norm import LayerNorm

    shape, D = (2, 13, 13, 128), 128
    drops = [Dropout(0.25, "row", 0), Dropout(0.25, "column", 1), Dropout(0.1, None, 2)]
    lns = [LayerNorm(D).cuda() for _ in range(4)]
    mats = [rand(30 + k, D, D, scale=D ** -0.5).requires_grad_() for k in range(3)]
    for k, ln in enumerate(lns):
        with torch.no_grad():
            ln.weight.add_(rand(40 + k, D, scale=0.1))
            ln.bias.add_(rand(50 + k, D, scale=0.1))
    z0, rng, gz, gl = rand(1, *shape), K().dropout_rng(99, 3), rand(2, *shape), rand(3, *shape)
    z, xn = z0, lns[0].with_grad(z0)
    for drop, mat, ln in zip(drops, mats, lns[1:]):
        z, xn = drop.add_ln(z, xn @ mat, ln, rng)
    leaves = mats + [t for ln in lns for t in (ln.weight, ln.bias)]
    got = torch.autograd.grad((z, xn), leaves, (gz, gl))
    ref_leaves = [t.detach().double().cpu().requires_grad_() for t in leaves]
    m6, p6 = ref_leaves[:3], ref_leaves[3:]
    f = torch.nn.functional.layer_norm
    r = z0.double().cpu()
    x6 = f(r, (D,), p6[0], p6[1])
    for k, drop in enumerate(drops):
        d = torch.tensor(dropped_of(z0, drop.p, rng, drop.site, drop.shared).reshape(shape).copy())
        r = r + torch.where(d, 0.0, (x6 @ m6[k]) / (1 - drop.p))
        x6 = f(r, (D,), p6[2 * k + 2], p6[2 * k + 3])
    # fp32 throughout; the matrix products err by sqrt(128) u of their terms, three updates deep: 1e-5 of the largest value
    assert (z.double().cpu() - r).abs().max() <= 1e-5 * r.abs().max()
    assert (xn.double().cpu() - x6).abs().max() <= 1e-5 * x6.abs().max()
    for g, w in zip(got, torch.autograd.grad((r, x6), ref_leaves, (gz.double().cpu(), gl.double().cpu()))):
        assert (g.double().cpu() - w).abs().max() <= 3e-5 * w.abs().max()


# -------------------------------------------------------------------------------------------------- more of dropout's ends

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_no_dropout_keeps_every_bit(dtype):
    x = rand(3, 20, 6, 51, dtype=dtype)
    x[::2, ::3, ::7], x[1::2, ::3, ::5], x[0, 0, :2] = float("inf"), float("nan"), -0.0
    bits = torch.int32 if dtype == F32 else torch.int16
    for p in (0.0, 2.0 ** -34):  # the second rounds to no draw at all
        for shared in (None, "row", "column"):
            assert torch.equal(K().dropout(x, p, K().dropout_rng(1), 2, shared).view(bits), x.view(bits))


# -------------------------------------------------------------------------------------------------- more sizes past 32 bits

BIG = (1025, 1024, 2048)  # 2^31 + 2^21 elements; more rows than a forward launch has workgroups, which turn once more


def big(seed, dtype):
    """Rows of a tensor of size BIG: 1024 of them, repeated, and others in the last 80."""
    rows, D = BIG[0] * BIG[1], BIG[2]
    x = acts(seed, 1024, D, dtype).repeat(BIG[0], 1)
    x[rows - 80:] = acts(seed + 5, 80, D, dtype)
    return x


def check_param_sums(dw, db, dy, x):
    """dw and db against sums in float64 on the device, a slice of rows at a time, with dw_tol's tolerance."""
    depth = len(x) // 256 + 128
    rw, rb, tw, tb = (torch.zeros(x.shape[1], dtype=torch.float64, device="cuda") for _ in range(4))
    for i in range(0, len(x), 2 ** 15):
        xs, g = x[i:i + 2 ** 15].double(), dy[i:i + 2 ** 15].double()
        c = xs - xs.mean(-1, keepdim=True)
        rstd = 1 / ((c * c).mean(-1, keepdim=True) + 1e-5).sqrt()
        xh, E = c * rstd, U * (16 * xs.abs().amax(-1, keepdim=True) * rstd + 14)
        rw += (g * xh).sum(0)
        rb += g.sum(0)
        tw += (g.abs() * (1 + xh.abs()) * E).sum(0) + depth * U * (g * xh).abs().sum(0)
        tb += depth * U * g.abs().sum(0)
    close(dw, np64(rw), np64(tw))
    close(db, np64(rb), np64(tb))


def test_layer_norm_gradients_past_32_bits():
    x, dy, w = big(1, F16), big(11, F16), params(2, BIG[2])[0]
    dx, dw, db = K().layer_norm_bwd(dy, x, w)
    tail = [np64(t[-1200:]) for t in (dy, x)]
    close(dx[-1200:], T.ln_grads(*tail, np64(w))[0], dx_tol(*tail, np64(w)))
    check_param_sums(dw, db, dy, x)


@pytest.mark.parametrize("shared", [None, "row", "column"])
def test_residual_update_past_32_bits(shared):
    """The residual update and its backward pass: the last rows' values, draws and gradients, and the sums over all rows."""
    rows, D = BIG[0] * BIG[1], BIG[2]
    z, y, (w, b), rng, p = big(1, F32), big(21, F16), params(2, D), K().dropout_rng(2 ** 33 + 7, 5), 0.25
    zn, xn = K().dropout_add_ln(z.view(BIG), y.view(BIG), w, b, 1e-5, p, rng, 6, shared)
    zn, xn = zn.view(rows, D), xn.view(rows, D)
    n = 1200
    d = T.dropped(BIG, p, 2 ** 33 + 7, 5, 6, shared, first_row=rows - n, rows=n)
    zt, yt, znt, xnt = (np64(t[-n:]) for t in (z, y, zn, xn))
    close(zn[-n:], zt + T.dropout(yt, p, d), 3 * U * np.abs(yt) / (1 - p))
    close(xn[-n:], T.ln(znt, np64(w), np64(b)), ln_tol(znt, np64(w), np64(b)))
    dz, dy, dw, db = K().dropout_add_ln_bwd(z.view(BIG), xn.view(BIG), zn.view(BIG), w, 1e-5, p, rng, 6, shared)
    rz, ry, _, _ = T.residual_grads(zt, xnt, znt, p, d, np64(w))
    tol = dx_tol(xnt, znt, np64(w)) + 2 * U * np.abs(rz)
    close(dz.view(rows, D)[-n:], rz, tol)
    got = dy.view(rows, D)[-n:]
    assert (np64(got)[d] == 0).all()
    close(got, ry, (tol + 2 * U * np.abs(rz)) / (1 - p))
    check_param_sums(dw, db, xn, zn)


@pytest.mark.parametrize("shared", [None, "row", "column"])
def test_dropout_of_odd_rows_past_32_bits(shared):
    shape, rng, p = (1026, 1025, 2047), K().dropout_rng(9, 2 ** 40), 0.5
    rows, D = shape[0] * shape[1], shape[2]
    x = acts(3, 1025, D, F16).repeat(shape[0], 1)
    x[x == 0] = 1
    y = K().dropout(x.view(shape), p, rng, 8, shared).view(rows, D)
    n = 1200
    d = T.dropped(shape, p, 9, 2 ** 40, 8, shared, first_row=rows - n, rows=n)
    assert np.array_equal(np64(y[-n:]) == 0, d)
    close(y[-n:], T.dropout(np64(x[-n:]), p, d), 2 * U * np.abs(np64(x[-n:])) / (1 - p))


# -------------------------------------------------------------------------------------------------- LayerNorm's two kernels

@pytest.mark.parametrize("D", [64, 128, 384, 1024])
def test_layer_norm_parameters_at_any_element(D):
    """A weight and a bias that are slices at odd offsets, with x and y at whole boundaries: the bits of aligned ones."""
    w, b = params(3, D)
    for off in (1, 2, 3):
        ws, bs = torch.zeros(D + 5, device="cuda"), torch.zeros(D + 5, device="cuda")
        ws[off:off + D], bs[5 - off:5 - off + D] = w, b
        wo, bo = ws[off:off + D], bs[5 - off:5 - off + D]
        for tx, ty in ((F32, F32), (F32, F16), (F16, F16), (BF16, BF16)):
            x = acts(D, 37, D, tx)
            assert torch.equal(K().layer_norm(x, wo, bo, out_dtype=ty), K().layer_norm(x, w, b, out_dtype=ty))
    z, y = rand(1, 9, 9, 128), rand(2, 9, 9, 128)

    class LN:
        eps = 1e-5

    def add_ln(w, b):
        LN.weight, LN.bias = w, b
        return K().add_ln(z.clone(), y, LN, out_dtype=F32)

    w, b = params(5, 128)
    ws, bs = torch.cat([w[:1], w]), torch.cat([b[:3], b])
    assert torch.equal(add_ln(ws[1:], bs[3:]), add_ln(w, b))


# The widths and types that LayerNorm served before it took every width: SHA-256 of the outputs (fp32 and fp16 in, fp32 and
# fp16 out, in that order) of the library as it was then, for the inputs below.
EARLIER = {
    64: "eaba80f696e4beb0",
    128: "6511081e6816421d",
    192: "f6c8ad3a965efa8e",
    256: "93d555ca95c6be38",
    320: "c882499ddb6a75fe",
    384: "6fae8af8104e92a7",
    512: "cb0af66ac15ca896",
    768: "d27715d0c777c274",
    1024: "6d5eb8b9f369ed98",
}


def earlier_digest(layer_norm, D):
    """Inputs from integers alone, so that they are the same anywhere."""
    import hashlib

    r, c = np.arange(131, dtype=np.int64)[:, None], np.arange(D, dtype=np.int64)
    x = ((r * D + c) * 2654435761 % 2 ** 32) / 2.0 ** 29 - 4 + r % 7
    w, b = 1 + (c * 40503 % 65536 - 32768) / 2.0 ** 18, (c * 30011 % 65536 - 32768) / 2.0 ** 16
    x, w, b = (torch.tensor(v, dtype=F32, device="cuda") for v in (x, w, b))
    digest = hashlib.sha256()
    for tx in (F32, F16):
        for ty in (F32, F16):
            for args in ((w, b), (None, None)):
                digest.update(layer_norm(x.to(tx), *args, 1e-5, out_dtype=ty).cpu().numpy().tobytes())
    return digest.hexdigest()[:16]


@pytest.mark.parametrize("D", EARLIER)
def test_earlier_widths_keep_their_bits(D):
    assert earlier_digest(K().layer_norm, D) == EARLIER[D]


def test_layer_norm_without_the_binding(monkeypatch):
    """Where the torch binding is not built, LayerNorm goes through the C ABI: the same bits, on the caller's stream."""
    from boltz_mlx_amd import _lib

    cases = []
    for k, (tx, ty) in enumerate(TYPES):
        for D in (77, 128, 384, 2055):
            x, (w, b) = acts(k, 33, D, tx), params(D, D)
            cases.append((x, w, b, ty))
            cases.append((x.t().contiguous().t(), w.half(), None, ty))
    want = [K().layer_norm(x, w, b, 1e-5, out_dtype=ty) for x, w, b, ty in cases]
    torch.cuda.synchronize()
    assert _lib._train is not None
    monkeypatch.setattr(_lib, "_train", None)
    monkeypatch.setattr(_lib, "_no_train", True)
    with torch.cuda.stream(torch.cuda.Stream()):
        got = [K().layer_norm(x, w, b, 1e-5, out_dtype=ty) for x, w, b, ty in cases]
        assert K().layer_norm(cases[0][0][:0], None, None).shape == (0, 77)
    torch.cuda.synchronize()
    for a, c, (_, _, _, ty) in zip(got, want, cases):
        assert a.dtype == ty and torch.equal(a, c)


def test_layer_norm_past_one_launch():
    """More rows than the kernel of the earlier widths can launch threads for (16 a row, 2^32 in all)."""
    rows, D = 2 ** 28 + 5, 64
    x, (w, b) = torch.zeros(rows, D, dtype=F16, device="cuda"), params(3, D)
    x[:1000], x[-1000:] = acts(1, 1000, D, F16), acts(2, 1000, D, F16)
    y = K().layer_norm(x, w, b, out_dtype=F16)
    for part in (slice(0, 1000), slice(rows - 1000, rows)):
        close(y[part], T.ln(np64(x[part]), np64(w), np64(b)), ln_tol(np64(x[part]), np64(w), np64(b)))
    assert torch.equal(y[1000:-1000:4099], b.half().expand(y[1000:-1000:4099].shape))


# -------------------------------------------------------------------------------------------------- in place, from C

@pytest.mark.parametrize("D", [9, 77, 128, 1021, 2055, 8191])
def test_backward_passes_in_place(D):
    """An output of a backward pass that is one of its inputs: the bits of the call with buffers of their own."""
    from boltz_mlx_amd import _lib

    rows, st = 700, torch.cuda.current_stream().cuda_stream
    x, dy, dz_new, w = acts(1, rows, D, F32), rand(2, rows, D), rand(3, rows, D), 1 + rand(4, D, scale=0.1)
    n = _lib.load().bzpf_layernorm_bwd_ws(rows, D)
    ws, dw, db = torch.empty(n // 4 + 1, device="cuda"), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    tail = (dw.data_ptr(), db.data_ptr(), ws.data_ptr(), n, rows, D, st)
    for k in range(2):
        a, g = x.clone(), dy.clone()
        out = (a, g)[k]
        _lib.call("bzpf_layernorm_bwd", g.data_ptr(), 0, a.data_ptr(), 0, w.data_ptr(), 1e-5, out.data_ptr(), *tail)
        assert all(torch.equal(p, q) for p, q in zip((out, dw, db), K().layer_norm_bwd(dy, x, w)))
    rng = K().dropout_rng(7)
    want = K().dropout_add_ln_bwd(dz_new, dy, x, w, 1e-5, 0.3, rng, 1)
    for i, j in ((0, 1), (1, 2), (2, 0)):
        t = [v.clone() for v in (dz_new, dy, x)]
        _lib.call("bzpf_dropout_add_ln_bwd", t[0].data_ptr(), t[1].data_ptr(), 0, t[2].data_ptr(), w.data_ptr(), 1e-5, 0.3,
                  rng.data_ptr(), 1, 0, 1, 1, t[i].data_ptr(), t[j].data_ptr(), 0, *tail)
        assert all(torch.equal(p, q) for p, q in zip((t[i], t[j], dw, db), want))
