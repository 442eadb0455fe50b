"""The sequence attention's gradients over long axes: a bias of more than 2^31 elements with gradients that are not zero, its own
and shared by samples; few queries against a long axis and the reverse. Tolerances as test_gpu_attention.py derives them."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_attention import BF16, F16, F32, STEP, U, K, check, close, inputs, np64, rand  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mult", [1, 2])
def test_attention_gradients_past_32_bits(mult):
    """Each row has two keys that take its weight (others have less than e^-50 of it, 2e-18 in all), so that its gradients are those
    of two keys; every key belongs to two rows. All rows' gradients against float64, those of the bias at the rows' keys and, at the last
    rows, everywhere."""
    H, C, N = 2, 8, 32771
    S, h, tiny = mult, STEP[F16], 2.0 ** -25
    q, k, v = (rand(i, S, N, H * C, dtype=F16) for i in range(3))
    dout = rand(4, S, N, H * C, dtype=F16)
    row = torch.arange(N, device="cuda")
    at = torch.stack([N - 1 - row, (N - 1 - row + N // 2) % N])  # [2, N]
    bias = torch.zeros(H, N, N, device="cuda", dtype=F16)
    assert bias.numel() > 2 ** 31
    bias[:, row, at[0]] = 64.0
    bias[:, row, at[1]] = 64.0
    o, stats = K().attention(q, k, v, H, bias=bias[None], multiplicity=mult)
    dq, dk, dv, _, db = K().attention_bwd(dout, q, k, v, H, o, stats, bias=bias[None], multiplicity=mult)

    hd = lambda t: t.double().view(S, N, H, C).transpose(1, 2)  # noqa: E731
    q, k, v, d, o = hd(q), hd(k), hd(v), hd(dout), hd(o)
    k2, v2 = k[:, :, at], v[:, :, at]  # [S, H, 2, N, C]
    x = (q[:, :, None] * k2).sum(-1) / C ** 0.5
    ax = (q[:, :, None] * k2).abs().sum(-1) / C ** 0.5 + 64
    p = x.softmax(2)
    dp = (d[:, :, None] * v2).sum(-1)
    delta = (p * dp).sum(2, keepdim=True)
    ds = p * (dp - delta)
    E = 2 * (U * (C + 6) * ax).amax(2, keepdim=True) + U * 208
    Ep = 2 * E + U * (N + 16)
    edp = U * 2 * C * (d[:, :, None] * v2).abs().sum(-1)
    dd = (p * (Ep * dp.abs() + edp)).sum(2, keepdim=True) + U * N * (p * dp.abs()).sum(2, keepdim=True)
    eds = p * (dp.abs() + delta.abs()) * (Ep + 4 * U) + p * (edp + dd)
    near = lambda got, ref, tol: close(got, ref.cpu().numpy(), tol.cpu().numpy(), F16)  # noqa: E731
    want = (p[..., None] * v2).sum(2)
    t_out = (p[..., None] * v2.abs()).sum(2) * (E[:, :, 0, :, None] + h + U * N) + want.abs() * (E[:, :, 0, :, None] + U * N + 8 * U)
    near(o, want, t_out)
    rest = 1e-17  # the other keys' part, of sums of unit-sized products
    mine = db[0][:, row, at].double()  # [H, 2, N]
    near(mine, ds.sum(0), (eds + 4 * U * mult * ds.abs()).sum(0) + rest)
    raw = (d.abs() * (t_out + h * (want.abs() + t_out) + tiny)).sum(-1)[:, :, None]
    scale = C ** -0.5
    pk = (p[..., None] * k2).sum(2).abs()
    low = tiny * C ** 0.5
    taken = ((h * (ds.abs() + p * raw) + low).sum(2))[..., None] * pk * (1 + h)
    tq = scale * (((eds + h * (ds.abs() + 2 * p * raw) + low * (1 + raw))[..., None] * k2.abs()).sum(2) +
                  U * N * ((ds.abs() + p * raw)[..., None] * k2.abs()).sum(2) + taken)
    near(hd(dq), scale * (ds[..., None] * k2).sum(2), tq)

    def keys(t):  # [S, H, 2, N, C] of rows: the sums over the rows of each key
        out = torch.zeros(S, H, N, C, dtype=torch.float64, device="cuda")
        for i in range(2):
            out.index_add_(2, at[i], t[:, :, i])
        return out

    # the other rows' ds and p round to 0, or are below 2^-24 in fp16: N of them at most half of that each
    q2, d2 = q[:, :, None].expand(k2.shape), d[:, :, None].expand(k2.shape)
    near(hd(dk), scale * keys(ds[..., None] * q2), scale * keys((eds + h * ds.abs() + tiny + U * N * ds.abs())[..., None] * q2.abs()) + rest)
    near(hd(dv), keys(p[..., None] * d2), keys((p * (Ep + h + U * N) + tiny)[..., None] * d2.abs()) + rest)
    last = db[0][:, -40:].double()
    last[:, torch.arange(40, device="cuda"), at[0, -40:]] = 0
    last[:, torch.arange(40, device="cuda"), at[1, -40:]] = 0
    assert float(last.abs().max()) < 1e-15
    assert float(ds.abs().amax(2).median()) > 0.1  # there is something to compare


@pytest.mark.parametrize("S, mult, H, C, N, M", [(2, 2, 3, 64, 1, 5000), (1, 1, 1, 40, 2, 30011), (1, 1, 5, 72, 2, 4096), (2, 1, 2, 32, 8, 9001),
                                                 (1, 1, 2, 24, 9001, 1), (2, 1, 2, 48, 7000, 3), (1, 1, 1, 64, 20011, 8)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_gradients_of_long_axes(S, mult, H, C, N, M, dtype):
    """Few queries against many keys, and few keys that many queries see."""
    for n, (bias, gate, mask) in enumerate([("same", True, "tail"), (None, False, None), ("same", False, "holes")]):
        check(inputs(10 * n + C, S, mult, H, C, N, M, dtype, bias, gate, mask), H)


def test_attention_refuses_too_many_rows_by_name():
    """More than 2^22 queries or keys: the package's own error from both directions."""
    from boltz_mlx_amd._lib import BzpfError

    many, one = torch.zeros(2 ** 22 + 1, 8, device="cuda", dtype=F16), torch.zeros(1, 8, device="cuda", dtype=F16)
    for q, k in ((many, one), (one, many)):
        with pytest.raises(BzpfError, match="1 to 2\\^22 queries and keys"):
            K().attention(q, k, k, 1)
        with pytest.raises(BzpfError, match="1 to 2\\^22 queries and keys"):
            K().attention_bwd(q, q, k, k, 1, q, torch.zeros(1, len(q), 2, device="cuda"))
