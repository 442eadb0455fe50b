"""The sequence attention's gradients in fp16 where ds = p (dp - delta) is far past the type's largest number and the gradients
formed from it are not: few keys, so that p is not small, and queries and keys that are. Tolerances are those of
test_gpu_attention.py and what the scaling of ds before its rounding loses: a key's (for dq: a row's) ds are scaled by 2^-12 or 2^-24
only where the largest of them is 2^16 or more before the last step of 2^12, so at least 2^4 after it; an error of fp16's 2^-25 below
2^-14 is then at most 2^-29 of the largest, and 2^-28 with the sums of them that dq takes off."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_attention import F16, F32, call, call_bwd, close, heads, inputs, np64, rand, rows, tolerances  # noqa: E402

pytestmark = pytest.mark.gpu


def aligned(seed, S, mult, H, C, N, M, bias, gate, small, size, big):
    """Inputs whose dp is C * big * size up to their gates, of alternating signs: every other key and query has the other sign,
    so that sums over them (out, dv, delta) stay in range."""
    a = inputs(seed, S, mult, H, C, N, M, F16, bias, gate, None)
    sign = torch.sign(rand(seed + 1, H * C))
    turn = lambda n: 1.0 - 2.0 * (torch.arange(n, device="cuda") % 2)[:, None]  # noqa: E731
    a["q"], a["k"] = (rand(seed + i, S, n, H * C, scale=small, dtype=F16) for i, n in ((2, N), (3, M)))
    a["v"] = (sign * turn(M) * size * (1 + rand(seed + 4, S, M, H * C, scale=0.1))).to(F16)
    return a, (sign * turn(N) * big * (1 + rand(seed + 5, S, N, H * C, scale=0.1))).to(F16)


def check_large(a, dout, H, need_bias=True):
    o, stats = call(a, H)
    want, _, tol, grads = tolerances(a, H, F16, dout)
    C, mult = dout.shape[-1] // H, a["mult"]
    q, k, v, g, bias = (np64(a[n]) for n in ("q", "k", "v", "g", "bias"))
    d = np64(dout) if g is None else np64(dout) / (1 + np.exp(-g))
    x = heads(q, H) @ heads(k, H).swapaxes(-1, -2) / np.sqrt(C) + (0 if bias is None else np.repeat(bias, mult, 0))
    p = np.exp(x - x.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    dp = heads(d, H) @ heads(v, H).swapaxes(-1, -2)
    ds = np.abs(p * (dp - (p * dp).sum(-1, keepdims=True)))
    more = 2.0 ** -28 / np.sqrt(C)
    tol["k"] = tol["k"] + more * rows(ds.max(-2)[..., None] * heads(np.abs(q), H).sum(-2, keepdims=True))
    tol["q"] = tol["q"] + more * rows(ds.max(-1)[..., None] * heads(np.abs(k), H).sum(-2, keepdims=True))
    got = call_bwd(dout, a, H, o, stats, need_bias=need_bias)
    again = call_bwd(dout, a, H, o, stats, need_bias=need_bias)
    close(o, want, tol["out"])
    for n, ref in grads.items():
        if n == "bias" and not need_bias:
            continue
        # what passes the type's largest number is infinite (a pair bias's gradient is ds itself; a few of the others' elements)
        fits, over = np.abs(ref) < 65000, np.abs(ref) > 66000
        assert n == "bias" or over.mean() < 0.01
        close(got[n][torch.from_numpy(fits).cuda()], ref[fits], np.broadcast_to(tol[n], ref.shape)[fits])
        assert np.array_equal(np64(got[n])[over], np.sign(ref[over]) * np.inf)
        assert torch.equal(got[n], again[n])
    return ds.max()


# S, mult, H, C, N, M: one query, both forms of the tiles (and heads of more channels than the split form takes), a shared bias
LARGE = [(1, 1, 1, 64, 1, 2), (1, 1, 2, 64, 8, 2), (2, 1, 3, 64, 200, 3), (2, 2, 2, 32, 70, 5), (1, 1, 2, 48, 40, 70), (20, 1, 16, 64, 8, 4),
         (20, 4, 16, 40, 10, 3), (3, 1, 2, 128, 34, 4), (1, 1, 1, 64, 260, 130)]


@pytest.mark.parametrize("S, mult, H, C, N, M", LARGE)
@pytest.mark.parametrize("bias, gate, need_bias", [(None, False, True), (None, True, True), ("same", True, False), ("same", False, True)])
def test_attention_ds_past_fp16(S, mult, H, C, N, M, bias, gate, need_bias):
    """ds up to 16 times fp16's largest number for three keys or fewer, of some keys and rows alone for more."""
    a, dout = aligned(S + M, S, mult, H, C, N, M, bias, gate, 0.02 if N < 200 else 0.005, 16.0, 2000.0 * (64 / C))
    top = check_large(a, dout, H, need_bias)
    assert M > 5 or top > 65504


@pytest.mark.parametrize("S, H, N", [(1, 2, 8), (20, 16, 8), (1, 1, 70)])
@pytest.mark.parametrize("M", [2, 4])
def test_attention_ds_far_past_fp16(S, H, N, M):
    """ds up to 2^36, about the most that finite operands give, and queries and keys below 2^-17."""
    a, dout = aligned(7, S, 1, H, 64, N, M, None, False, 2.0 ** (-20 if N < 70 else -22), 4e4, 4e4)
    assert check_large(a, dout, H) > 2.0 ** 33


def test_attention_ds_large_in_some_keys_and_rows():
    """Queries that see two keys alone by their biases, with large gradients; others with ordinary ones: the keys and rows of the
    latter keep their accuracy beside those."""
    S, H, C, N, M = 1, 2, 64, 64, 64
    a, dout = aligned(3, S, 1, H, C, N, M, "same", False, 0.02, 16.0, 1.0)
    a["bias"].fill_(-float("inf"))
    a["bias"][:, :, :32, :2] = 0.0
    a["bias"][:, :, 32:, 2:] = rand(9, S, H, 32, M - 2, dtype=F16)
    dout[:, :32] *= 1000
    dout[:, 32:] *= 2.0 ** -6
    o, stats = call(a, H)
    _, _, tol, grads = tolerances(a, H, F16, dout)
    got = call_bwd(dout, a, H, o, stats)
    # the first keys and rows have their own scale, 2^-12: 2^-28 of the largest ds (below 2^20) times 64 rows of |q| or |k| < 0.1
    large = 2.0 ** -28 * 2 ** 20 * 64 * 0.1 / 8
    for n, cut in (("k", 2), ("q", 32)):
        close(got[n][:, :cut], grads[n][:, :cut], tol[n][:, :cut] + large)
        close(got[n][:, cut:], grads[n][:, cut:], tol[n][:, cut:])


def test_attention_gradients_out_of_range_are_infinite():
    """dk and dq that pass fp16's largest number themselves are infinite with their signs, not NaN, and others unharmed; gradients
    that are not finite on their way in end in finite time."""
    a, dout = aligned(5, 1, 1, 1, 64, 8, 2, None, False, 1.0, 16.0, 4000.0)
    o, stats = call(a, 1)
    d = call_bwd(dout, a, 1, o, stats)
    _, _, _, grads = tolerances(a, 1, F16, dout)
    for n in ("q", "k"):
        over = np.abs(grads[n]) > 66000
        assert over.any() and np.array_equal(np64(d[n])[over], np.sign(grads[n][over]) * np.inf)
        assert np.isfinite(np64(d[n])[np.abs(grads[n]) < 65000]).all()
    dout[0, 3, 5] = float("inf")
    d = call_bwd(dout, a, 1, o, stats)
    assert not torch.isfinite(d["q"][0, 3]).any() and not torch.isfinite(d["k"]).any()


@pytest.mark.parametrize("N, M", [(8, 2), (70, 3), (40, 200)])
def test_attention_small_gradients_of_few_keys(N, M):
    """The other end: gradients of 2^-10, whose ds are below fp16's 2^-14."""
    a = inputs(6, 1, 1, 2, 64, N, M, F16, None, True, None)
    dout = rand(8, 1, N, 128, scale=2.0 ** -10, dtype=F16)
    o, stats = call(a, 2)
    _, _, tol, grads = tolerances(a, 2, F16, dout)
    d = call_bwd(dout, a, 2, o, stats)
    for n, x in grads.items():
        close(d[n], x, tol[n])


@pytest.mark.parametrize("N, M, C", [(4000, 40, 8), (9000, 3, 24), (2500, 300, 16)])
def test_attention_small_gradients_of_many_queries(N, M, C):
    """dk as a sum of many ds far below 2^-14, each off by fp16's 2^-25 after its scaling by 2^k <= sqrt(N / C): 2^-25 / 2^k. Errors
    of independent roundings within bounds b have squares of at most the sum of b^2 (b^2 / 3 where they are even)."""
    H = 2
    a = inputs(6, 1, 1, H, C, N, M, F16, "same", False, None)
    dout = rand(8, 1, N, H * C, scale=2.0 ** -9 / N ** 0.5 * M ** 0.5, dtype=F16)
    o, stats = call(a, H)
    d = call_bwd(dout, a, H, o, stats)
    _, _, _, grads = tolerances(a, H, F16, dout)
    q, k, v, bias = (np64(a[n]) for n in ("q", "k", "v", "bias"))
    x = heads(q, H) @ heads(k, H).swapaxes(-1, -2) / np.sqrt(C) + bias
    p = np.exp(x - x.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    dp = heads(np64(dout), H) @ heads(v, H).swapaxes(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdims=True))
    assert np.median(np.abs(ds)) < 2.0 ** -14
    h, tiny = 2.0 ** -11, 2.0 ** -25
    b = (h * np.abs(ds) + tiny / 2.0 ** (int(np.log2(N // C)) // 2)) ** 2
    bound = rows(b.swapaxes(-1, -2) @ heads(q, H) ** 2) / C + (h * np.abs(grads["k"]) + tiny) ** 2
    assert ((np64(d["k"]) - grads["k"]) ** 2).sum() <= bound.sum()


def test_attention_fp32_as_before():
    """fp32 operands have no such step."""
    a, dout = aligned(7, 1, 1, 2, 64, 8, 2, None, False, 0.02, 16.0, 2000.0)
    a = {n: t.float() if torch.is_tensor(t) else t for n, t in a.items()}
    o, stats = call(a, 2)
    _, _, tol, grads = tolerances(a, 2, F32, dout.float())
    for n, x in grads.items():
        close(call_bwd(dout.float(), a, 2, o, stats)[n], x, tol[n])
