"""The sequence attention's training form on the GPU (position bias by buckets, norms of queries and keys with the rotation,
the attention and its gradients) against the float64 oracle.

Tolerances, from the kernels' arithmetic: u = 2^-24 is fp32's half step, h the half step of a half type (fp16 2^-11, bf16
2^-8; 0 in fp32). Bounds are sums over the terms' sizes, first order.
Position bias: one addition in fp32, one rounding. Its gradient: a sum whose terms pass at most as many additions as a wave
makes for its rows, and those of the waves and of the partial sums.
Norms: a sum of C <= 256 squares passes at most 22 additions, halved by the root: xh errs by 16u; an angle by 4u (its turns'
rounding) and the 2^-52 of its turns, its sine and cosine by 2u more. y: 32u of the pair's sizes. dx, with G the pair's sizes
of dy: g errs by 10u G, the mean of w g xh by 60u of the mean of the sizes: rstd u (32 |w| G + 96 |xh| mean(|w| G |xh|)).
Attention. x: ex = u (C + 4) sum |q k| / sqrt(C) + 2u |x|. e = exp(x - top): relative E = 2 max(ex) + u (2 |x - top| + 8), at the
largest |x - top| below 100 (past it e < 2^-140 adds nothing). The sum of M terms: E + u (M / 2 + 8). So p: Ep = 2E + u (M + 16).
out: sum p |v| (E + h + u M) + |out| (E + u M + 8u), gated, and what fp16 loses below 2^-14: 2^-25 a term.
Backward, with T the bound of out and its rounding: dO errs by 8u + h^2 of its size (two parts), dp by u (2 C) sum |dO v| + those;
delta is mended by the sum of ds over the row, which leaves the errors of its terms: dd = sum p (ep |dp| + edp); so
ds: p (|dp| + |delta|) (Ep + 4u) + p (edp + dd), dbias that and its rounding; dq: the sum over keys of (eds + h |ds|) |k| +
u M sum |ds k| and the mending's own p k term |delta's error| h sum p |k|; dk over queries; dv: sum over queries of p |dO| (Ep +
h + u N) + p |edO|; dg: |dout| T |1 - s| + 8u."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attention as T  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
STEP = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 1e-37, F16: 2.0 ** -25, BF16: 1e-37}
PAIRS = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]


def K():
    from boltz_mlx_amd import kernels

    return kernels


def A():
    from boltz_mlx_amd import autograd

    return autograd


def rand(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def np64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def close(got, ref, tol, dtype=None):
    dtype = dtype or got.dtype
    got = np64(got)
    assert got.shape == ref.shape
    fine = np.isfinite(ref)
    assert np.array_equal(got[~fine], ref[~fine], equal_nan=True)
    tol = np.broadcast_to(tol, ref.shape)[fine]
    err, ref = np.abs(got[fine] - ref[fine]), ref[fine]
    lim = tol + (STEP[dtype] * (np.abs(ref) + tol) + TINY[dtype] + U * np.abs(ref))
    bad = ~(err <= lim)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float((err / lim).max()))


# -------------------------------------------------------------------------------------------------- position bias

def positions(seed, *shape, chains=1):
    """Rising positions with gaps, and the chains that the tokens are in."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pos = (1 + torch.randint(0, 3, shape, generator=g, device="cuda")).cumsum(-1) - 5
    return pos, (torch.arange(shape[-1], device="cuda") * chains // shape[-1]).expand(shape).contiguous()


def grad_depth(B, H, N, M):
    """Additions that a term passes at most: those of its wave's rows (32 pairs and three parts in a product at most), of the
    four waves, and of the partial sums, 16 at a time."""
    others = B * -(-H // 16) * -(-M // 128)
    blocks = min(-(-768 // others), -(-N // 8))
    return 97 * -(-N // blocks) + 4 + B * blocks * -(-M // 128) // 16 + 16


BIASES = [
    # B, H, N, M, edges, chains
    (1, 1, 1, 1, [0], 1), (1, 16, 29, 29, "clip32", 1), (2, 5, 33, 70, "clip5", 3), (3, 2, 130, 3, [-7, 0, 2, 40], 2),
    (1, 3, 7, 1030, "clip32", 2), (1, 7, 257, 255, "log", 1), (2, 16, 400, 400, "clip32", 5), (1, 33, 64, 9, "clip1", 4),
    (1, 2, 300, 2049, "far", 1), (1, 1, 5, 8, [], 1), (1, 40, 20, 21, "most", 1),
]
EDGES = {"clip32": lambda: K().clipped_edges(32), "clip5": lambda: K().clipped_edges(5), "clip1": lambda: K().clipped_edges(1),
         "log": lambda: [-64, -32, -16, -8, -4, -2, -1, 0, 1, 2, 4, 8, 16, 32, 64], "far": lambda: [-9000, -1, 0, 7000],
         "most": lambda: K().clipped_edges(127)}


@pytest.mark.parametrize("B, H, N, M, edges, chains", BIASES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rel_bias(B, H, N, M, edges, chains, dtype):
    edges = EDGES[edges]() if isinstance(edges, str) else edges
    b = K().rel_buckets(edges, chains > 1)
    pq, cq = positions(1, B, N, chains=chains)
    pk, ck = (pq, cq) if N == M else positions(2, B, M, chains=chains)
    if dtype == F16:
        pq, pk, cq, ck = (x.int() for x in (pq, pk, cq, ck))
    table = rand(3, b.count, H, dtype=dtype)
    at = T.buckets(edges, *(x.cpu().numpy() for x in (pq, pk))) if chains == 1 else \
        T.buckets(edges, *(x.cpu().numpy() for x in (pq, pk, cq, ck)))
    if chains == 1:
        cq = ck = None
    y = K().rel_bias(table, b, pq, pk, cq, ck)
    assert y.dtype == dtype and np.array_equal(np64(y), T.rel_bias(np64(table), at))
    add = rand(4, B, H, N, M, dtype=dtype)
    y = K().rel_bias(table, b, pq, pk, cq, ck, add=add)
    close(y, T.rel_bias(np64(table), at, np64(add)), 0.0)
    dy = rand(5, B, H, N, M, scale=0.1, dtype=dtype)
    d = K().rel_bias_bwd(dy, b, pq, pk, cq, ck)
    want, size = T.rel_bias_grad(np64(dy), at, b.count), T.rel_bias_grad(np.abs(np64(dy)), at, b.count)
    assert d.dtype == F32
    close(d, want, grad_depth(B, H, N, M) * U * size)
    assert torch.equal(d, K().rel_bias_bwd(dy, b, pq, pk, cq, ck))  # a fixed order of sums


@pytest.mark.parametrize("lut, count", [([0, 1, 2], 3), ([1, 1, 4, 4, 4, 20], 21), ([0], 1), ([2, 2], 40), ([0, 17, 33, 90], 91)])
def test_rel_bias_look_up_tables_of_ones_own(lut, count):
    """A table that skips buckets, has equal entries, or shares the bucket of other groups' pairs with its end."""
    H, N, M = 18, 70, 100
    g = torch.Generator(device="cuda").manual_seed(2)
    pq, pk = (torch.randint(-8, 8, (n,), generator=g, device="cuda") for n in (N, M))
    cq, ck = ((torch.arange(n, device="cuda") * 2) // n for n in (N, M))
    for other in (False, True):
        b = K().RelBuckets(torch.tensor(lut, dtype=torch.uint8, device="cuda"), -2, count, other)
        d = (pq[:, None] - pk[None]).cpu().numpy()
        at = np.array(lut)[np.clip(d + 2, 0, len(lut) - 1)]
        if other:
            at = np.where((cq[:, None] == ck[None]).cpu().numpy(), at, count - 1)
        table, dy = rand(1, count, H), rand(3, H, N, M)
        assert np.array_equal(np64(K().rel_bias(table, b, pq, pk, cq, ck)), T.rel_bias(np64(table), at))
        close(K().rel_bias_bwd(dy, b, pq, pk, cq, ck), T.rel_bias_grad(np64(dy), at, count),
              grad_depth(1, H, N, M) * U * T.rel_bias_grad(np.abs(np64(dy)), at, count))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N, M", [(31, 65), (70, 77), (9, 8), (40, 129), (33, 96), (5, 7)])
def test_rel_bias_values_inside_dwords(N, M, dtype):
    """Rows of odd lengths in 16-bit types, tensors that begin inside a dword."""
    H, b = 5, K().rel_buckets(K().clipped_edges(7))
    pq, pk = positions(1, N)[0], positions(2, M)[0]
    at = T.buckets(K().clipped_edges(7), pq.cpu().numpy(), pk.cpu().numpy())
    table = rand(3, b.count, H, dtype=dtype)
    for offset in (0, 1, 2):
        dy, add = (rand(s, offset + H * N * M, scale=0.1, dtype=dtype)[offset:].view(H, N, M) for s in (4, 5))
        close(K().rel_bias_bwd(dy, b, pq, pk), T.rel_bias_grad(np64(dy), at, b.count),
              grad_depth(1, H, N, M) * U * T.rel_bias_grad(np.abs(np64(dy)), at, b.count))
        close(K().rel_bias(table, b, pq, pk, add=add), T.rel_bias(np64(table), at, np64(add)), 0.0)


@pytest.mark.parametrize("M", [5, 77, 130])
def test_rel_bias_numbers_past_32_bits(M):
    """Neighbouring keys 2^45 positions apart, groups whose numbers differ in their upper halves alone, queries of a group that
    no key has; one bucket for pairs of different groups that the edges reach too, and one that they do not."""
    H, N = 3, 70
    g = torch.Generator(device="cuda").manual_seed(4)
    big = lambda n: torch.randint(-3, 4, (n,), generator=g, device="cuda") * 2 ** 45 + torch.randint(0, 9, (n,), generator=g, device="cuda")
    near = lambda n: torch.randint(0, 40, (n,), generator=g, device="cuda") + 2 ** 45
    group = lambda n: torch.randint(0, 3, (n,), generator=g, device="cuda") * 2 ** 32 + 7
    few = lambda n: (torch.arange(n, device="cuda") * 3 // n) % 3
    for pos, ids in ((big, None), (near, group), (big, few), (near, few)):
        for other in (True, False):
            edges = K().clipped_edges(6)
            b = K().rel_buckets(edges, other)
            pq, pk = pos(N), pos(M)
            cq, ck = (None, None) if ids is None else (ids(N), ids(M))
            if ids is not None:
                cq[3], cq[9] = 2 ** 40, -1
            np_ = lambda *t: [x.cpu().numpy() for x in t]
            at = T.buckets(edges, *np_(pq, pk)) if not other or ids is None else T.buckets(edges, *np_(pq, pk, cq, ck))
            table, dy = rand(1, b.count, H), rand(3, H, N, M)
            assert np.array_equal(np64(K().rel_bias(table, b, pq, pk, cq, ck)), T.rel_bias(np64(table), at))
            close(K().rel_bias_bwd(dy, b, pq, pk, cq, ck), T.rel_bias_grad(np64(dy), at, b.count),
                  grad_depth(1, H, N, M) * U * T.rel_bias_grad(np.abs(np64(dy)), at, b.count))


def test_rel_bias_unordered_positions_and_shared_batches():
    """Positions in any order (chunks whose ends say nothing), a batch from one side alone, or from the pair bias alone."""
    H, N, M = 3, 50, 77
    g = torch.Generator(device="cuda").manual_seed(3)
    edges = K().clipped_edges(6)
    b = K().rel_buckets(edges, True)
    pq, pk = (torch.randint(-9, 9, (n,), generator=g, device="cuda") for n in (N, M))
    cq, ck = (torch.randint(0, 3, (n,), generator=g, device="cuda") for n in (N, M))
    table, add, dy = rand(1, b.count, H), rand(2, 4, H, N, M), rand(3, 4, H, N, M)
    at = T.buckets(edges, *(x.cpu().numpy() for x in (pq, pk, cq, ck)))
    assert np.array_equal(np64(K().rel_bias(table, b, pq, pk, cq, ck)), T.rel_bias(np64(table), at))
    close(K().rel_bias(table, b, pq, pk, cq, ck, add=add), T.rel_bias(np64(table), at, np64(add)), 0.0)
    close(K().rel_bias_bwd(dy, b, pq, pk, cq, ck), T.rel_bias_grad(np64(dy), at, b.count),
          grad_depth(4, H, N, M) * U * T.rel_bias_grad(np.abs(np64(dy)), at, b.count))
    pb, cb = torch.stack([pk, pk + 2, pk.flip(0), pk - 40]), torch.stack([ck, ck, ck.flip(0), ck])
    at = T.buckets(edges, np.broadcast_to(pq.cpu().numpy(), (4, N)), pb.cpu().numpy(), np.broadcast_to(cq.cpu().numpy(), (4, N)),
                   cb.cpu().numpy())
    assert np.array_equal(np64(K().rel_bias(table, b, pq, pb, cq, cb)), T.rel_bias(np64(table), at))
    far = torch.tensor([-2 ** 61, 0, 2 ** 61], device="cuda")  # differences of 62 bits
    at = T.buckets(edges, far.cpu().numpy(), far.cpu().numpy())
    assert np.array_equal(np64(K().rel_bias(table, b._replace(other=False), far)), T.rel_bias(np64(table), at))


def test_rel_bias_views_and_empty():
    b = K().rel_buckets(K().clipped_edges(3))
    pos, table = torch.arange(40, device="cuda"), rand(1, 7, 4)
    want = K().rel_bias(table, b, pos)
    assert torch.equal(K().rel_bias(table.t().contiguous().t(), b, torch.arange(80, device="cuda")[::2] // 2), want)
    dy = rand(2, 4, 40, 40)
    assert torch.equal(K().rel_bias_bwd(dy.transpose(1, 2).contiguous().transpose(1, 2), b, pos), K().rel_bias_bwd(dy, b, pos))
    big = torch.zeros(4 * 1600 + 1, device="cuda", dtype=F16)[1:].view(4, 40, 40)  # an odd offset
    assert torch.equal(K().rel_bias(table, b, pos, add=big), want.half())
    assert K().rel_bias(table, b, pos[:0], pos).shape == (4, 0, 40)
    assert (K().rel_bias_bwd(dy[:, :, :0], b, pos, pos[:0]) == 0).all()


def test_rel_bias_long():
    """More than 2^31 elements: the last rows, and a gradient whose values say where they were."""
    H, N = 16, 11700
    b = K().rel_buckets(K().clipped_edges(32))
    pos, table = torch.arange(N, device="cuda"), rand(1, 65, H, dtype=BF16)
    y = K().rel_bias(table, b, pos)
    assert y.numel() > 2 ** 31
    at = (pos[-3:, None] - pos[None]).clamp(-32, 32) + 32
    assert torch.equal(y[:, -3:], table[at].permute(2, 0, 1))
    y.zero_()
    y[15, N - 1] = 1.0
    y[15, N - 1, N - 1] = 3.0
    d = K().rel_bias_bwd(y, b, pos)
    want = torch.zeros(65, H, device="cuda")
    want[32, 15], want[64, 15], want[33:64, 15] = 3.0, N - 32.0, 1.0
    assert torch.equal(d, want)


# -------------------------------------------------------------------------------------------------- norms and rotation

def pair_sizes(x, H, rotary, interleaved):
    """For each element the sum of its pair's sizes."""
    h = np.abs(x).reshape(len(x), H, -1).copy()
    first = np.arange(0, rotary, 2) if interleaved else np.arange(rotary // 2)
    second = first + (1 if interleaved else rotary // 2)
    s = h[..., first] + h[..., second]
    h[..., first] = h[..., second] = s
    return h


def norm_tols(dy, x, w, H, rotary, interleaved, pos, eps=1e-5):
    """Tolerances of y, dx and dw."""
    rows, C = len(x), x.shape[1] // H
    h = x.reshape(rows, H, C)
    rs = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    xh, w = np.abs(h * rs), np.ones(C) if w is None else np.abs(w)
    far = 0 if pos is None else np.abs(np.asarray(pos, dtype=np.float64)).max() * 2.0 ** -50
    ty = (32 * U + far) * pair_sizes((xh * w).reshape(x.shape), H, rotary, interleaved)
    G = pair_sizes(dy, H, rotary, interleaved)
    eg = (10 * U + far) * G
    mean = (w * G * xh).mean(-1, keepdims=True)
    tdx = rs * (w * (eg + 22 * U * G) + xh * (96 * U + 2 * far) * mean)
    depth = 64 + rows * H // 64
    tdw = (eg * xh + 24 * U * G * xh).sum((0, 1)) + depth * U * (G * xh).sum((0, 1))
    return ty.reshape(x.shape), tdx.reshape(x.shape), tdw


def check_norms(x, w, H, pos, rotary, interleaved, y=None, dy=None, dx=None, dw=None):
    C = x.shape[-1] // H
    kw = dict(rotary=rotary, interleaved=interleaved)
    xn = np64(x).reshape(-1, H * C)
    p = None if pos is None else pos.cpu().numpy().reshape(-1)
    if p is not None and len(p) < len(xn):
        p = np.tile(p, len(xn) // len(p))
    dyn = np.ones_like(xn) if dy is None else np64(dy).reshape(-1, H * C)
    ty, tdx, tdw = norm_tols(dyn, xn, np64(w), H, rotary, interleaved, p)
    if y is not None:
        close(y.reshape(-1, H * C), T.qk_norm_rope(xn, np64(w), H, p, **kw), ty)
    if dy is not None:
        rx, rw = T.qk_norm_rope_grads(dyn, xn, np64(w), H, p, **kw)
        close(dx.reshape(-1, H * C), rx, tdx)
        close(dw, rw, tdw)


# C, rotary, interleaved: every number of pairs a lane holds (8, 4, 2, 1) and of lanes a head, both layouts, tails
HEADS = [(2, 2, False), (2, 0, True), (6, 4, True), (8, 8, False), (10, 6, False), (16, 16, True), (24, 24, False), (24, 12, True),
         (32, 32, False), (48, 48, True), (48, 16, False), (64, 64, False), (66, 66, False), (96, 64, True), (100, 52, False),
         (128, 128, False), (128, 64, True), (130, 130, True), (190, 62, False), (254, 254, False), (254, 2, True), (256, 256, True),
         (256, 0, False)]


@pytest.mark.parametrize("C, rotary, interleaved", HEADS)
def test_qk_norm_rope(C, rotary, interleaved):
    for n, (tx, ty) in enumerate(PAIRS):
        rows, H, Hk = [1, 2, 5, 33, 130, 7, 64][n], [1, 4, 3, 16, 5, 8, 12][n], [1, 2, 1, 16, 5, 4, 3][n]
        q, k = rand(n, rows, H * C, dtype=tx), rand(n + 50, rows, Hk * C, scale=3.0, dtype=tx)
        wq, wk = 1 + rand(1, C, scale=0.2), (None if n == 3 else 1 + rand(2, C, scale=0.2))
        pos = torch.arange(rows, device="cuda") * [1, 3, 1000003, 77, 1, 12345, 1][n] + [0, -5, 7, 10 ** 7, 0, 3, 2 ** 24][n]
        if n % 2:
            pos = pos.int()
        kw = dict(rotary=rotary, interleaved=interleaved)
        qn, kn = K().qk_norm_rope(q, k, wq, wk, H, pos, out_dtype=ty, **kw)
        assert qn.dtype == kn.dtype == ty and qn.shape == q.shape and kn.shape == k.shape
        dq, dk = rand(3, rows, H * C, scale=0.1, dtype=ty), rand(4, rows, Hk * C, scale=0.1, dtype=ty)
        gq, gk, gwq, gwk = K().qk_norm_rope_bwd(dq, dk, q, k, wq, wk, H, pos, **kw)
        assert gq.dtype == gk.dtype == tx and gwq.dtype == gwk.dtype == F32
        check_norms(q, wq, H, pos, rotary, interleaved, qn, dq, gq, gwq)
        check_norms(k, wk, Hk, pos, rotary, interleaved, kn, dk, gk, gwk)


@pytest.mark.parametrize("rows, H, Hk, C, dtype", [(9000, 4, 4, 32, F32), (5001, 16, 2, 48, BF16), (20011, 1, 1, 64, F16),
                                                   (700, 64, 64, 24, F32), (3, 300, 7, 128, BF16), (1, 1024, 1024, 8, F32)])
def test_qk_norm_rope_many(rows, H, Hk, C, dtype):
    """Several workgroups with several tokens each, more heads than a wave holds, heads split over waves."""
    q, k, w = rand(1, rows, H * C, dtype=dtype), rand(2, rows, Hk * C, dtype=dtype), 1 + rand(3, C, scale=0.1)
    pos = torch.arange(rows, device="cuda")
    qn, kn = K().qk_norm_rope(q, k, w, w, H, pos)
    dq, dk = rand(4, rows, H * C, scale=0.1, dtype=dtype), rand(5, rows, Hk * C, scale=0.1, dtype=dtype)
    g = K().qk_norm_rope_bwd(dq, dk, q, k, w, w, H, pos)
    check_norms(q, w, H, pos, C, False, qn, dq, g[0], g[2])
    check_norms(k, w, Hk, pos, C, False, kn, dk, g[1], g[3])
    assert all(torch.equal(a, b) for a, b in zip(g, K().qk_norm_rope_bwd(dq, dk, q, k, w, w, H, pos)))


def test_qk_norm_rope_views_positions_and_none():
    """Slices of a fused projection, odd offsets, batches that share their positions, no positions, no rows."""
    B, N, H, C = 3, 37, 4, 24
    packed = rand(1, B, N, 4 * H * C, dtype=F16)
    q, k = packed[..., :H * C], packed[..., H * C:2 * H * C]
    w, pos = 1 + rand(2, C, scale=0.1), torch.arange(N, device="cuda") + 100
    want = K().qk_norm_rope(q.contiguous(), k.contiguous(), w, w, H, pos.expand(B, N).contiguous())
    for a, b in zip(K().qk_norm_rope(q, k, w, w, H, pos), want):
        assert torch.equal(a, b)
    flat = torch.empty(B * N * H * C + 1, device="cuda", dtype=F16)[1:].view(B, N, H * C)
    flat.copy_(q)
    assert torch.equal(K().qk_norm_rope(flat, k, w, w, H, pos)[0], want[0])
    swapped = K().qk_norm_rope(q.transpose(0, 1), k.transpose(0, 1), w, w, H, pos[:, None].expand(N, B))
    assert torch.equal(swapped[0], want[0].transpose(0, 1))
    strided = torch.empty(B, N, 2 * H * C, device="cuda", dtype=F16)[..., ::2]
    strided.copy_(q)
    assert torch.equal(K().qk_norm_rope(strided, k, w, w, H, pos)[0], want[0])
    assert torch.equal(K().qk_norm_rope(q[:1].expand(B, N, -1), k, w, w, H, pos)[0][2], want[0][0])
    still = K().qk_norm_rope(q, k, w, None, H)
    check_norms(q, w, H, None, 0, False, still[0])
    check_norms(k, None, H, None, 0, False, still[1])
    out = K().qk_norm_rope(q[:, :0], k[:, :0], w, w, H, pos[:0])
    assert out[0].shape == (B, 0, H * C)
    g = K().qk_norm_rope_bwd(out[0], out[1], q[:, :0], k[:, :0], w, w, H, pos[:0])
    assert (g[2] == 0).all() and (g[3] == 0).all() and g[0].shape == (B, 0, H * C)
    assert K().qk_norm_rope_bwd(want[0], want[1], q, k, w, w, H, pos, need_weights=False)[2:] == (None, None)


def test_qk_norm_rope_extremes():
    """Rows of zeros, of tiny and of large values; one token far away against one position less."""
    C = 64
    x = torch.zeros(4, C, device="cuda")
    x[1], x[2], x[3] = 1e-18, 1e15, rand(1, C)
    pos = torch.tensor([5, 6, 7, 2 ** 40], device="cuda")
    q, k = K().qk_norm_rope(x, x, None, None, 1, pos)
    check_norms(x, None, 1, pos, C, False, q)
    assert torch.equal(q, k) and (q[0] == 0).all()
    dy = rand(2, 4, C)
    g = K().qk_norm_rope_bwd(dy, dy, x, x, None, None, 1, pos)
    check_norms(x, None, 1, pos, C, False, q, dy, g[0], g[2])


def test_qk_norm_rope_long():
    """More than 2^31 elements."""
    rows, H, C = 2 ** 20 + 3, 16, 128
    q = rand(1, 1024, H * C, dtype=BF16).repeat(1025, 1)[:rows]
    pos = torch.arange(rows, device="cuda", dtype=torch.int32)
    w = 1 + rand(2, C, scale=0.1)
    qn, _ = K().qk_norm_rope(q, q[:, :C], w, w, H, pos)
    assert qn.numel() > 2 ** 31
    check_norms(q[-3:], w, H, pos[-3:], C, False, qn[-3:])
    del qn
    dy = torch.zeros_like(q)
    dy[-1] = rand(3, H * C, dtype=BF16)
    gq, _, gw, _ = K().qk_norm_rope_bwd(dy, dy[:, :C], q, q[:, :C], w, w, H, pos)
    check_norms(q[-2:], w, H, pos[-2:], C, False, None, dy[-2:], gq[-2:], gw)


# -------------------------------------------------------------------------------------------------- attention

def inputs(seed, S, mult, H, C, N, M, dtype, bias="same", gate=True, mask="tail", scale=1.0):
    a = {"q": rand(seed, S, N, H * C, scale=scale, dtype=dtype), "k": rand(seed + 1, S, M, H * C, scale=scale, dtype=dtype),
         "v": rand(seed + 2, S, M, H * C, dtype=dtype), "g": rand(seed + 3, S, N, H * C, dtype=dtype) if gate else None}
    a["bias"] = None if bias is None else rand(seed + 4, S // mult, H, N, M, dtype=dtype if bias == "same" else bias)
    a["mask"] = None
    if mask:
        m = torch.ones(S, M, device="cuda")
        for s in range(S):
            if mask == "tail":
                m[s, max(1, M - 3 * s - M // 5):] = 0
            elif mask == "holes":
                m[s] = (rand(seed + 9 + s, M) > 0.3).float()
        if mask == "holes" and S > 1:
            m[S - 1] = 0  # no key: runs without its mask
        a["mask"] = m
    a["mult"] = mult
    return a


def heads(x, H):
    return x.reshape(*x.shape[:-1], H, -1).swapaxes(-2, -3)


def rows(x):
    return x.swapaxes(-2, -3).reshape(*x.shape[:-3], x.shape[-2], -1)


def tolerances(a, H, dtype, dout=None):
    """The docstring's bounds of out, stats and the gradients, in float64."""
    h, tiny = STEP[dtype], 2.0 ** -25 if dtype == F16 else 0.0
    q, k, v, g, bias = (np64(a[n]) for n in ("q", "k", "v", "g", "bias"))
    mask, mult = np64(a["mask"]), a["mult"]
    M, N, C = k.shape[1], q.shape[1], q.shape[2] // H
    out, stats, p = T.attention(q, k, v, H, g, bias, mask, mult)
    if mask is not None:
        on = mask != 0
        on = on | ~on.any(1, keepdims=True)
        k, v = np.where(on[..., None], k, 0.0), np.where(on[..., None], v, 0.0)
    x = heads(q, H) @ heads(k, H).swapaxes(-1, -2) / np.sqrt(C)
    ax = heads(np.abs(q), H) @ heads(np.abs(k), H).swapaxes(-1, -2) / np.sqrt(C)
    if bias is not None:
        b = np.repeat(bias, mult, 0)
        x, ab = x + b, np.where(np.isfinite(b), np.abs(b), 0.0)
        ax = ax + np.minimum(ab, 1e30)
    top = stats[..., :1]
    ref = np.where(np.isfinite(top), top, 0.0)
    seen = p > 0
    ex = np.where(seen, U * (C + 6) * ax, 0.0).max(-1, keepdims=True)
    E = 2 * ex + U * (2 * np.where(seen, np.minimum(np.abs(x - ref), 100), 0).max(-1, keepdims=True) + 8)
    Ep = 2 * E + U * (M + 16)
    total = np.maximum(stats[..., 1:], 1.0)
    s = 1.0 if g is None else 1 / (1 + np.exp(-g))
    pv = p @ heads(np.abs(v), H)
    t_out = rows(pv * (E + h + U * M) + np.abs(p @ heads(v, H)) * (E + U * M + 8 * U) +
                 tiny * heads(np.abs(v), H).sum(-2, keepdims=True) / total) * s
    t = {"out": t_out, "stats": np.concatenate([ex + U * np.abs(ref), stats[..., 1:] * (E + U * (M / 2 + 8)) + 1e-30], -1)}
    if dout is None:
        return out, stats, t, None
    dout = np64(dout)
    grads = T.attention_grads(dout, q, np64(a["k"]), np64(a["v"]), H, g, bias, mask, mult)
    d = dout if g is None else dout * s
    ed = np.abs(d) * (8 * U + h * h) + tiny * (g is not None) if g is not None else 0 * d
    d, ed, ak, aq, av = heads(d, H), heads(ed, H), heads(np.abs(k), H), heads(np.abs(q), H), heads(np.abs(v), H)
    dp = d @ heads(v, H).swapaxes(-1, -2)
    edp = U * 2 * C * (np.abs(d) @ av.swapaxes(-1, -2)) + ed @ av.swapaxes(-1, -2)
    delta = (p * dp).sum(-1, keepdims=True)
    dd = (p * (Ep * np.abs(dp) + edp)).sum(-1, keepdims=True) + U * M * (p * np.abs(dp)).sum(-1, keepdims=True)
    if dtype == F32:  # delta is formed from out: its error there
        dd = dd + heads(np.abs(dout) * (t_out + U * C * np.abs(out)), H).sum(-1, keepdims=True)
    ds = p * (dp - delta)
    eds = p * (np.abs(dp) + np.abs(delta)) * (Ep + 4 * U) + p * (edp + dd)
    # what out's rounding leaves of delta before it is mended, which meets p k rounded
    raw = heads(np.abs(dout) * ((t_out + h * (np.abs(out) + t_out) + tiny) * 1.0), H).sum(-1, keepdims=True)
    scale = 1 / np.sqrt(C)
    low = tiny * np.sqrt(C / total)  # fp16's ds at p total / 2^n, 2^n <= sqrt(C total): its 2^-25 counts 2^n / total at most
    # Half types take the rounded ds' own sum off dq: with e_j the rounding of ds_j, (sum of e_j ds_j) (sum of p k) on top of the
    # (sum of e_j ds_j k_j) that the products have, together sum of e_j ds_j (k_j - sum of p k); raw's part of ds as there.
    taken = (h * (np.abs(ds) + p * raw) + low * np.ones_like(ds)).sum(-1, keepdims=True) * np.abs(p @ heads(k, H)) * (1 + h)
    t["q"] = scale * rows((eds + h * (np.abs(ds) + 2 * p * raw) + low * (1 + raw)) @ ak + U * M * ((np.abs(ds) + p * raw) @ ak) + taken)
    t["k"] = scale * rows((eds + h * np.abs(ds) + tiny).swapaxes(-1, -2) @ aq + U * N * (np.abs(ds).swapaxes(-1, -2) @ aq))
    t["v"] = rows((p * (Ep + h + U * N) + tiny).swapaxes(-1, -2) @ np.abs(d) + p.swapaxes(-1, -2) @ ed)
    if g is not None:
        t["g"] = np.abs(dout) * (t_out + STEP[dtype] * (np.abs(out) + t_out) + tiny) * np.abs(1 - s) + 10 * U * np.abs(dout * out)
    if bias is not None:
        t["bias"] = (eds + 4 * U * mult * np.abs(ds)).reshape(-1, mult, *eds.shape[1:]).sum(1)
    return out, stats, t, grads


def call(a, H):
    return K().attention(a["q"], a["k"], a["v"], H, g=a["g"], bias=a["bias"], mask=a["mask"], multiplicity=a["mult"])


def call_bwd(dout, a, H, out, stats, **kw):
    d = K().attention_bwd(dout, a["q"], a["k"], a["v"], H, out, stats, g=a["g"], bias=a["bias"], mask=a["mask"],
                          multiplicity=a["mult"], **kw)
    return dict(zip(("q", "k", "v", "g", "bias"), d))


def check(a, H, backward=True):
    dtype = a["q"].dtype
    o, stats = call(a, H)
    assert o.dtype == dtype and stats.dtype == F32
    dout = rand(77, *o.shape, scale=0.1, dtype=dtype) if backward else None
    want, wstats, tol, grads = tolerances(a, H, dtype, dout)
    close(o, want, tol["out"])
    close(stats, wstats, tol["stats"])
    if backward:
        d = call_bwd(dout, a, H, o, stats)
        assert (d["g"] is None) == (a["g"] is None) and (d["bias"] is None) == (a["bias"] is None)
        for n, x in grads.items():
            assert d[n].dtype == (a["bias"].dtype if n == "bias" else dtype)
            close(d[n], x, tol[n])
    return o, stats


SHAPES = [
    # S, mult, H, C, N, M: one token, whole and odd tiles on both sides, every number of channel steps
    (1, 1, 1, 8, 1, 1), (1, 1, 16, 24, 1, 50), (2, 1, 3, 16, 31, 33), (2, 2, 2, 32, 64, 64), (1, 1, 4, 40, 65, 127),
    (3, 3, 2, 48, 100, 100), (2, 1, 2, 56, 33, 1), (2, 1, 1, 64, 129, 130), (1, 1, 2, 72, 40, 41), (2, 2, 1, 96, 70, 66),
    (1, 1, 1, 104, 35, 96), (2, 1, 1, 128, 96, 63), (4, 2, 5, 24, 21, 19),
]


@pytest.mark.parametrize("S, mult, H, C, N, M", SHAPES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention(S, mult, H, C, N, M, dtype):
    for n, (bias, gate, mask) in enumerate([("same", True, "tail"), (None, False, None), ("same", False, "holes"),
                                            (None, True, "holes")]):
        check(inputs(10 * n + C, S, mult, H, C, N, M, dtype, bias, gate, mask), H)


@pytest.mark.parametrize("S, mult, H, C, N, M, dtype", [
    (1, 1, 16, 24, 400, 400, F32), (5, 5, 16, 48, 200, 200, F16), (33, 1, 16, 32, 130, 140, BF16), (40, 4, 13, 24, 129, 65, F32),
    (36, 1, 15, 64, 70, 70, F16), (1, 1, 2, 64, 1, 3000, BF16), (1, 1, 2, 32, 700, 2, F16), (36, 3, 16, 128, 33, 40, BF16),
])
def test_attention_larger(S, mult, H, C, N, M, dtype):
    """Both workgroup sizes, many samples, a long axis on either side."""
    check(inputs(1, S, mult, H, C, N, M, dtype, "same", True, "tail"), H)


@pytest.mark.parametrize("S, mult, H, C, N, M", [
    (3, 1, 4, 72, 40, 41), (2, 2, 3, 96, 70, 66), (6, 1, 2, 104, 35, 96), (3, 3, 2, 128, 96, 63), (7, 1, 2, 56, 33, 1), (7, 1, 1, 16, 31, 33),
    (1, 1, 8, 8, 100, 100), (25, 5, 2, 120, 33, 7), (13, 1, 3, 88, 6, 200),
])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_tiles(S, mult, H, C, N, M, dtype):
    """More than 192 rows in all: 32 x 32 tiles, every number of channel steps."""
    test_attention(S, mult, H, C, N, M, dtype)


@pytest.mark.parametrize("bias", [F16, BF16])
def test_attention_half_bias_with_fp32(bias):
    check(inputs(3, 4, 2, 3, 24, 50, 61, F32, bias), 3)
    check(inputs(3, 2, 1, 2, 32, 33, 64, F32, bias, False, "holes"), 2)


@pytest.mark.parametrize("S, mult, H, C, N, M, dtype", [
    (1, 1, 16, 24, 1, 400, F32), (2, 2, 3, 64, 1, 5000, F32), (1, 1, 2, 128, 3, 2050, BF16), (3, 1, 1, 8, 4, 1025, F16),
    (1, 1, 1, 40, 2, 30011, BF16), (65, 5, 16, 32, 1, 257, F16), (2, 1, 4, 96, 4, 1, F32), (1, 1, 5, 72, 2, 4096, F16),
])
def test_attention_few_queries(S, mult, H, C, N, M, dtype):
    """One to four queries: keys by groups of lanes, a long axis split over workgroups."""
    for n, (bias, gate, mask) in enumerate([("same", True, "tail"), (None, False, None), ("same", False, "holes")]):
        check(inputs(10 * n + C, S, mult, H, C, N, M, dtype, bias, gate, mask), H, backward=M < 3000)


@pytest.mark.parametrize("N", [1, 40, 200])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_bars_of_different_sizes(N, dtype):
    """Rows that the bias bars altogether, with the type's lowest value in some places and -1e30 in others: a softmax over
    the latter's keys, in whatever order they come."""
    H, C, M = 2, 16, 700
    a = inputs(8, 1, 1, H, C, N, M, dtype, mask=None)
    low = torch.finfo(dtype).min
    for bars in ((low, -1e30), (-1e30, low)):
        a["bias"].fill_(low)
        a["bias"][..., 300:310] = -1e30
        if bars[0] != low:
            a["bias"][..., 300:310] = low
            a["bias"][..., :20] = -1e30
        at = (a["bias"][0, 0, 0] > -2e30).nonzero()[:, 0]
        o, stats = call(a, H)
        v = heads(np64(a["v"]), H)[:, :, at.cpu().numpy()]
        want = rows(np.broadcast_to(v.mean(2, keepdims=True), (1, H, N, C))) / (1 + np.exp(-np64(a["g"])))
        close(o, want, (STEP[dtype] + 64 * U) * np.abs(v).mean())
        assert (stats[..., 1] == len(at)).all() and (stats[..., 0] > -1.1e30).all()


@pytest.mark.parametrize("N, M", [(1, 300), (40, 300), (300, 40)])
@pytest.mark.parametrize("base", [9e5, -1.04e6, 1.0485775e6, 3e7, -1e9, -1e10, 4e12, -1e15, -1e30, 1.3e30, 3e38])
def test_attention_logits_far_from_zero(N, M, base):
    """Logits (the biases alone: q is 0) that are a large number and small steps from it, as far as fp32 has them: the softmax
    of the steps, forward and backward. p errs by u (2 |x - top| + 8 + M), and no step is past 100."""
    H, C = 2, 16
    for dtype, bias in ((F32, F32), (F32, BF16)):
        a = inputs(12, 1, 1, H, C, N, M, dtype, bias=bias, mask=None)
        a["q"].zero_()
        step = torch.randint(0, 9, a["bias"].shape, generator=torch.Generator().manual_seed(5)).cuda()
        a["bias"] = (torch.tensor(base, dtype=F32, device="cuda") - step).to(bias)
        o, stats = call(a, H)
        dout = rand(7, *o.shape, scale=0.1)
        d = call_bwd(dout, a, H, o, stats)
        want, wstats, _ = T.attention(*(np64(a[n]) for n in ("q", "k", "v")), H, np64(a["g"]), np64(a["bias"]), None, 1)
        grads = T.attention_grads(np64(dout), *(np64(a[n]) for n in ("q", "k", "v")), H, np64(a["g"]), np64(a["bias"]), None, 1)
        e = U * (2 * 8 + 8 + M)
        assert np.array_equal(np64(stats)[..., 0], wstats[..., 0])
        close(stats[..., 1], wstats[..., 1], e * wstats[..., 1])
        big = np.abs(np64(a["v"])).max()
        close(o, want, 4 * e * big)
        # dp of sizes up to C |dO| |v|, delta the same; sums over N or M of them with |k|
        size = C * np.abs(np64(dout)).max() * big * np.abs(np64(a["k"])).max()
        for n in ("q", "v", "bias"):
            close(d[n], grads[n], 8 * e * size * (N if n == "v" else 1))
        assert (d["k"] == 0).all()


def test_attention_is_seq_attention():
    """The inference kernels' result for the same inputs (their tolerance: both against the oracle's bound)."""
    N, H, C = 64, 4, 32
    for dtype in (F32, F16):
        a = inputs(1, 1, 1, H, C, N, N, dtype)
        want, _, tol, _ = tolerances(a, H, dtype)
        o = K().seq_attention(a["q"][0], a["k"][0], a["v"][0], a["g"][0], a["bias"][0], a["mask"][0], 1e6, H)
        lim = 4 * tol["out"][0] + 4 * STEP[dtype] * np.abs(want[0]) + 1e-5
        assert (np.abs(np64(o) - np64(call(a, H)[0])[0]) <= lim).all()


@pytest.mark.parametrize("N", [45, 5])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_masked_places_hold_anything(dtype, N):
    """Infinities and NaN in keys, values and biases that the mask leaves out; their gradients are 0."""
    S, H, C, M = 2, 3, 24, 70
    a = inputs(5, S, 1, H, C, N, M, dtype, mask="tail")
    a["mask"][0, 10], a["mask"][1, 0] = 0, 0
    o, stats = call(a, H)
    dout = rand(7, *o.shape, scale=0.1, dtype=dtype)
    d = call_bwd(dout, a, H, o, stats)
    off = a["mask"] == 0
    b = dict(a)
    for n, bad in (("k", float("nan")), ("v", float("inf"))):
        b[n] = a[n].clone()
        b[n][off] = bad
    b["bias"] = a["bias"].clone()
    b["bias"].transpose(1, 3)[off] = float("nan")
    o2, stats2 = call(b, H)
    assert torch.equal(o, o2) and torch.equal(stats, stats2)
    d2 = call_bwd(dout, b, H, o2, stats2)
    assert all(torch.equal(d[n], d2[n]) for n in d)
    assert (d["k"][off] == 0).all() and (d["v"][off] == 0).all() and (d["bias"].transpose(1, 3)[off] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("mult, S", [(1, 2), (2, 2), (1, 6), (2, 6)])
def test_attention_rows_without_keys(dtype, mult, S):
    """A bias that is -inf over a row (the row gives 0 and takes no gradient), over some of one, or the type's lowest value
    over a whole row (a softmax over equals) or over some."""
    H, C, N, M = 2, 32, 40, 77
    a = inputs(6, S, mult, H, C, N, M, dtype, mask="tail")
    low = torch.finfo(dtype).min
    a["bias"][:, 0, 3] = -float("inf")
    a["bias"][:, 1, 4, 5:] = -float("inf")
    a["bias"][:, 0, 6] = low
    a["bias"][:, 1, 7, 2:60] = low
    a["bias"][:, :, 8:10, :65] = -float("inf")
    o, stats = call(a, H)
    keep = torch.arange(N, device="cuda") != 6
    dout = rand(7, *o.shape, scale=0.1, dtype=dtype)
    d = call_bwd(dout, a, H, o, stats)
    assert (o[:, 3, :C] == 0).all() and (d["q"][:, 3, :C] == 0).all() and (d["bias"][:, 0, 3] == 0).all()
    assert torch.isinf(stats[:, 0, 3, 0]).all() and (stats[:, 0, 3, 1] == 0).all()
    want, wstats, tol, grads = tolerances(a, H, dtype, dout)
    assert all(torch.isfinite(x).all() for x in d.values())
    # at the type's lowest value a row's logits lose their own differences to it, in fp32 as in fp16 and bf16's (float64 keeps
    # those of fp16's lowest): there the row is compared with the softmax over equals
    rowsel = keep.cpu().numpy()
    close(o[:, keep], want[:, rowsel], tol["out"][:, rowsel])
    close(d["bias"][:, :, keep], grads["bias"][:, :, rowsel], tol["bias"][:, :, rowsel])
    if dtype != F16:
        on = a["mask"] != 0
        for s in range(S):
            v = a["v"][s, on[s], :C].double().mean(0) * torch.sigmoid(a["g"][s, 6, :C].double())
            lim = float(a["v"].abs().max()) * (STEP[dtype] * 2 + 1e-5)
            assert (o[s, 6, :C].double() - v).abs().max() <= lim


@pytest.mark.parametrize("S, N, M", [(1, 64, 600), (4, 64, 600), (1, 5, 900)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_large_gradients(dtype, S, N, M):
    """Gradients of an output that are thousands: products with v pass fp16's largest number, no gradient does."""
    H, C = 3, 64
    a = inputs(8, S, 1, H, C, N, M, dtype)
    a["v"] = rand(10, S, M, H * C, scale=4.0, dtype=dtype)
    o, stats = call(a, H)
    dout = rand(9, *o.shape, scale=4e3, dtype=dtype)
    want, _, tol, grads = tolerances(a, H, dtype, dout)
    d = call_bwd(dout, a, H, o, stats)
    s = 1 / (1 + np.exp(-np64(a["g"])))
    assert np.abs(heads(np64(dout) * s, H) @ heads(np64(a["v"]), H).swapaxes(-1, -2)).max() > 65504
    for n, x in grads.items():
        assert np.abs(x).max() < 65504
        close(d[n], x, tol[n])


def test_attention_large_logits():
    """Logits of hundreds: one key has all of a row's weight."""
    for dtype in (F32, F16, BF16):
        check(inputs(8, 2, 1, 2, 32, 50, 60, dtype, scale=8.0), 2)


def test_attention_views_and_strides():
    """Parts of a fused projection, odd offsets, samples that share keys, transposed layouts, an unbatched call."""
    S, H, C, N = 3, 4, 24, 50
    packed = rand(1, S, N, 4 * H * C, dtype=F16)
    q, k, v, g = packed.chunk(4, -1)
    bias, mask = rand(2, S, H, N, N, dtype=F16), torch.ones(S, N, device="cuda")
    mask[1, 30:] = 0
    a = {"q": q.contiguous(), "k": k.contiguous(), "v": v.contiguous(), "g": g.contiguous(), "bias": bias, "mask": mask, "mult": 1}
    o, stats = call(a, H)
    dout = rand(3, *o.shape, dtype=F16)
    d = call_bwd(dout, a, H, o, stats)

    def same(b):
        o2, stats2 = call({**a, **b}, H)
        assert torch.equal(o, o2) and torch.equal(stats, stats2)
        d2 = call_bwd(dout, {**a, **b}, H, o2, stats2)
        assert all(torch.equal(d[n], d2[n]) for n in d)

    same({"q": q, "k": k, "v": v, "g": g})
    odd = torch.empty(S, N, 4 * H * C + 1, device="cuda", dtype=F16)  # rows at odd elements
    odd[..., 1:] = packed
    same(dict(zip("qkvg", odd[..., 1:].chunk(4, -1))))
    flat = torch.empty(bias.numel() + 3, device="cuda", dtype=F16)[3:].view(bias.shape)
    flat.copy_(bias)
    same({"bias": flat})
    same({"q": q.transpose(0, 1).contiguous().transpose(0, 1), "k": k.transpose(1, 2).contiguous().transpose(1, 2),
          "bias": bias.transpose(2, 3).contiguous().transpose(2, 3)})
    one = K().attention(q[1], k[1], v[1], H, g=g[1], bias=bias[1], mask=mask[1])
    assert torch.equal(one[0], o[1]) and torch.equal(one[1], stats[1])
    d1 = K().attention_bwd(dout[1], q[1], k[1], v[1], H, *one, g=g[1], bias=bias[1], mask=mask[1])
    assert all(torch.equal(x, d[n][1]) for n, x in zip(("q", "k", "v", "g", "bias"), d1))
    shared = K().attention(q, k[:1].expand(S, N, -1), v[:1].expand(S, N, -1), H)
    assert torch.equal(shared[0][2], K().attention(q[2], k[0], v[0], H)[0])


def test_attention_empty():
    a = inputs(1, 2, 1, 2, 16, 5, 7, F32)
    o, stats = K().attention(a["q"][:, :0], a["k"], a["v"], 2)
    assert o.shape == (2, 0, 32) and stats.shape == (2, 2, 0, 2)
    d = K().attention_bwd(o, a["q"][:, :0], a["k"], a["v"], 2, o, stats)
    assert (d[1] == 0).all() and (d[2] == 0).all() and d[0].shape == (2, 0, 32)
    o, stats = K().attention(a["q"], a["k"][:, :0], a["v"][:, :0], 2)
    assert (o == 0).all() and (stats[..., 1] == 0).all() and torch.isneginf(stats[..., 0]).all()
    d = K().attention_bwd(o, a["q"], a["k"][:, :0], a["v"][:, :0], 2, o, stats)
    assert (d[0] == 0).all() and d[1].shape == (2, 0, 32)
    assert K().attention(a["q"][:0], a["k"][:0], a["v"][:0], 2)[0].shape == (0, 5, 32)


def test_attention_repeats_bit_for_bit():
    for dtype, mult in ((F32, 1), (BF16, 2), (F16, 1)):
        a = inputs(9, 4, mult, 8, 48, 150, 170, dtype)
        o, stats = call(a, 8)
        dout = rand(1, *o.shape, dtype=dtype)
        first = call_bwd(dout, a, 8, o, stats)
        for _ in range(3):
            o2, stats2 = call(a, 8)
            again = call_bwd(dout, a, 8, o2, stats2)
            assert torch.equal(o, o2) and torch.equal(stats, stats2) and all(torch.equal(first[n], again[n]) for n in first)
        some = call_bwd(dout, a, 8, o, stats, need_bias=False)
        assert some["bias"] is None and all(torch.equal(some[n], first[n]) for n in "qkvg")


def test_attention_past_32_bits():
    """A bias of more than 2^31 elements, each row with one key that takes its weight; the last rows and their gradients."""
    H, C, N, M = 2, 8, 32771, 32771
    q, k = torch.zeros(N, H * C, device="cuda", dtype=F16), torch.zeros(M, H * C, device="cuda", dtype=F16)
    v = rand(1, M, H * C, dtype=F16)
    bias = torch.zeros(H, N, M, device="cuda", dtype=F16)
    assert bias.numel() > 2 ** 31
    to = torch.arange(N, device="cuda").flip(0)
    bias[:, torch.arange(N, device="cuda"), to] = 60.0
    o, stats = K().attention(q, k, v, H, bias=bias)
    assert torch.equal(o[-40:], v[to[-40:]]) and torch.equal(o[:40], v[to[:40]])
    dout = rand(2, N, H * C, dtype=F16)
    d = K().attention_bwd(dout, q, k, v, H, o, stats, bias=bias)
    assert torch.equal(d[2][to[-40:]], dout[-40:]) and d[4].shape == bias.shape
    assert float(d[4][:, -40:].abs().max()) < 1e-2 and float(d[0].abs().max()) < 1e-2


# -------------------------------------------------------------------------------------------------- gradients

def test_autograd_is_the_backward_functions():
    """The autograd forms: the bits of the functions, gradients in their leaves' types, what needs none gets none."""
    S, H, C, N = 2, 3, 24, 40
    a = inputs(1, S, 2, H, C, N, N, F32)
    leaf = {n: a[n].clone().requires_grad_() for n in ("q", "k", "v", "g", "bias")}
    o = A().attention(leaf["q"], leaf["k"], leaf["v"], H, g=leaf["g"], bias=leaf["bias"], mask=a["mask"], multiplicity=2)
    dout = rand(3, *o.shape)
    o.backward(dout)
    o2, stats = call(a, H)
    d = call_bwd(dout, a, H, o2, stats)
    assert torch.equal(o, o2) and all(torch.equal(leaf[n].grad, d[n]) for n in leaf)
    o = A().attention(leaf["q"], a["k"], a["v"], H, bias=a["bias"], multiplicity=2)
    (gq,) = torch.autograd.grad(o, leaf["q"], dout)
    b = {**a, "g": None, "mask": None}
    o2, stats = call(b, H)
    assert torch.equal(gq, call_bwd(dout, b, H, o2, stats)["q"])
    o = A().attention(a["q"], a["k"], a["v"], H, g=a["g"], bias=leaf["bias"], multiplicity=2)
    (gb,) = torch.autograd.grad(o, leaf["bias"], dout)
    b = {**a, "mask": None}
    o2, stats = call(b, H)
    assert torch.equal(gb, call_bwd(dout, b, H, o2, stats)["bias"])

    q, k = leaf["q"], leaf["k"]
    w, wk, pos = (1 + rand(4, C, scale=0.1)).half().requires_grad_(), (1 + rand(5, C)).requires_grad_(), torch.arange(N, device="cuda")
    qn, kn = A().qk_norm_rope(q, k, w, wk, H, pos, rotary=16)
    g = torch.autograd.grad((qn, kn), (q, k, w, wk), (dout, 2 * dout))
    want = K().qk_norm_rope_bwd(dout, 2 * dout, a["q"], a["k"], w, wk, H, pos, rotary=16)
    assert g[2].dtype == F16 and torch.equal(g[0], want[0]) and torch.equal(g[1], want[1])
    assert torch.equal(g[2], want[2].half()) and torch.equal(g[3], want[3])
    qn, kn = A().qk_norm_rope(q, k, None, wk, H, pos)
    (gk,) = torch.autograd.grad(kn, wk, dout)  # the queries' output is not used
    assert torch.equal(gk, K().qk_norm_rope_bwd(torch.zeros_like(dout), dout, a["q"], a["k"], None, wk, H, pos)[3])

    b = K().rel_buckets(K().clipped_edges(8), True)
    chain = pos // 15
    table, add = rand(6, b.count, H).bfloat16().requires_grad_(), rand(7, S, H, N, N, dtype=F16).requires_grad_()
    y = A().rel_bias(table, b, pos, group_q=chain, add=add)
    assert y.dtype == F16
    dy = rand(8, *y.shape, dtype=F16)
    gt, ga = torch.autograd.grad(y, (table, add), dy)
    assert gt.dtype == BF16 and torch.equal(ga, dy)
    assert torch.equal(gt, K().rel_bias_bwd(dy, b, pos, group_q=chain).bfloat16())
    (ga,) = torch.autograd.grad(A().rel_bias(table.detach(), b, pos, group_q=chain, add=add), add, dy)
    assert torch.equal(ga, dy)


def test_gradients_against_differences():
    """Directional differences of the fp32 forward passes: an error of 2^-11 of a sum of thousands of terms, h^2 / 2 curvature."""
    H, C, N = 2, 16, 30
    a = inputs(2, 1, 1, H, C, N, N, F32)
    names = ("q", "k", "v", "g", "bias")
    dout = rand(5, 1, N, H * C)

    def f(x):
        return float((A().attention(x["q"], x["k"], x["v"], H, g=x["g"], bias=x["bias"], mask=a["mask"]).double() * dout).sum())

    leaf = {n: a[n].clone().requires_grad_() for n in names}
    o = A().attention(leaf["q"], leaf["k"], leaf["v"], H, g=leaf["g"], bias=leaf["bias"], mask=a["mask"])
    grads = dict(zip(names, torch.autograd.grad(o, list(leaf.values()), dout)))
    for n in names:
        # along the gradient's own direction, of unit length: the change is its norm, far above the rounding of the sums
        d = grads[n] / grads[n].norm()
        h = 0.02
        diff = (f({**a, n: a[n] + h * d}) - f({**a, n: a[n] - h * d})) / (2 * h)
        assert abs(diff - float(grads[n].norm())) <= 2e-2 * float(grads[n].norm()), n


def test_refuses_gradients_of_gradients_and_changed_inputs():
    a = inputs(1, 1, 1, 2, 16, 9, 9, F32)
    q = a["q"].clone().requires_grad_()
    o = A().attention(q, a["k"], a["v"], 2)
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(o.sum(), q, create_graph=True)
    o = A().attention(q, a["k"], a["v"], 2)
    a["k"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


# -------------------------------------------------------------------------------------------------- together

def chain(x, H, table, add, b, pos, chains, wq, wk, mask, mult):
    """Positions, norms and attention as a training step has them, from the fused projection's rows."""
    q, k, v, g = x.chunk(4, -1)
    qn, kn = A().qk_norm_rope(q, k, wq, wk, H, pos, out_dtype=x.dtype)
    bias = A().rel_bias(table, b, pos, group_q=chains, add=add)
    return A().attention(qn, kn, v, H, g=g, bias=bias, mask=mask, multiplicity=mult)


def chain_inputs(dtype, seed=0):
    S, mult, H, C, N = 4, 2, 4, 24, 70
    b = K().rel_buckets(K().clipped_edges(8), True)
    pos = torch.arange(N, device="cuda") % 40
    args = dict(H=H, b=b, pos=pos, chains=(torch.arange(N, device="cuda") >= 40).long(), mask=torch.ones(S, N, device="cuda"), mult=mult)
    args["mask"][2, 50:] = 0
    leaves = dict(x=rand(seed + 1, S, N, 4 * H * C, dtype=dtype), table=rand(seed + 2, b.count, H),
                  add=rand(seed + 3, S // mult, H, N, N, dtype=dtype), wq=1 + rand(seed + 4, C, scale=0.1), wk=1 + rand(seed + 5, C, scale=0.1))
    return args, leaves, rand(seed + 6, S, N, H * C, scale=0.1, dtype=dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_together(dtype):
    """The three as one step, against the oracle's chain in float64: an fp32 chain to the parts' bounds together, a half one to
    eight half steps of the largest value (every one of its seven roundings on the way to it, and the sum)."""
    args, leaves, dout = chain_inputs(dtype)
    leaves = {n: t.requires_grad_() for n, t in leaves.items()}
    o = chain(**args, **leaves)
    grads = dict(zip(leaves, torch.autograd.grad(o, list(leaves.values()), dout)))
    H, pos, mult = args["H"], args["pos"].cpu().numpy(), args["mult"]
    x, S, N = np64(leaves["x"]), leaves["x"].shape[0], leaves["x"].shape[1]
    W = x.shape[-1] // 4
    q, k, v, g = (x[..., i * W:(i + 1) * W] for i in range(4))
    p = np.tile(pos, S)
    qn, kn = (T.qk_norm_rope(t.reshape(-1, W), np64(leaves[n]), H, p).reshape(S, N, W) for t, n in ((q, "wq"), (k, "wk")))
    at = T.buckets(K().clipped_edges(8), pos, pos, args["chains"].cpu().numpy(), args["chains"].cpu().numpy())
    bias = T.rel_bias(np64(leaves["table"]), at, np64(leaves["add"]))
    want = T.attention(qn, kn, v, H, g, bias, np64(args["mask"]), mult)[0]
    d = T.attention_grads(np64(dout), qn, kn, v, H, g, bias, np64(args["mask"]), mult)
    dq, dwq = T.qk_norm_rope_grads(d["q"].reshape(-1, W), q.reshape(-1, W), np64(leaves["wq"]), H, p)
    dk, dwk = T.qk_norm_rope_grads(d["k"].reshape(-1, W), k.reshape(-1, W), np64(leaves["wk"]), H, p)
    ref = {"x": np.concatenate([dq.reshape(q.shape), dk.reshape(k.shape), d["v"], d["g"]], -1), "wq": dwq, "wk": dwk,
           "table": T.rel_bias_grad(d["bias"], at, args["b"].count), "add": d["bias"]}
    step = STEP[dtype] or 64 * U
    for got, r in [(o, want)] + [(grads[n], ref[n]) for n in ref]:
        assert np.abs(np64(got) - r).max() <= 8 * step * np.abs(r).max()


def test_captured_and_replayed():
    """A step in a HIP graph, replayed several times over changed inputs with eager work between: each replay's bits are the
    eager step's. Two graphs with workspaces of their own alternate."""
    def fresh(seed):
        args, leaves, dout = chain_inputs(BF16, seed)
        return args, {n: t.requires_grad_() for n, t in leaves.items()}, dout

    def step(args, leaves, dout):
        o = chain(**args, **leaves)
        return [o.detach()] + list(torch.autograd.grad(o, list(leaves.values()), dout))

    graphs = []
    for seed in (0, 100):
        args, leaves, dout = fresh(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(args, leaves, dout)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(args, leaves, dout)
        graphs.append((graph, leaves, dout, out, args))
    for turn in range(4):
        for n, (graph, leaves, dout, out, args) in enumerate(graphs):
            new = chain_inputs(BF16, 1000 * turn + n)
            with torch.no_grad():
                for name, t in leaves.items():
                    t.copy_(new[1][name])
                dout.copy_(new[2])
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            want = step(new[0], {k: t.requires_grad_() for k, t in new[1].items()}, new[2])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (turn, n)


def test_few_queries_captured_and_on_streams():
    """One query against a long axis, whose parts meet in a workspace: replays of two graphs in turn with eager calls between,
    two threads at once."""
    import threading

    H, C, M = 3, 40, 9000
    graphs = []
    for seed in (1, 2):
        a = inputs(seed, 2, 1, H, C, 1, M, BF16, mask="tail")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(a, H)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(a, H)
        graphs.append((graph, a, out))
    for turn in range(4):
        for n, (graph, a, out) in enumerate(graphs):
            new = inputs(100 * turn + n, 2, 1, H, C, 1, M, BF16, mask="tail")
            for name in ("q", "k", "v", "g", "bias", "mask"):
                a[name].copy_(new[name])
            graph.replay()
            got = [t.clone() for t in out]
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, call(new, H))), (turn, n)
    data = [inputs(s, 1, 1, H, C, 2, M, F16) for s in (5, 6)]
    want = [call(a, H) for a in data]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = call(data[i], H)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(x, y) for g, w in zip(got, want) for x, y in zip(g, w))


def test_attention_one_row_has_any_pitch():
    """Dimensions of one, whose strides say nothing: one query, one key, one sample; samples that share a query or keys."""
    S, H, C, M = 3, 2, 16, 20
    a = inputs(3, S, 1, H, C, 1, M, F32)
    want = call(a, H)
    odd = dict(a)
    for n in ("q", "g"):
        odd[n] = torch.as_strided(a[n], a[n].shape, (H * C, 2 ** 40, 1))
    assert all(torch.equal(x, y) for x, y in zip(call(odd, H), want))
    dout = rand(9, S, 1, H * C)
    d, dodd = call_bwd(dout, a, H, *want), call_bwd(dout, odd, H, *want)
    assert all(torch.equal(d[n], dodd[n]) for n in d)
    one = inputs(4, 1, 1, H, C, 50, 1, F32, mask=None)
    odd = dict(one)
    for n in ("k", "v"):
        odd[n] = torch.as_strided(one[n], one[n].shape, (2 ** 41, 2 ** 40, 1))
    assert all(torch.equal(x, y) for x, y in zip(call(odd, H), call(one, H)))
    same = dict(a, q=a["q"][:1].expand(S, -1, -1), k=a["k"][:1].expand(S, -1, -1))
    check(same, H)


def test_streams_and_threads():
    """Calls on other streams and from two threads at once: the bits of the calls alone."""
    import threading

    a = [inputs(s, 2, 1, 4, 32, 90, 80, BF16) for s in (1, 2)]
    want = [call(x, 4) for x in a]
    dout = rand(5, 2, 90, 128, dtype=BF16)
    wantd = [call_bwd(dout, x, 4, *w) for x, w in zip(a, want)]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                o = call(a[i], 4)
                got[i] = (o, call_bwd(dout, a[i], 4, *o))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert torch.equal(got[i][0][0], want[i][0]) and all(torch.equal(got[i][1][n], wantd[i][n]) for n in wantd[i])


# -------------------------------------------------------------------------------------------------- modules

def module(seed, c_s, c_z, H, **kw):
    from boltz_mlx_amd.layers.attentionv2 import AttentionPairBias

    m = AttentionPairBias(c_s, c_z, H, **kw).cuda()
    with torch.no_grad():
        for n, p in enumerate(m.parameters()):
            p.copy_(rand(seed + n, *p.shape, scale=0.2) + (1.0 if p.dim() == 1 and n else 0.0))
    return m


def module64(m, s, z, mask, mult, k_in=None, norm=None, rel=None, pos=None, chain=None):
    """AttentionPairBias with positions in torch's float64 operations on the CPU."""
    c = lambda t: t.detach().double().cpu().requires_grad_()  # noqa: E731
    P = {n: c(p) for n, p in m.named_parameters()}
    H, C = m.num_heads, m.head_dim
    B, N, _ = s.shape
    k_in = s if k_in is None else k_in
    lin = torch.nn.functional.linear
    hd = lambda t: t.view(B, -1, H, C).transpose(1, 2)  # noqa: E731
    q, k = hd(lin(s, P["proj_q.weight"], P["proj_q.bias"])), hd(lin(k_in, P["proj_k.weight"]))
    v, g = hd(lin(k_in, P["proj_v.weight"])), lin(s, P["proj_g.weight"])
    if norm is not None:
        P["norm.q_weight"], P["norm.k_weight"] = c(norm.q_weight), c(norm.k_weight)
        a = pos.double().cpu()[:, None] * 10000.0 ** (-torch.arange(0, C, 2, dtype=torch.float64) / C)

        def turned(x, w):
            x = x / (x.square().mean(-1, keepdim=True) + norm.eps).sqrt() * w
            x, y = x[..., :C // 2], x[..., C // 2:]
            return torch.cat([x * a.cos() - y * a.sin(), x * a.sin() + y * a.cos()], -1)

        q, k = turned(q, P["norm.q_weight"]), turned(k, P["norm.k_weight"])
    x = q @ k.transpose(-1, -2).contiguous() / C ** 0.5
    if z is not None:
        zn = torch.nn.functional.layer_norm(z, (z.shape[-1],), P["proj_z.0.weight"], P["proj_z.0.bias"], 1e-5)
        x = x + lin(zn, P["proj_z.1.weight"]).permute(0, 3, 1, 2).repeat_interleave(mult, 0)
    if rel is not None:
        P["rel.table"] = c(rel.table)
        at = T.buckets(K().clipped_edges(5), pos.cpu().numpy(), pos.cpu().numpy(), chain.cpu().numpy(), chain.cpu().numpy())
        x = x + P["rel.table"][torch.tensor(at)].permute(2, 0, 1)
    x = x.masked_fill(mask.cpu()[:, None, None] == 0, -torch.inf)
    o = (x.softmax(-1) @ v).transpose(1, 2).reshape(B, N, -1) * torch.sigmoid(g)
    return lin(o, P["proj_o.weight"]), P


@pytest.mark.parametrize("positions_too", [False, True])
def test_attention_pair_bias_with_grad(positions_too):
    from boltz_mlx_amd.layers.positions import QKNorm, RelativeBias

    B, mult, N, H, C, cz = 4, 2, 37, 3, 24, 16
    m = module(1, H * C, cz, H)
    s, z, mask = rand(50, B, N, H * C).requires_grad_(), rand(51, B // mult, N, N, cz).requires_grad_(), torch.ones(B, N, device="cuda")
    mask[1, 30:] = 0
    pos = torch.arange(N, device="cuda") % 20
    chain = torch.arange(N, device="cuda") // 20
    kw, extra = {}, {}
    if positions_too:
        norm, rel = QKNorm(C).cuda(), RelativeBias(H, edges=K().clipped_edges(5)).cuda()
        with torch.no_grad():
            norm.q_weight.add_(rand(60, C, scale=0.1))
            rel.table.copy_(rand(61, *rel.table.shape, scale=0.3))
        kw = dict(qk_norm=norm, rel_bias=rel, pos=pos, chain=chain)
        extra = dict(norm=norm, rel=rel, pos=pos, chain=chain)
    o = m.with_grad(s, z, mask, multiplicity=mult, **kw)
    dout = rand(52, *o.shape)
    o.backward(dout)
    s64, z64 = (t.detach().double().cpu().requires_grad_() for t in (s, z))
    want, P = module64(m, s64, z64, mask, mult, **extra)
    want.backward(dout.double().cpu())
    got = {n: p.grad for n, p in m.named_parameters()}
    if positions_too:
        got |= {"norm.q_weight": norm.q_weight.grad, "norm.k_weight": norm.k_weight.grad, "rel.table": rel.table.grad}
    pairs = [("out", o, want), ("s", s.grad, s64.grad), ("z", z.grad, z64.grad)] + [(n, got[n], P[n].grad) for n in got]
    for n, a, b in pairs:
        # fp32 throughout: sums of at most 148 * 72 terms of unit-sized products, 2^-24 each, in the products before and after.
        # A LayerNorm bias before proj_z adds one number to all logits of a head, which the softmax does not see: its gradient is
        # 0, a sum of the terms that the weight's gradient has (times a normalised z), so that these say how far rounding goes.
        size = (P["proj_z.0.weight"].grad if n == "proj_z.0.bias" else b).abs().max()
        assert (a.detach().double().cpu() - b).abs().max() <= 400 * U * size, n
    if not positions_too:
        bias = rand(53, B // mult, H, N, N)
        o = m.with_grad(s, None, mask, multiplicity=mult, pair_bias=bias)
        fwd = m(s.detach(), None, mask, s.detach(), multiplicity=mult, pair_bias=bias)
        assert (fwd - o).abs().max() <= 400 * U * o.abs().max()
        other = m.with_grad(s, None, mask, k_in=s.detach().clone(), multiplicity=mult, pair_bias=bias)
        assert (other - o).abs().max() <= 400 * U * o.abs().max()


def test_modules_in_half_types_and_batches():
    from boltz_mlx_amd.layers.positions import QKNorm, RelativeBias

    B, N, H, C = 2, 20, 2, 16
    m = module(3, H * C, None, H, compute_pair_bias=False)
    norm, rel = QKNorm(C, rotary=8, interleaved=True).cuda(), RelativeBias(H, 4).cuda()
    pos = torch.stack([torch.arange(N, device="cuda"), torch.arange(N, device="cuda") * 2])
    mask = torch.ones(B, N, device="cuda")
    s = rand(5, B, N, H * C)
    with torch.no_grad():
        want = m.with_grad(s, None, mask, qk_norm=norm, rel_bias=rel, pos=pos, chain=pos // 9)
        for t in (F16, BF16):
            got = m.with_grad(s.to(t), None, mask, qk_norm=norm, rel_bias=rel, pos=pos, chain=pos // 9)
            # a dozen roundings on the way, each of at most a half step of the largest value
            assert got.dtype == t and (got.float() - want).abs().max() <= 16 * STEP[t] * want.abs().max()
    assert set(rel.state_dict()) == {"table"} and set(norm.state_dict()) == {"q_weight", "k_weight"}
    bias = rel(pos[0])
    assert bias.shape == (H, N, N) and bias.requires_grad and (bias == 0).all()
