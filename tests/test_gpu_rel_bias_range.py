"""The position bias where positions, their distances and the buckets' borders are as large as they may be: positions and the
lowest distance below 2^62 in size, so that distances take 63 bits and their distance from the border 64. Tolerances are those of
test_gpu_attention.py."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attention as T  # noqa: E402
from test_gpu_attention import F16, F32, BF16, K, U, close, grad_depth, np64, rand  # noqa: E402

pytestmark = pytest.mark.gpu

MOST = 2 ** 62 - 1


def check(edges, pq, pk, dtype, groups=None):
    H, N, M = 3, len(pq), len(pk)
    b = K().rel_buckets(edges, groups is not None)
    pq, pk = (torch.tensor(p, dtype=torch.int64, device="cuda") for p in (pq, pk))
    cq, ck = (None, None) if groups is None else (torch.tensor(g, device="cuda") for g in groups)
    at = T.buckets(edges, pq.cpu().numpy(), pk.cpu().numpy(), *([] if groups is None else [np.array(g) for g in groups]))
    table, dy = rand(1, b.count, H, dtype=dtype), rand(2, H, N, M, dtype=dtype)
    same = np.array_equal(np64(K().rel_bias(table, b, pq, pk, cq, ck)), T.rel_bias(np64(table), at))
    assert same
    close(K().rel_bias_bwd(dy, b, pq, pk, cq, ck), T.rel_bias_grad(np64(dy), at, b.count),
          grad_depth(1, H, N, M) * U * T.rel_bias_grad(np.abs(np64(dy)), at, b.count))
    return at


EDGES = {"clip32": list(range(-31, 33)), "low": [3 - MOST, 5 - MOST, 40 - MOST], "high": [MOST - 40, MOST - 5, MOST - 1], "one": [0],
         "many": list(range(MOST - 120, MOST - 20))}


@pytest.mark.parametrize("edges", EDGES)
@pytest.mark.parametrize("M", [5, 24, 77])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rel_bias_ends_of_the_positions(edges, M, dtype):
    """Keys together at one end, in the middle, or each far from its neighbours; queries at both ends and between."""
    span = [-MOST, -MOST + 7, -2 ** 61, -40, 0, 31, 2 ** 61, MOST - 7, MOST]
    pq = [span[i % 9] for i in range(70)]
    for first in (-MOST, -2 ** 61 - 20, -30, 2 ** 61, MOST - M):
        check(EDGES[edges], pq, [first + i for i in range(M)], dtype)
    check(EDGES[edges], pq, [span[(5 * i + 2) % 9] for i in range(M)], dtype)
    check(EDGES[edges], pq, [MOST - i for i in range(M)], dtype, groups=([i // 40 for i in range(70)], [i // 17 for i in range(M)]))


@pytest.mark.parametrize("N, M", [(40, 8), (70, 130), (40, 3)])
def test_rel_bias_borders_far_from_zero(N, M):
    """Distances across borders that are themselves almost 2^62."""
    for sign, edges in ((1, "high"), (1, "many"), (-1, "low")):
        pq, pk = [sign * (2 ** 61 + i) for i in range(N)], [-sign * (2 ** 61 - 1) - sign * (i % 60) + sign * 40 for i in range(M)]
        at = check(EDGES[edges], pq, pk, F32)
        assert len(np.unique(at)) > 1


@pytest.mark.parametrize("value", [float(np.finfo(np.float32).max), -3.395e38, 3e38, 2.0 ** -126, 1.5 * 2.0 ** -130])
@pytest.mark.parametrize("M", [5, 40])
def test_rel_bias_gradient_of_the_largest_and_smallest_numbers(value, M):
    """One gradient in each bucket that is as large (or as small) as fp32 has them: the table's gradient is itself. Numbers below
    2^-126 + 16 bits may lose what lies below bf16's smallest, 2^-133, in each of three parts."""
    b = K().rel_buckets(list(range(-6, 8)))
    pos = torch.arange(30, device="cuda")
    dy = torch.zeros(2, 30, M, device="cuda")
    want = np.zeros((b.count, 2))
    for h in range(2):
        for bucket in range(b.count):
            j = (12 if M > 20 else 2) + (0 if h else 2)
            i = j + bucket - 7  # the pair of the bucket's distance
            if 0 <= i < 30:
                dy[h, i, j] = value
                want[bucket, h] = np.float32(value)
    got = np64(K().rel_bias_bwd(dy, b, pos, torch.arange(M, device="cuda")))
    assert np.abs(got - want).max() <= (0 if abs(value) > 1 else 3 * 2.0 ** -133)
