"""Refusals of the sequence attention's training form: every argument is checked on the host before a launch. No device calls:
the C entry points are given host addresses, which they must refuse before they could use them."""

from __future__ import annotations

import ctypes

import pytest
import torch

from boltz_mlx_amd import _lib
from boltz_mlx_amd import autograd as A
from boltz_mlx_amd import kernels as K

HOST = ctypes.create_string_buffer(1 << 20)
P = (ctypes.addressof(HOST) + 63) // 64 * 64  # aligned addresses that no launch may see, 32 KiB apart
AT = [P + (i << 15) for i in range(30)]
F32, F16, BF16 = 0, 1, 2


def rc(name, args, change):
    unknown = set(change) - set(args)
    assert not unknown, unknown
    code = getattr(_lib.load(), name)(*{**args, **change}.values())
    if code:
        assert name.encode() in _lib.load().bzpf_last_error()
    return code


REL = dict(table=AT[0], lut=AT[1], lo=-3, span=7, count=8, pos_q=AT[2], pos_k=AT[3], group_q=AT[4], group_k=AT[5], wide=1, batch_q=4,
           batch_k=6, add=AT[6], out=AT[7], dt=F16, B=2, H=3, N=4, M=6, stream=None)


@pytest.mark.parametrize("change", [
    {"table": None}, {"lut": None}, {"pos_q": None}, {"pos_k": None}, {"out": None}, {"group_q": None}, {"group_k": None},
    {"table": AT[0] + 2}, {"out": AT[7] + 1}, {"add": AT[6] + 1}, {"pos_q": AT[2] + 4}, {"wide": 0, "pos_k": AT[3] + 2},
    {"dt": 3}, {"dt": -1}, {"count": 0}, {"count": 257}, {"span": 0}, {"span": 16385}, {"lo": 2 ** 62}, {"lo": -2 ** 62},
    {"B": -1}, {"B": 65536}, {"H": 0}, {"H": 65536}, {"N": -1}, {"M": -1}, {"N": 2 ** 31}, {"H": 65535, "N": 2 ** 30, "M": 2 ** 30},
    {"batch_q": 3}, {"batch_k": 5}, {"batch_q": -4}, {"batch_q": 2 ** 60}, {"out": AT[6]}, {"out": AT[6] + 100}, {"out": AT[1] - 8},
    {"out": AT[2] + 40},
])
def test_rel_bias_refuses(change):
    assert rc("bzpf_rel_bias", REL, change) == -1


def test_rel_bias_takes_no_pairs():
    for change in ({"N": 0}, {"M": 0}, {"B": 0}):
        assert rc("bzpf_rel_bias", {**REL, "table": None, "out": None, "pos_q": None}, change) == 0


REL_BWD = dict(dout=AT[0], dt=F32, lut=AT[1], lo=-3, span=7, count=8, pos_q=AT[2], pos_k=AT[3], group_q=None, group_k=None, wide=0,
               batch_q=0, batch_k=0, dtable=AT[4], ws=AT[5], ws_bytes=1 << 15, B=1, H=3, N=40, M=60, stream=None)


@pytest.mark.parametrize("change", [
    {"dout": None}, {"dout": AT[0] + 2}, {"dtable": None}, {"ws": None}, {"dtable": AT[4] + 1}, {"ws_bytes": 4}, {"dt": 4},
    {"B": 0}, {"N": 0}, {"M": 0}, {"count": 300}, {"group_q": AT[6]}, {"dtable": AT[0] + 28000}, {"ws": AT[4]}, {"ws": AT[0]}, {"B": 65535, "H": 17, "N": 1, "M": 1, "ws_bytes": 1 << 40},
])
def test_rel_bias_bwd_refuses(change):
    assert rc("bzpf_rel_bias_bwd", REL_BWD, change) == -1


QK = dict(q=AT[0], ldq=64, k=AT[1], ldk=32, x_dt=F16, w_q=AT[2], w_k=AT[3], eps=1e-5, pos=AT[4], wide=1, pos_rows=5, base=1e4, rotary=16,
          interleaved=0, qn=AT[5], kn=AT[6], y_dt=F16, rows=5, H=4, Hk=2, C=16, stream=None)


@pytest.mark.parametrize("change", [
    {"q": None}, {"k": None}, {"qn": None}, {"kn": None}, {"q": AT[0] + 1}, {"w_q": AT[2] + 2}, {"pos": AT[4] + 4}, {"kn": AT[6] + 1},
    {"x_dt": BF16}, {"y_dt": 5}, {"x_dt": -1}, {"C": 0}, {"C": 15}, {"C": 258}, {"rotary": 18}, {"rotary": -2}, {"rotary": 7},
    {"H": 0}, {"Hk": 0}, {"H": 1025}, {"rows": -1}, {"ldq": 63}, {"ldk": 31}, {"pos_rows": 0}, {"base": 0.0}, {"base": -1.0},
    {"base": float("inf")}, {"base": float("nan")}, {"ldq": 2 ** 61}, {"rows": 2 ** 60}, {"qn": AT[0]}, {"kn": AT[5]}, {"kn": AT[4] + 8},
    {"qn": AT[2] - 4}, {"qn": AT[0] + 600},
])
def test_qk_norm_rope_refuses(change):
    assert rc("bzpf_qk_norm_rope", QK, change) == -1


QK_BWD = dict(dqn=AT[0], dkn=AT[1], y_dt=F32, q=AT[2], ldq=64, k=AT[3], ldk=32, x_dt=BF16, w_q=AT[4], w_k=AT[5], eps=1e-5, pos=None,
              wide=0, pos_rows=0, base=1e4, rotary=16, interleaved=1, dq=AT[6], dk=AT[7], dw_q=AT[8], dw_k=AT[9], ws=AT[10],
              ws_bytes=1 << 16, rows=5, H=4, Hk=2, C=16, stream=None)


@pytest.mark.parametrize("change", [
    {"dqn": None}, {"dkn": None}, {"dq": None}, {"dk": None}, {"q": None}, {"ws": None}, {"ws_bytes": 1000}, {"dq": AT[6] + 1},
    {"dw_q": AT[8] + 2}, {"ws": AT[10] + 2}, {"rows": 0}, {"C": 3}, {"dq": AT[2]}, {"dk": AT[6] + 64}, {"dw_k": AT[8]}, {"dw_q": AT[4]},
    {"ws": AT[9]}, {"y_dt": F16},
])
def test_qk_norm_rope_bwd_refuses(change):
    assert rc("bzpf_qk_norm_rope_bwd", QK_BWD, change) == -1


ATT = dict(q=AT[0], ldq=48, sq=240, k=AT[1], ldk=48, sk=336, v=AT[2], ldv=48, sv=336, g=AT[3], ldg=48, sg=240, bias=AT[4], bias_dt=F16,
           mult=2, mask=AT[5], out=AT[6], stats=AT[7], ws=None, ws_bytes=0, dt=F16, S=2, H=3, C=16, N=5, M=7, stream=None)


@pytest.mark.parametrize("change", [
    {"q": None}, {"k": None}, {"v": None}, {"out": None}, {"stats": None}, {"q": AT[0] + 1}, {"k": AT[1] + 1}, {"v": AT[2] + 1},
    {"g": AT[3] + 1}, {"bias": AT[4] + 1}, {"mask": AT[5] + 2}, {"out": AT[6] + 1}, {"stats": AT[7] + 2}, {"dt": 3}, {"bias_dt": F32},
    {"bias_dt": BF16}, {"dt": F32, "bias_dt": 7}, {"C": 0}, {"C": 12}, {"C": 136}, {"H": 0}, {"S": 0}, {"mult": 0}, {"mult": 3}, {"N": 0},
    {"M": 0}, {"N": -1}, {"N": 2 ** 22 + 1}, {"M": 2 ** 22 + 1}, {"ldq": 47}, {"ldk": 40}, {"ldv": 0}, {"ldg": 1}, {"sq": -1}, {"sv": -8},
    {"sk": 2 ** 62}, {"ldk": 2 ** 23}, {"ldg": 2 ** 60}, {"out": AT[0]}, {"out": AT[1] + 600}, {"out": AT[4]}, {"stats": AT[6]}, {"stats": AT[5]},
    {"out": AT[3] + 900}, {"ws": AT[8] + 8}, {"ws_bytes": -1},
    {"S": 2 ** 20, "H": 16, "sq": 0, "sk": 0, "sv": 0, "sg": 0}, {"N": 2 ** 22, "H": 129, "C": 8, "S": 4, "mult": 4}, {"M": 2 ** 22, "S": 128},
])
def test_attention_refuses(change):
    assert rc("bzpf_attention", ATT, change) == -1


@pytest.mark.parametrize("ws, size, what", [(None, 1 << 40, "ws holds 0"), (1 << 40, 1000, "ws holds 1000"),
                                            ((1 << 40) + 4, 1 << 40, "16-byte"), (1 << 44, 1 << 40, "overlaps")])
def test_attention_refuses_workspaces(ws, size, what):
    """One query against a long axis, whose parts meet in the workspace."""
    few = dict(q=1 << 41, k=1 << 42, sk=0, v=1 << 43, sv=0, g=None, bias=None, mult=1, mask=None, out=1 << 44, stats=1 << 45, S=1, N=1, M=50001)
    assert _lib.load().bzpf_attention_ws(1, 3, 16, 1, 50001) > 1000
    assert rc("bzpf_attention", ATT, dict(few, ws=ws, ws_bytes=size)) == -1
    assert what in _lib.load().bzpf_last_error().decode()


ATT_BWD = dict(dout=AT[8], q=AT[0], ldq=48, sq=240, k=AT[1], ldk=48, sk=336, v=AT[2], ldv=48, sv=336, g=AT[3], ldg=48, sg=240,
               bias=AT[4], bias_dt=F16, mult=2, mask=AT[5], out=AT[6], stats=AT[7], dq=AT[9], dk=AT[10], dv=AT[11], dg=AT[12],
               dbias=AT[13], ws=AT[14], ws_bytes=1 << 15, dt=F16, S=2, H=3, C=16, N=5, M=7, stream=None)


@pytest.mark.parametrize("change", [
    {"dout": None}, {"dq": None}, {"dk": None}, {"dv": None}, {"dg": None}, {"ws": None}, {"g": None}, {"bias": None}, {"dq": AT[9] + 1},
    {"dbias": AT[13] + 1}, {"ws": AT[14] + 8}, {"ws_bytes": 100}, {"dq": AT[0]}, {"dk": AT[1]}, {"dv": AT[10]}, {"dg": AT[3] + 2},
    {"dbias": AT[4]}, {"ws": AT[7]}, {"dq": AT[8] + 500}, {"dt": BF16}, {"C": 4}, {"M": 0},
])
def test_attention_bwd_refuses(change):
    assert rc("bzpf_attention_bwd", ATT_BWD, change) == -1


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.bzpf_attention_bwd_ws(F32, 2, 3, 16, 5, 7, 0) >= 2 * 3 * 5 * 4
    assert lib.bzpf_attention_bwd_ws(F32, 2, 3, 16, 5, 7, 1) >= 2 * 3 * 5 * 4 + 2 * 3 * 5 * 16 * 4
    for bad in ((3, 2, 3, 16, 5, 7, 0), (F32, 0, 3, 16, 5, 7, 0), (F32, 2, 3, 12, 5, 7, 0), (F32, 2, 3, 16, 0, 7, 0), (F32, 2, 3, 136, 5, 7, 1)):
        assert lib.bzpf_attention_bwd_ws(*bad) == -1
    assert lib.bzpf_attention_ws(20, 3, 16, 5, 10000) == lib.bzpf_attention_ws(1, 1, 16, 1, 1) == 0 < lib.bzpf_attention_ws(2, 3, 16, 5, 10000)
    for bad in ((0, 3, 16, 5, 7), (2, 0, 16, 5, 7), (2, 3, 20, 5, 7), (2, 3, 16, 0, 7), (2, 3, 16, 5, (1 << 22) + 1)):
        assert lib.bzpf_attention_ws(*bad) == -1
    assert lib.bzpf_rel_bias_bwd_ws(1, 16, 400, 400, 66) > 0 and lib.bzpf_qk_norm_rope_bwd_ws(24) > 0
    assert lib.bzpf_rel_bias_bwd_ws(1, 16, 400, 400, 0) == lib.bzpf_rel_bias_bwd_ws(0, 1, 1, 1, 1) == -1
    assert lib.bzpf_qk_norm_rope_bwd_ws(25) == lib.bzpf_qk_norm_rope_bwd_ws(258) == -1


def refused(kind, what, call):
    with pytest.raises(kind, match=what):
        call()


def test_rel_bias_wrappers_refuse():
    b = K.rel_buckets(K.clipped_edges(3), True, device="cpu")
    t, pos = torch.zeros(8, 4), torch.arange(6)
    batch = torch.zeros(2, 6, dtype=torch.int64)
    for what, call in [
        ("table must be", lambda: K.rel_bias(t[:7], b, pos)), ("table must be", lambda: K.rel_bias(t[0], b, pos)),
        ("one integer type", lambda: K.rel_bias(t, b, pos.float())), ("one integer type", lambda: K.rel_bias(t, b, pos, pos.int())),
        ("one integer type", lambda: K.rel_bias(t, b, pos, group_q=pos.int())), ("positions must be", lambda: K.rel_bias(t, b, pos[0])),
        ("positions must be", lambda: K.rel_bias(t, b, batch[None])), ("different batch sizes", lambda: K.rel_bias(t, b, batch, batch[:1])),
        ("queries and keys, or for neither", lambda: K.rel_bias(t, b, pos, pos, pos)),
        ("their positions' shapes", lambda: K.rel_bias(t, b, pos, group_q=pos[:5])),
        ("add must be", lambda: K.rel_bias(t, b, pos, add=torch.zeros(4, 6, 5))), ("add must be", lambda: K.rel_bias(t, b, batch, add=torch.zeros(4, 6, 6))),
        ("heads and the output's type", lambda: K.rel_bias(t, b, pos, add=torch.zeros(3, 6, 6))),
        ("heads and the output's type", lambda: K.rel_bias(t, b, pos, add=torch.zeros(4, 6, 6), out_dtype=torch.half)),
        ("dbias must be", lambda: K.rel_bias_bwd(torch.zeros(4, 6, 5), b, pos)), ("rel_buckets", lambda: K.rel_bias(t, b._replace(lut=b.lut.int()), pos)),
        ("ROCm device", lambda: K.rel_bias(t, b, pos)), ("ROCm device", lambda: A.rel_bias(t, b, pos)),
        ("ROCm device", lambda: K.rel_bias_bwd(torch.zeros(4, 6, 6), b, pos)),
    ]:
        refused(ValueError, what, call)
    for call in (lambda: K.rel_bias(t.double(), b, pos), lambda: K.rel_bias(t, b, pos, out_dtype=torch.int32)):
        refused(TypeError, "unsupported dtype", call)


def test_qk_norm_rope_wrappers_refuse():
    q, k, w, pos = torch.zeros(2, 5, 64), torch.zeros(2, 5, 32), torch.ones(16), torch.arange(5)
    for what, call in [
        ("need q", lambda: K.qk_norm_rope(q, k, w, w, 3)), ("need q", lambda: K.qk_norm_rope(q, k, w, w, 0)), ("need q", lambda: K.qk_norm_rope(q, k[0], w, w, 4)),
        ("even 2 to 256", lambda: K.qk_norm_rope(q, q, None, None, 64)), ("even 2 to 256", lambda: K.qk_norm_rope(torch.zeros(1, 258), torch.zeros(1, 258), None, None, 1)),
        ("q's rows", lambda: K.qk_norm_rope(q, k[:, :4], w, w, 4)), ("q's rows", lambda: K.qk_norm_rope(q, k[..., :24], w, w, 4)),
        ("one type on one device", lambda: K.qk_norm_rope(q, k.half(), w, w, 4)), ("weights must be", lambda: K.qk_norm_rope(q, k, w[:8], w, 4)),
        ("weights must be", lambda: K.qk_norm_rope(q, k, w, w[None], 4)), ("rotary must be", lambda: K.qk_norm_rope(q, k, w, w, 4, pos, rotary=18)),
        ("rotary must be", lambda: K.qk_norm_rope(q, k, w, w, 4, pos, rotary=3)), ("base must be", lambda: K.qk_norm_rope(q, k, w, w, 4, pos, base=0.0)),
        ("pos must hold", lambda: K.qk_norm_rope(q, k, w, w, 4, pos[:4])), ("pos must hold", lambda: K.qk_norm_rope(q, k, w, w, 4, pos.float())),
        ("pos must hold", lambda: K.qk_norm_rope(q, k, w, w, 4, pos[None])), ("shapes of q and k", lambda: K.qk_norm_rope_bwd(q, q, q, k, w, w, 4)),
        ("shapes of q and k", lambda: K.qk_norm_rope_bwd(q, k.half(), q, k, w, w, 4)), ("ROCm device", lambda: K.qk_norm_rope(q, k, w, w, 4, pos)),
        ("ROCm device", lambda: A.qk_norm_rope(q, k, w, w, 4, pos)), ("ROCm device", lambda: K.qk_norm_rope_bwd(q, k, q, k, w, w, 4)),
    ]:
        refused(ValueError, what, call)
    refused(TypeError, "unsupported dtype", lambda: K.qk_norm_rope(q.double(), k.double(), None, None, 4))


def test_attention_wrappers_refuse():
    q, k, bias, mask = torch.zeros(4, 5, 32), torch.zeros(4, 6, 32), torch.zeros(2, 2, 5, 6), torch.ones(4, 6)
    o, st = torch.zeros(4, 5, 32), torch.zeros(4, 2, 5, 2)
    for what, call in [
        ("need q", lambda: K.attention(q, k, k[:, :5], 2)), ("need q", lambda: K.attention(q, k, k, 3)), ("need q", lambda: K.attention(q, k[0], k[0], 2)),
        ("need q", lambda: K.attention(q, k[:3], k[:3], 2)), ("need q", lambda: K.attention(q, k[..., :16], k[..., :16], 2)), ("need q", lambda: K.attention(q, k, k, 0)),
        ("8 to 128 channels", lambda: K.attention(q, k, k, 8)), ("8 to 128 channels", lambda: K.attention(torch.zeros(1, 1, 136), torch.zeros(1, 1, 136), torch.zeros(1, 1, 136), 1)),
        ("q's shape", lambda: K.attention(q, k, k, 2, g=k)), ("one type on one device", lambda: K.attention(q, k, k.half(), 2)),
        ("one type on one device", lambda: K.attention(q, k, k, 2, g=q.half())), ("multiplicity", lambda: K.attention(q, k, k, 2, multiplicity=3)),
        ("multiplicity", lambda: K.attention(q, k, k, 2, multiplicity=0)), ("bias must be", lambda: K.attention(q, k, k, 2, bias=bias)),
        ("bias must be", lambda: K.attention(q, k, k, 2, bias=bias[:1], multiplicity=2)), ("bias must be", lambda: K.attention(q, k, k, 2, bias=bias[0], multiplicity=2)),
        ("bias must be", lambda: K.attention(q, k, k, 2, bias=bias[..., :5], multiplicity=2)), ("mask must be", lambda: K.attention(q, k, k, 2, mask=mask[:, :5])),
        ("mask must be", lambda: K.attention(q, k, k, 2, mask=mask.bool())), ("mask must be", lambda: K.attention(q, k, k, 2, mask=mask.view(-1))),
        ("dout and out", lambda: K.attention_bwd(o[:, :4], q, k, k, 2, o, st)), ("dout and out", lambda: K.attention_bwd(o.half(), q, k, k, 2, o, st)),
        ("stats must be", lambda: K.attention_bwd(o, q, k, k, 2, o, st[..., :1])), ("ROCm device", lambda: K.attention(q, k, k, 2)),
        ("ROCm device", lambda: A.attention(q, k, k, 2)), ("ROCm device", lambda: K.attention_bwd(o, q, k, k, 2, o, st)),
    ]:
        refused(ValueError, what, call)
    for call in (lambda: K.attention(q.half(), k.half(), k.half(), 2, bias=bias, multiplicity=2),
                 lambda: K.attention(q, k, k, 2, bias=bias.double(), multiplicity=2), lambda: K.attention(q.double(), k.double(), k.double(), 2)):
        refused(TypeError, "bias must be of|unsupported dtype", call)
