"""Refusals of the training operators: every argument is checked on the host before a launch. No device calls: the C entry
points are given host addresses, which they must refuse before they could use them."""

from __future__ import annotations

import ctypes

import pytest
import torch

from boltz_mlx_amd import _lib
from boltz_mlx_amd import autograd as A
from boltz_mlx_amd import kernels as K

HOST = ctypes.create_string_buffer(4096)
P = (ctypes.addressof(HOST) + 63) // 64 * 64  # an aligned address that no launch may see
F32, F16, BF16 = 0, 1, 2


def rc(name, *args):
    return getattr(_lib.load(), name)(*args)


def ln_bwd(dy=P, dy_dt=F32, x=P, x_dt=F32, w=P, dx=P, dw=P, db=P, ws=P, ws_bytes=1 << 30, rows=8, D=128):
    return rc("bzpf_layernorm_bwd", dy, dy_dt, x, x_dt, w, 1e-5, dx, dw, db, ws, ws_bytes, rows, D, None)


def drop(x=P, x_dt=F32, p=0.5, rng=P, site=0, shared=0, I=1, J=1, y=P, y_dt=F32, rows=12, D=16):
    return rc("bzpf_dropout", x, x_dt, p, rng, site, shared, I, J, y, y_dt, rows, D, None)


def res(z=P, y=P, y_dt=F32, p=0.5, rng=P, site=0, shared=0, I=1, J=1, w=P, b=P, zn=P, ln=P, ln_dt=F32, rows=12, D=16):
    return rc("bzpf_dropout_add_ln", z, y, y_dt, p, rng, site, shared, I, J, w, b, 1e-5, zn, ln, ln_dt, rows, D, None)


def res_bwd(dzn=P, dln=P, ln_dt=F32, zn=P, w=P, p=0.5, rng=P, site=0, shared=0, I=1, J=1, dz=P, dy=P, y_dt=F32, dw=P,
            db=P, ws=P, ws_bytes=1 << 30, rows=12, D=16):
    return rc("bzpf_dropout_add_ln_bwd", dzn, dln, ln_dt, zn, w, 1e-5, p, rng, site, shared, I, J, dz, dy, y_dt, dw, db,
              ws, ws_bytes, rows, D, None)


@pytest.mark.parametrize("change", [
    {"dy": None}, {"x": None}, {"dx": None}, {"x": P + 2}, {"dw": P + 2}, {"ws": P + 1}, {"dy_dt": F16, "dy": P + 1},
    {"dy_dt": 3}, {"x_dt": -1}, {"x_dt": F16, "dy_dt": BF16}, {"D": 7}, {"D": 0}, {"D": -8}, {"D": 8193}, {"rows": 0},
    {"rows": -1}, {"rows": 100000, "ws": None}, {"rows": 100000, "ws_bytes": 64},
])
def test_layernorm_bwd_refuses(change):
    assert ln_bwd(**change) == -1
    assert b"bzpf_layernorm_bwd" in _lib.load().bzpf_last_error()


@pytest.mark.parametrize("change", [
    {"x": None}, {"y": None}, {"x": P + 1}, {"x_dt": F16, "y_dt": BF16}, {"x_dt": 7}, {"p": -0.1}, {"p": 1.5},
    {"p": float("nan")}, {"rng": None}, {"rng": P + 4}, {"site": -1}, {"site": 65536}, {"shared": 3}, {"shared": -1},
    {"shared": 1, "I": 5, "J": 2}, {"shared": 1, "I": 0, "J": 1}, {"shared": 2, "I": 4, "J": 5}, {"rows": -1}, {"D": 0},
    {"rows": 1 << 48, "D": 5},
])
def test_dropout_refuses(change):
    assert drop(**change) == -1
    assert b"bzpf_dropout" in _lib.load().bzpf_last_error()


@pytest.mark.parametrize("change", [
    {"z": None}, {"y": None}, {"zn": None}, {"ln": None}, {"z": P + 2}, {"w": P + 2}, {"y_dt": F16, "ln_dt": BF16},
    {"y_dt": 4}, {"D": 7}, {"D": 8193}, {"rows": -1}, {"p": 2.0}, {"rng": None}, {"shared": 1, "I": 3, "J": 8},
])
def test_dropout_add_ln_refuses(change):
    assert res(**change) == -1
    assert b"bzpf_dropout_add_ln" in _lib.load().bzpf_last_error()


@pytest.mark.parametrize("change", [
    {"dzn": P + 2}, {"dln": None}, {"zn": None}, {"dz": None}, {"dy": None}, {"y_dt": F16, "ln_dt": BF16}, {"D": 4},
    {"D": 8200}, {"rows": 0}, {"p": -1.0}, {"rng": None}, {"site": 70000}, {"rows": 100000, "ws_bytes": 4},
    {"rows": 100000, "ws": None},
])
def test_dropout_add_ln_bwd_refuses(change):
    assert res_bwd(**change) == -1
    assert b"bzpf_dropout_add_ln_bwd" in _lib.load().bzpf_last_error()


def test_layernorm_refuses_and_takes_no_rows():
    call = lambda **k: rc("bzpf_layernorm", *{**dict(x=P, xd=F32, w=P, b=P, eps=1e-5, y=P, yd=F32, rows=4, D=128,  # noqa: E731
                                                     st=None), **k}.values())
    for change in ({"x": None}, {"y": None}, {"xd": 3}, {"xd": F16, "yd": BF16}, {"D": 7}, {"D": 8193}, {"rows": -1},
                   {"w": P + 2}, {"x": P + 1}):
        assert call(**change) == -1, change
    assert call(rows=0, x=None, y=None) == 0
    assert drop(rows=0, x=None, y=None, rng=None) == 0
    assert res(rows=0, z=None, y=None) == 0


def test_workspace_sizes():
    ws = _lib.load().bzpf_layernorm_bwd_ws
    assert ws(1, 128) == 0 and ws(0, 128) == 0  # one workgroup writes the gradients itself
    assert ws(-1, 128) == -1 and ws(10, 7) == -1 and ws(10, 8193) == -1
    for rows, D in ((10 ** 6, 128), (10 ** 6, 8192), (5000, 77), (2 ** 40, 8)):
        n = ws(rows, D)
        assert n > 0 and n % (8 * D) == 0 and n // (8 * D) <= 1024  # whole [2][D] of fp32, at most 1024 workgroups


def refused(kind, what, call):
    with pytest.raises(kind, match=what):
        call()


def test_wrappers_refuse():
    """What the wrappers say to each wrong argument (they look at devices last, so that this needs none)."""
    x, w, rng = torch.zeros(2, 3, 4, 16), torch.ones(16), torch.zeros(2, dtype=torch.int64)
    shape, param, prob = "one shape on one device", "weight and bias must be", "p must lie"
    state, width, fp32 = "rng must be an int64", "8 to 8192 channels", "must be fp32"
    for what, call in [
        (shape, lambda: K.layer_norm_bwd(x[0], x, w)), (param, lambda: K.layer_norm_bwd(x, x, torch.ones(17))),
        ("one-dimensional", lambda: A.layer_norm(x, w[None])), (width, lambda: K.layer_norm_bwd(x[..., :7], x[..., :7], None)),
        (width, lambda: K.layer_norm_bwd(torch.zeros(2, 8193), torch.zeros(2, 8193), None)),
        ("rows of channels", lambda: K.layer_norm_bwd(torch.zeros(3, 0), torch.zeros(3, 0), None)),
        ("rows of channels", lambda: K.layer_norm_bwd(torch.tensor(1.0), torch.tensor(1.0), None)),
        (prob, lambda: K.dropout(x, 1.5, rng)), (prob, lambda: K.dropout(x, -0.5, rng)),
        (prob, lambda: K.dropout(x, float("nan"), rng)), (state, lambda: K.dropout(x, 0.5, None)),
        (state, lambda: K.dropout(x, 0.5, rng.int())), (state, lambda: K.dropout(x, 0.5, rng[:1])),
        (state, lambda: K.dropout(x, 0.5, torch.zeros(4, dtype=torch.int64)[::2])),
        ("site must lie", lambda: K.dropout(x, 0.5, rng, site=65536)), ("site must lie", lambda: K.dropout(x, 0.5, rng, -1)),
        ("shared must be", lambda: K.dropout(x, 0.5, rng, shared="rows")),
        ("rows or columns", lambda: K.dropout(x[0, 0], 0.5, rng, shared="row")),
        (fp32, lambda: K.dropout_add_ln(x.half(), x, w, w, 1e-5, 0.5, rng)),
        (shape, lambda: K.dropout_add_ln(x, x[0], w, w, 1e-5, 0.5, rng)),
        (param, lambda: K.dropout_add_ln(x, x, w[:3], w, 1e-5, 0.5, rng)),
        (param, lambda: K.dropout_add_ln(x, x, w, w[:3], 1e-5, 0.5, rng)),
        ("shared must be", lambda: K.dropout_add_ln(x, x, w, w, 1e-5, 0.5, rng, 0, "both")),
        (width, lambda: K.dropout_add_ln(x[..., :5], x[..., :5], None, None, 1e-5, 0.0, None)),
        (shape, lambda: K.dropout_add_ln_bwd(x[0], x, x, w, 1e-5, 0.5, rng)),
        (shape, lambda: K.dropout_add_ln_bwd(None, x[0], x, w, 1e-5, 0.5, rng)),
        (fp32, lambda: K.dropout_add_ln_bwd(x.half(), x, x, w, 1e-5, 0.5, rng)),
        (fp32, lambda: K.dropout_add_ln_bwd(x, x, x.half(), w, 1e-5, 0.5, rng)),
        (shape, lambda: A.dropout_add_ln(x, x[0], w, w)), (prob, lambda: A.dropout(x, 2.0, rng)),
        (param, lambda: A.layer_norm(x, w[:4])),
    ]:
        refused(ValueError, what, call)
    for call in (lambda: K.layer_norm_bwd(x, x.double(), w), lambda: K.dropout(x.long(), 0.5, rng),
                 lambda: K.dropout(x, 0.5, rng, out_dtype=torch.float64), lambda: A.layer_norm(x, w, w, out_dtype=torch.int8)):
        refused(TypeError, "unsupported dtype", call)


def test_layer_norm_refuses():
    x, w = torch.zeros(3, 16), torch.ones(16)
    refused(ValueError, "weight and bias", lambda: K.layer_norm(x, w[:15], None))
    refused(ValueError, "weight and bias", lambda: K.layer_norm(x, w, w[:, None].expand(16, 2)))
    refused(ValueError, "rows of channels", lambda: K.layer_norm(x[:, :0], None, None))
    refused(ValueError, "rows of channels", lambda: K.layer_norm(x[0, 0], None, None))
    refused(ValueError, "8 to 8192", lambda: K.layer_norm(x[:, :7], None, None))
    refused(TypeError, "unsupported dtype", lambda: K.layer_norm(x, w, w, out_dtype=torch.float64))


def test_cpu_tensors_are_refused():
    x, rng = torch.zeros(4, 16), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: K.layer_norm_bwd(x, x, None), lambda: K.dropout(x, 0.5, rng),
                 lambda: K.dropout_add_ln(x, x, None, None, 1e-5, 0.0, None),
                 lambda: K.dropout_add_ln_bwd(x, x, x, None, 1e-5, 0.0, None),
                 lambda: A.layer_norm(x), lambda: A.dropout(x, 0.5, rng), lambda: A.dropout_add_ln(x, x)):
        refused(ValueError, "ROCm device tensors", call)


def test_a_missing_binding_is_an_error(monkeypatch):
    import sys

    import boltz_mlx_amd

    monkeypatch.setattr(_lib, "_train", None)
    monkeypatch.setitem(sys.modules, "boltz_mlx_amd._train", None)
    monkeypatch.delattr(boltz_mlx_amd, "_train", raising=False)
    refused(_lib.BzpfError, "build it with", lambda: K.dropout(torch.zeros(3), 0.0, None))


def test_modules():
    from boltz_mlx_amd.layers.dropout import Dropout

    d = Dropout(0.25, shared="row", site=3)
    x = torch.zeros(2, 3)
    assert d.eval()(x, None) is x and Dropout(0.0).train()(x, None) is x
    assert "0.25" in repr(d) and "row" in repr(d)
    with pytest.raises(ValueError):
        Dropout(1.5)


def test_workspaces_hold_what_the_sum_reads():
    """The kernel that adds the workgroups' partial sums reads those of 512 workgroups at most."""
    ws = _lib.load().bzpf_layernorm_bwd_ws
    for D in (8, 16, 64, 77, 128, 129, 384, 1024, 1025, 1536, 1537, 2048, 2049, 4097, 8192):
        for rows in (300, 5000, 10 ** 5, 10 ** 6, 2 ** 33, 2 ** 45):
            assert ws(rows, D) // (8 * D) <= 512


# -------------------------------------------------------------------------------------------------- overlapping buffers

def overlapping(code):
    assert code == -1 and b"overlap" in _lib.load().bzpf_last_error()


Q, R, S, V = P + 768, P + 1536, P + 2304, P + 3072  # tensors of 12 x 16 fp32, one behind the other


@pytest.mark.parametrize("y, x_dt, y_dt", [(P, F32, F32), (P, F16, F16), (P, F32, BF16), (P + 764, F32, F32),
                                           (P - 764, F32, F32), (P + 382, F16, F16)])
def test_dropout_refuses_overlapping_buffers(y, x_dt, y_dt):
    """In place, a row's last chunk may read what its neighbour has already dropped and scaled (12 rows of 16)."""
    overlapping(drop(x=P, x_dt=x_dt, y=y, y_dt=y_dt))


@pytest.mark.parametrize("change", [{"zn": P}, {"zn": Q}, {"zn": S}, {"ln": P}, {"ln": Q}, {"ln": R + 4}, {"zn": Q - 4},
                                    {"ln": P, "ln_dt": F16}])
def test_dropout_add_ln_refuses_overlapping_buffers(change):
    overlapping(res(**{**dict(z=P, y=Q, zn=R, ln=S), **change}))


@pytest.mark.parametrize("change", [{"dx": P + 4}, {"dx": Q + 764}, {"dx": P - 4}, {"dx": P, "x_dt": F16}])
def test_layernorm_bwd_refuses_overlapping_buffers(change):
    overlapping(ln_bwd(**{**dict(dy=P, x=Q, dx=R, rows=12, D=16), **change}))


@pytest.mark.parametrize("change", [{"dz": P + 4}, {"dz": Q - 4}, {"dz": V}, {"dy": R + 8}, {"dy": P, "y_dt": F16},
                                    {"dz": R, "dy": R}])
def test_dropout_add_ln_bwd_refuses_overlapping_buffers(change):
    overlapping(res_bwd(**{**dict(dzn=P, dln=Q, zn=R, dz=S, dy=V), **change}))


# -------------------------------------------------------------------------------------------------- the binding

def python(code, *args):
    """The output of a program in a process of its own (what it loads stays out of this one)."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code, *args], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_binding_calls_the_loaded_library(tmp_path):
    """With a library loaded from elsewhere, the torch binding calls that one, and the package's own is not in the process."""
    import shutil

    other = tmp_path / "other.so"
    shutil.copy(_lib.LIB_PATH, other)
    out = python("import sys; from boltz_mlx_amd import _lib; _lib.load(sys.argv[1]); _lib.train(); "
                 "print(*sorted({w for w in open('/proc/self/maps').read().split() if w.startswith('/')}), sep='\\n')",
                 str(other)).splitlines()
    assert str(other) in out and any(w.endswith("/_train.so") for w in out)
    assert not any(w.endswith("/libbzpf.so") for w in out)


def test_layer_norm_needs_no_binding(monkeypatch):
    """Inference calls LayerNorm everywhere, and runs where the torch binding is not built: the same checks, through the C
    ABI (its results: tests/test_gpu_training.py)."""
    import sys

    import boltz_mlx_amd

    monkeypatch.setattr(_lib, "_train", None)
    monkeypatch.setattr(_lib, "_no_train", False)
    monkeypatch.setitem(sys.modules, "boltz_mlx_amd._train", None)
    monkeypatch.delattr(boltz_mlx_amd, "_train", raising=False)
    test_layer_norm_refuses()
    refused(TypeError, "unsupported dtype", lambda: K.layer_norm(torch.zeros(3, 16).double(), None, None))
    refused(ValueError, "ROCm device tensors", lambda: K.layer_norm(torch.zeros(3, 16), torch.ones(16), None))
    assert _lib._no_train


def test_binding_of_another_torch_is_refused():
    """A binding built with another torch does not load: the training operators say so, LayerNorm does without it."""
    out = python("""
import torch
torch.__version__ = "1.2.3"
from boltz_mlx_amd import _lib, kernels as K
for call in (lambda: K.layer_norm(torch.zeros(3, 16), None, None), lambda: K.dropout(torch.zeros(3), 0.0, None)):
    try:
        call()
    except (ValueError, _lib.BzpfError) as e:
        print(e)
""").splitlines()
    assert out[0] == "layer_norm: need ROCm device tensors"
    assert "this is 1.2.3" in out[1] and "build it with" in out[1]


def test_a_binding_that_does_not_compile_leaves_the_library(monkeypatch, tmp_path):
    """Where torch's headers cannot be compiled, the build says so, with libbzpf.so linked (inference needs no more) and no
    binding of earlier sources left beside it."""
    from boltz_mlx_amd import build as B

    def compile_(src):
        if src.endswith(".cpp"):
            raise RuntimeError("no headers")
        return src

    linked, old = [], tmp_path / "old.so"
    old.touch()
    monkeypatch.setattr(B, "TRAIN", str(old))
    monkeypatch.setattr(B, "_compile", compile_)
    monkeypatch.setattr(B, "_link", lambda out, objs, *libs: linked.append((out, list(objs))))
    refused(RuntimeError, "no headers", lambda: B.build(verbose=False))
    assert linked == [(B.LIB, B.sources())] and not old.exists()
