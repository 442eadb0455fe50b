"""The training operators of the pair and single tracks as measurable cases: LayerNorm with its backward pass, dropout
from a counter-based generator (no mask is stored) and the residual update z + dropout(y) with the LayerNorm that follows
it. Their sizes are those of the trunk (single 384, pair 128, MSA and template 64, diffusion tokens 768) and generic ones.

listed() are the fixed cases, draw(rng) gives more of the same ranges, prepare() makes what a program holds before the
call, run() is one pass, work() what the pass cannot do without and exact() the same pass in 64 bits. While `own` is
false, run() computes the plain form in elementary torch operations; otherwise it calls the framework.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# LayerNorm's input and output types (the residual update's y and LayerNorm output take the same pairs); one half type
# in a call.
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"),
         ("bf16", "f32")]


def listed() -> list:
    return [
        # the single track of one token: launch and host time
        {"name": "ln_forward_one_token", "op": "layer_norm", "pass": "forward", "b": 1, "i": 1, "j": 1, "d": 384,
         "x": "f32", "y": "bf16"},
        # the single track of an ordinary protein in a training step: forward and backward through autograd
        {"name": "ln_step_single_n400", "op": "layer_norm", "pass": "step", "b": 1, "i": 1, "j": 400, "d": 384,
         "x": "f32", "y": "f32"},
        # the pair representation of the largest complex: the backward pass with both parameter gradients
        {"name": "ln_backward_pair_n1000", "op": "layer_norm", "pass": "backward", "b": 1, "i": 1000, "j": 1000,
         "d": 128, "x": "f32", "y": "f16"},
        # the diffusion tokens of five samples, all in bf16
        {"name": "ln_backward_tokens_d768", "op": "layer_norm", "pass": "backward", "b": 5, "i": 1, "j": 400, "d": 768,
         "x": "bf16", "y": "bf16"},
        # an odd width and an odd row count
        {"name": "ln_forward_odd_d1021", "op": "layer_norm", "pass": "forward", "b": 1, "i": 1, "j": 4099, "d": 1021,
         "x": "f32", "y": "f32"},
        # wide rows, forward and backward
        {"name": "ln_step_wide_d8192", "op": "layer_norm", "pass": "step", "b": 1, "i": 2, "j": 1025, "d": 8192,
         "x": "bf16", "y": "bf16"},
        # a small tensor, forward and backward: launch and host time
        {"name": "dropout_step_small", "op": "dropout", "pass": "step", "b": 1, "i": 1, "j": 29, "d": 384, "x": "f32",
         "y": "f32", "p": 0.1, "shared": "none"},
        # a draw for each element of the MSA track over a deep alignment
        {"name": "dropout_forward_msa", "op": "dropout", "pass": "forward", "b": 1, "i": 1024, "j": 400, "d": 64,
         "x": "f16", "y": "f16", "p": 0.15, "shared": "none"},
        # the pair track's dropout with one draw for each row of pairs, forward and backward
        {"name": "dropout_step_pair_n400", "op": "dropout", "pass": "step", "b": 1, "i": 400, "j": 400, "d": 128,
         "x": "bf16", "y": "bf16", "p": 0.25, "shared": "row"},
        # one pair update of an ordinary protein: z + dropout(y) and the next module's LayerNorm
        {"name": "residual_forward_pair_n400", "op": "dropout_add_ln", "pass": "forward", "b": 1, "i": 400, "j": 400,
         "d": 128, "x": "f16", "y": "f16", "p": 0.25, "shared": "row"},
        # the backward pass of the ending node's update (one draw for each column) on the largest complex
        {"name": "residual_backward_pair_n1000", "op": "dropout_add_ln", "pass": "backward", "b": 1, "i": 1000,
         "j": 1000, "d": 128, "x": "f16", "y": "f16", "p": 0.25, "shared": "column"},
        # a batch of odd crops at an odd width, a draw for each element, forward and backward
        {"name": "residual_step_odd_d77", "op": "dropout_add_ln", "pass": "step", "b": 3, "i": 83, "j": 83, "d": 77,
         "x": "f32", "y": "bf16", "p": 0.1, "shared": "none"},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    op = rng.choice(["layer_norm", "layer_norm", "dropout", "dropout_add_ln", "dropout_add_ln"])
    # below eight channels a LayerNorm's gradient cancels (to eps / variance at two): no case of the range
    d = rng.choice([64, 128, 128, 256, 384, 512, 768, 1024, 2048, 4096, 8192]) if rng.random() < 0.6 else \
        _log(rng, 1 if op == "dropout" else 8, 8192)
    rows = _log(rng, 1, min(1_000_000, 64_000_000 // d))
    b = rng.choice([1, 1, 2, 3])
    i = max(1, min(_log(rng, 1, 1000), rows // b))
    x, y = rng.choice(PAIRS)
    case = {"op": op, "pass": rng.choice(["forward", "backward", "step"]), "b": b, "i": i, "j": max(1, rows // (b * i)),
            "d": d, "x": x, "y": y}
    if op == "dropout":
        case["y"] = x
        case["pass"] = rng.choice(["forward", "step"])
    if op != "layer_norm":
        case["p"] = rng.choice([0.0, 0.1, 0.15, 0.25, 0.5, round(rng.uniform(0.0, 0.9), 3)])
        case["shared"] = rng.choice(["none", "row", "column"])
    return case


def prepare(case: dict, seed: int) -> dict:
    """Activations with a mean and a scale of their own for each row and channel, LayerNorm weights near 1, gradients of
    a tenth, and the generator's (seed, offset) on the device."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b, i, j, d = case["b"], case["i"], case["j"], case["d"]
    grad = case["pass"] == "step"

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def acts(scale, dtype):
        t = rand(b, i, j, d)
        t *= scale * (1 + 0.5 * rand(d).abs())
        t += 0.5 * scale * rand(b, i, j, 1)
        return t.to(dtype).requires_grad_(grad)

    st = {"case": dict(case), "site": 1 + case["d"] % 7}
    st["rng"] = torch.randint(0, 2 ** 62, (2,), generator=gen, device="cuda", dtype=torch.int64)
    if case["op"] != "dropout":
        st["w"] = (1 + 0.1 * rand(d)).requires_grad_(grad)
        st["b"] = (0.1 * rand(d)).requires_grad_(grad)
    if case["op"] == "dropout_add_ln":
        st["z"] = acts(3.0, torch.float32)  # the stream before the update; after it in the backward pass alone
        if case["pass"] != "backward":
            st["y"] = acts(1.0, TYPES[case["x"]])
        if case["pass"] != "forward":
            st["dz"] = 0.1 * rand(b, i, j, d)
            st["dxn"] = (0.1 * rand(b, i, j, d)).to(TYPES[case["y"]])
    else:
        st["x"] = acts(1.0, TYPES[case["x"]])
        if case["pass"] != "forward":
            st["dy"] = (0.1 * rand(b, i, j, d)).to(TYPES[case["y"]])
    return st


def run(st: dict):
    if own:
        return _own(st)
    with torch.no_grad():
        return _plain(st)


# -------------------------------------------------------------------------------------------------- the framework's calls

def _own(st: dict):
    from boltz_mlx_amd import autograd as A
    from boltz_mlx_amd import kernels as K

    case = st["case"]
    op, which = case["op"], case["pass"]
    out = TYPES[case["y"]]
    shared = None if case.get("shared", "none") == "none" else case["shared"]
    if op == "layer_norm":
        if which == "forward":
            return {"y": K.layer_norm(st["x"], st["w"], st["b"], EPS, out_dtype=out)}
        if which == "backward":
            dx, dw, db = K.layer_norm_bwd(st["dy"], st["x"], st["w"], EPS)
            return {"dx": dx, "dw": dw, "db": db}
        y = A.layer_norm(st["x"], st["w"], st["b"], EPS, out_dtype=out)
        dx, dw, db = torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if op == "dropout":
        if which == "forward":
            return {"y": K.dropout(st["x"], case["p"], st["rng"], st["site"], shared)}
        y = A.dropout(st["x"], case["p"], st["rng"], st["site"], shared)
        (dx,) = torch.autograd.grad(y, (st["x"],), st["dy"])
        return {"y": y.detach(), "dx": dx}
    if which == "forward":
        zn, xn = K.dropout_add_ln(st["z"], st["y"], st["w"], st["b"], EPS, case["p"], st["rng"], st["site"], shared,
                                  out_dtype=out)
        return {"z": zn, "xn": xn}
    if which == "backward":
        dz, dy, dw, db = K.dropout_add_ln_bwd(st["dz"], st["dxn"], st["z"], st["w"], EPS, case["p"], st["rng"],
                                              st["site"], shared, y_dtype=TYPES[case["x"]])
        return {"dz": dz, "dy": dy, "dw": dw, "db": db}
    zn, xn = A.dropout_add_ln(st["z"], st["y"], st["w"], st["b"], EPS, case["p"], st["rng"], st["site"], shared,
                              out_dtype=out)
    dz, dy, dw, db = torch.autograd.grad((zn, xn), (st["z"], st["y"], st["w"], st["b"]), (st["dz"], st["dxn"]))
    return {"z": zn.detach(), "xn": xn.detach(), "dz": dz, "dy": dy, "dw": dw, "db": db}


# -------------------------------------------------------------------------------------------------- the plain forms

LOW = 0xFFFFFFFF


def _words(blocks: int, rng: torch.Tensor, site: int) -> torch.Tensor:
    """[blocks, 4] words of Philox4x32-10 (Salmon et al. 2011), key = the seed, counter = (block, site, offset)."""
    n = torch.arange(blocks, device=rng.device)
    k0, k1 = rng[0] & LOW, (rng[0] >> 32) & LOW
    c0, c1 = n & LOW, (n >> 32) | (site << 16)
    c2, c3 = rng[1] & LOW, (rng[1] >> 32) & LOW
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & LOW) ^ c1 ^ k0, p1 & LOW, ((p0 >> 32) & LOW) ^ c3 ^ k1, p0 & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return torch.stack([c0.expand(blocks), c1.expand(blocks), c2.expand(blocks), c3.expand(blocks)], 1)


def _dropped(case: dict, st: dict) -> torch.Tensor:
    """Where the draw is below p, broadcastable over [b, i, j, d]."""
    b, i, j, d = case["b"], case["i"], case["j"], case["d"]
    limit = round(case["p"] * 2 ** 32)
    if case["shared"] == "none":
        per = (d + 3) // 4
        return (_words(b * i * j * per, st["rng"], st["site"]) < limit).view(b, i, j, 4 * per)[..., :d]
    shape = (b, i, 1, 1) if case["shared"] == "row" else (b, 1, j, 1)
    n = math.prod(shape)
    return (_words((n + 3) // 4, st["rng"], st["site"]) < limit).view(-1)[:n].view(shape)


def _drop(t: torch.Tensor, case: dict, dropped: torch.Tensor) -> torch.Tensor:
    return torch.where(dropped, 0.0, t * (1.0 / (1.0 - case["p"])))


def _normalised(x: torch.Tensor):
    c = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / ((c * c).mean(-1, keepdim=True) + EPS).sqrt()
    return c * rstd, rstd


def _norm_grads(g: torch.Tensor, xh: torch.Tensor, rstd: torch.Tensor, w: torch.Tensor):
    gw = g * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return dx, (g * xh).sum((0, 1, 2)), g.sum((0, 1, 2))


def _plain(st: dict):
    case = st["case"]
    op, which = case["op"], case["pass"]
    tx, ty = TYPES[case["x"]], TYPES[case["y"]]
    out = {}
    if op == "layer_norm":
        xh, rstd = _normalised(st["x"].float())
        if which != "backward":
            out["y"] = (xh * st["w"] + st["b"]).to(ty)
        if which != "forward":
            dx, out["dw"], out["db"] = _norm_grads(st["dy"].float(), xh, rstd, st["w"])
            out["dx"] = dx.to(tx)
        return out
    dropped = _dropped(case, st)
    if op == "dropout":
        out["y"] = _drop(st["x"].float(), case, dropped).to(ty)
        if which != "forward":
            out["dx"] = _drop(st["dy"].float(), case, dropped).to(tx)
        return out
    zn = st["z"]
    if which != "backward":
        out["z"] = zn = zn + _drop(st["y"].float(), case, dropped)
    xh, rstd = _normalised(zn)
    if which != "backward":
        out["xn"] = (xh * st["w"] + st["b"]).to(ty)
    if which != "forward":
        dx, out["dw"], out["db"] = _norm_grads(st["dxn"].float(), xh, rstd, st["w"])
        out["dz"] = st["dz"] + dx
        out["dy"] = _drop(out["dz"], case, dropped).to(tx)
    return out


# -------------------------------------------------------------------------------------------------- work and exact values

def work(case: dict) -> dict:
    n, d = case["b"] * case["i"] * case["j"] * case["d"], case["d"]
    sx, sy, op, which = SIZE[case["x"]], SIZE[case["y"]], case["op"], case["pass"]
    fwd, bwd = which != "backward", which != "forward"
    if op == "layer_norm":
        # x once; y; dy and dx; the weight, the bias and their gradients
        return {"bytes": n * (sx + fwd * sy + bwd * (sx + sy)) + 4 * d * (1 + fwd + 2 * bwd),
                "flops": n * (6 + 2 * fwd + 9 * bwd)}
    draws = 20 / 4 * n if case["shared"] == "none" else 0  # twenty products for four draws
    if op == "dropout":
        return {"bytes": n * (sx + sy) * (fwd + bwd), "flops": int(draws + n * (fwd + bwd))}
    # z, y, the new z and its LayerNorm; the two gradients that come and the two that go (the new z too in a backward pass)
    return {"bytes": n * (fwd * (8 + sx + sy) + bwd * (8 + sx + sy) + (which == "backward") * 4) +
            4 * d * (1 + fwd + 2 * bwd), "flops": int(draws + n * (6 + 4 * fwd + 11 * bwd))}


def _high(a: torch.Tensor, m: int) -> torch.Tensor:
    """The upper 32 bits of a * m for 32-bit a and m, in 16-bit limbs."""
    a0, a1, m0, m1 = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
    mid = a1 * m0 + (a0 * m0 >> 16)
    return a1 * m1 + (mid >> 16) + ((mid & 0xFFFF) + a0 * m1 >> 16)


def exact(case: dict, seed: int):
    st = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    b, i, j, d = case["b"], case["i"], case["j"], case["d"]
    fwd, bwd = case["pass"] != "backward", case["pass"] != "forward"
    keep = None
    if case["op"] != "layer_norm":
        key, offset = (int(v) for v in st["rng"].tolist())
        count = {"none": b * i * j * (-(-d // 4)), "row": -(-b * i // 4), "column": -(-b * j // 4)}[case["shared"]]
        n = torch.arange(count, device="cuda")
        c = [n % 2 ** 32, n // 2 ** 32 + st["site"] * 2 ** 16, torch.full_like(n, offset % 2 ** 32),
             torch.full_like(n, offset // 2 ** 32)]
        for turn in range(10):
            k0 = (key + turn * 0x9E3779B9) % 2 ** 32
            k1 = (key // 2 ** 32 + turn * 0xBB67AE85) % 2 ** 32
            high0, high1 = _high(c[0], 0xD2511F53), _high(c[2], 0xCD9E8D57)
            low0, low1 = c[0] * 0xD2511F53 & LOW, c[2] * 0xCD9E8D57 & LOW
            c = [high1 ^ c[1] ^ k0, low1, high0 ^ c[3] ^ k1, low0]
        u = torch.stack(c, -1).flatten().double() / 2.0 ** 32
        keep = u >= round(case["p"] * 2 ** 32) / 2.0 ** 32
        if case["shared"] == "none":
            keep = keep.view(b, i, j, -1)[..., :d]
        elif case["shared"] == "row":
            keep = keep[:b * i].view(b, i, 1, 1)
        else:
            keep = keep[:b * j].view(b, 1, j, 1)

    def thinned(t):
        return torch.where(keep, t / (1 - case["p"]), torch.zeros_like(t))

    out = {}
    if case["op"] == "dropout":
        out["y"] = thinned(st["x"].double())
        if bwd:
            out["dx"] = thinned(st["dy"].double())
        return out
    x = st["x" if case["op"] == "layer_norm" else "z"].double()
    if case["op"] == "dropout_add_ln" and fwd:
        x = x + thinned(st["y"].double())
        out["z"] = x
    w = st["w"].double()
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    dev = torch.sqrt(var + EPS)
    xh = (x - mean) / dev
    if fwd:
        out["y" if case["op"] == "layer_norm" else "xn"] = xh * w + st["b"].double()
    if bwd:
        g = st["dy" if case["op"] == "layer_norm" else "dxn"].double()
        out["dw"], out["db"] = torch.einsum("bijd,bijd->d", g, xh), g.sum((0, 1, 2))
        g = g * w
        dx = (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) / dev
        if case["op"] == "layer_norm":
            out["dx"] = dx
        else:
            out["dz"] = st["dz"].double() + dx
            out["dy"] = thinned(out["dz"])
    return out
