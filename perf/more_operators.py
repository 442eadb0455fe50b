"""The sequence attention's training form with its positions as measurable cases: the learned relative position bias by
buckets, the norms of queries and keys for each head with the position rotation, and the attention that reads both, each
with its gradients. Their sizes are those of the single track (16 heads of 24), of the diffusion tokens (16 heads of 48, five
samples that share one bias) and generic ones.

listed() are the fixed cases, draw(rng) gives more of the same ranges, prepare() makes what a program holds before the call,
run() is one pass, work() what the pass cannot do without and exact() the same pass in 64 bits. While `own` is false, run()
computes the plain form in elementary torch operations; otherwise it calls the framework.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# input and output types of the norms (one half type in a call)
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"),
         ("bf16", "f32")]


def listed() -> list:
    return [
        # the position bias of a small crop: launch and host time
        {"name": "bias_forward_small", "op": "rel_bias", "pass": "forward", "b": 1, "h": 16, "n": 29, "m": 29, "kind": "clip",
         "reach": 32, "chains": 1, "add": False, "t": "f32"},
        # a training step over two crops of three chains: the position bias added to the pair bias, and the table's gradient
        {"name": "bias_step_crops_n400", "op": "rel_bias", "pass": "step", "b": 2, "h": 16, "n": 400, "m": 400, "kind": "clip",
         "reach": 32, "chains": 3, "add": True, "t": "f16"},
        # the table's gradient over a long sequence, logarithmic buckets
        {"name": "bias_backward_log_n2000", "op": "rel_bias", "pass": "backward", "b": 1, "h": 16, "n": 2000, "m": 2000,
         "kind": "log", "reach": 512, "chains": 1, "add": False, "t": "bf16"},
        # one token's query and key at a far position: launch and host time
        {"name": "norms_forward_one_token", "op": "qk_norm_rope", "pass": "forward", "b": 1, "n": 1, "h": 16, "hk": 16, "c": 24,
         "rotary": 24, "interleaved": False, "far": 1000000, "packed": True, "x": "f32", "y": "f32"},
        # the single track of an ordinary protein in a training step, q and k as parts of the fused projection's rows
        {"name": "norms_step_single_n400", "op": "qk_norm_rope", "pass": "step", "b": 1, "n": 400, "h": 16, "hk": 16, "c": 24,
         "rotary": 24, "interleaved": False, "far": 400, "packed": True, "x": "f32", "y": "f32"},
        # the gradients over a batch of long sequences, a quarter of the key heads, half of each head rotated
        {"name": "norms_backward_long", "op": "qk_norm_rope", "pass": "backward", "b": 8, "n": 4001, "h": 16, "hk": 4, "c": 128,
         "rotary": 64, "interleaved": True, "far": 100000, "packed": False, "x": "bf16", "y": "bf16"},
        # one token against an ordinary protein's keys
        {"name": "attention_forward_one_token", "op": "attention", "pass": "forward", "s": 1, "mult": 1, "h": 16, "c": 24,
         "n": 1, "m": 400, "t": "f32", "bias": "f32", "gate": True, "pad": 0.1},
        # the single track of an ordinary protein in a training step
        {"name": "attention_step_single_n400", "op": "attention", "pass": "step", "s": 1, "mult": 1, "h": 16, "c": 24, "n": 400,
         "m": 400, "t": "f32", "bias": "f32", "gate": True, "pad": 0.1},
        # the diffusion tokens in a training step: five samples share one bias
        {"name": "attention_step_samples_n400", "op": "attention", "pass": "step", "s": 5, "mult": 5, "h": 16, "c": 48,
         "n": 400, "m": 400, "t": "f16", "bias": "f16", "gate": True, "pad": 0.05},
        # odd lengths and an odd head count, fewer keys than queries, one sample without any key
        {"name": "attention_backward_odd", "op": "attention", "pass": "backward", "s": 3, "mult": 1, "h": 7, "c": 40, "n": 777,
         "m": 613, "t": "bf16", "bias": "bf16", "gate": False, "pad": 0.3},
        # a long sequence, forward
        {"name": "attention_forward_long", "op": "attention", "pass": "forward", "s": 1, "mult": 1, "h": 16, "c": 64, "n": 4096,
         "m": 4096, "t": "bf16", "bias": "bf16", "gate": False, "pad": 0.0},
        # the gradients over a batch of large complexes
        {"name": "attention_backward_n2000", "op": "attention", "pass": "backward", "s": 2, "mult": 1, "h": 16, "c": 64,
         "n": 2000, "m": 2000, "t": "bf16", "bias": "bf16", "gate": True, "pad": 0.05},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    op = rng.choice(["rel_bias", "qk_norm_rope", "attention", "attention"])
    if op == "rel_bias":
        b, h = rng.choice([1, 1, 2, 3]), rng.choice([1, 4, 8, 16, rng.randint(1, 32)])
        n = _log(rng, 1, min(4000, math.isqrt(64_000_000 // (b * h))))
        m = n if rng.random() < 0.7 else _log(rng, 1, min(4000, 64_000_000 // (b * h * n)))
        kind = rng.choice(["clip", "log"])
        return {"op": op, "pass": rng.choice(["forward", "backward", "step"]), "b": b, "h": h, "n": n, "m": m, "kind": kind,
                "reach": _log(rng, 1, 64) if kind == "clip" else _log(rng, 32, 1024), "chains": rng.choice([1, 1, 2, 5]),
                "add": rng.random() < 0.5, "t": rng.choice(["f32", "f16", "bf16"])}
    if op == "qk_norm_rope":
        c = rng.choice([16, 24, 32, 48, 64, 128]) if rng.random() < 0.6 else 2 * _log(rng, 4, 128)
        h = rng.choice([1, 3, 4, 8, 16, 24])
        hk = rng.choice([k for k in (h, h, h // 2, 1) if k and h % k == 0])
        b = rng.choice([1, 1, 2, 5])
        n = max(1, _log(rng, 1, min(8000, 80_000_000 // (b * c * (h + hk)))))
        x, y = rng.choice(PAIRS)
        return {"op": op, "pass": rng.choice(["forward", "backward", "step"]), "b": b, "n": n, "h": h, "hk": hk, "c": c,
                "rotary": rng.choice([c, c, 2 * rng.randint(0, c // 2)]), "interleaved": rng.random() < 0.4,
                "far": rng.choice([400, 4000, 100000, 10000000]), "packed": rng.random() < 0.5, "x": x, "y": y}
    c = rng.choice([24, 32, 48, 64]) if rng.random() < 0.7 else 8 * rng.randint(1, 16)
    h, mult = rng.choice([1, 4, 8, 16, rng.randint(1, 16)]), rng.choice([1, 1, 1, 2, 5])
    s = mult * rng.choice([1, 1, 2])
    most = 128_000_000 * 64 // (s * h * c)  # queries times keys
    n = _log(rng, 1, min(3000, math.isqrt(most)))
    m = n if rng.random() < 0.7 else _log(rng, 1, min(3000, most // n))
    t = rng.choice(["f32", "f16", "bf16", "bf16"])
    return {"op": op, "pass": rng.choice(["forward", "backward", "step"]), "s": s, "mult": mult, "h": h, "c": c, "n": n, "m": m,
            "t": t, "bias": rng.choice(["none", t, t, rng.choice(["f16", "bf16"]) if t == "f32" else t]), "gate": rng.random() < 0.7,
            "pad": rng.choice([0.0, 0.05, 0.1, 0.3])}


def edges_of(case: dict) -> list:
    """The buckets' borders: one for each distance up to the reach, or distances that grow by a quarter from 8 on."""
    reach = case["reach"]
    if case["kind"] == "clip":
        return list(range(1 - reach, reach + 1))
    steps, at = list(range(1, 9)), 8
    while at + max(1, at // 4) <= reach:
        at += max(1, at // 4)
        steps.append(at)
    return [1 - d for d in reversed(steps)] + steps


def prepare(case: dict, seed: int) -> dict:
    """Positions are residue numbers with gaps that begin anew in each chain; activations have a scale of their own for each
    row and channel; gradients are of a tenth; the tail of each sample is padding, and one sample of several with much
    padding has no key at all."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def ints(hi, *shape):
        return torch.randint(0, hi, shape, generator=gen, device="cuda")

    grad = case["pass"] == "step"
    st = {"case": dict(case), "own": {}}
    if case["op"] == "rel_bias":
        b, h, n, m = case["b"], case["h"], case["n"], case["m"]
        t, other = TYPES[case["t"]], case["chains"] > 1
        st["edges"] = edges_of(case)
        st["count"] = len(st["edges"]) + 1 + other

        def positions(k):
            chain = (torch.arange(k, device="cuda") * case["chains"] // k).expand(b, k)
            gaps = 1 + (ints(20, b, k) == 0) * ints(12, b, k)
            gaps[:, 0] += ints(40, b)
            total = gaps.cumsum(1)
            start = total.gather(1, torch.searchsorted(chain.contiguous(), chain.contiguous()))
            return (total - start + 1).contiguous(), chain.contiguous()

        st["pos_q"], st["chain_q"] = positions(n)
        st["pos_k"], st["chain_k"] = (st["pos_q"], st["chain_q"]) if n == m else positions(m)
        st["table"] = (0.5 * rand(st["count"], h)).requires_grad_(grad)
        if case["add"]:
            st["add"] = rand(b, h, n, m).to(t).requires_grad_(grad)
        if case["pass"] != "forward":
            st["dy"] = (0.1 * rand(b, h, n, m)).to(t)
        if own:
            from boltz_mlx_amd import kernels as K

            st["own"]["buckets"] = K.rel_buckets(st["edges"], other=other)
        return st
    if case["op"] == "qk_norm_rope":
        b, n, h, hk, c = case["b"], case["n"], case["h"], case["hk"], case["c"]
        tx, ty = TYPES[case["x"]], TYPES[case["y"]]
        scale = 0.5 + rand(c).abs()
        rows = torch.cat([rand(b, n, h, c) * scale * (0.2 + rand(b, n, h, 1).abs()),
                          rand(b, n, hk, c) * scale * (0.2 + rand(b, n, hk, 1).abs())], 2).reshape(b, n, (h + hk) * c)
        if case["packed"]:  # the projection's rows: q, k, then v and g
            rows = torch.cat([rows, rand(b, n, (h + hk) * c)], 2).to(tx)
            st["q"], st["k"] = rows[..., :h * c].detach(), rows[..., h * c:(h + hk) * c].detach()
        else:
            st["q"], st["k"] = rows[..., :h * c].to(tx).contiguous(), rows[..., h * c:].to(tx).contiguous()
        st["q"].requires_grad_(grad), st["k"].requires_grad_(grad)
        st["wq"] = (1 + 0.1 * rand(c)).requires_grad_(grad)
        st["wk"] = (1 + 0.1 * rand(c)).requires_grad_(grad)
        st["pos"] = ints(case["far"], b, 1) + torch.arange(n, device="cuda")
        if case["pass"] != "forward":
            st["dq"], st["dk"] = (0.1 * rand(b, n, h * c)).to(ty), (0.1 * rand(b, n, hk * c)).to(ty)
        return st
    s, mult, h, c, n, m = (case[k] for k in ("s", "mult", "h", "c", "n", "m"))
    t = TYPES[case["t"]]
    for name, rows in (("q", n), ("k", m), ("v", m)) + ((("g", n),) if case["gate"] else ()):
        st[name] = rand(s, rows, h * c).mul_(0.5 + rand(h * c).abs()).to(t).requires_grad_(grad)
    if case["bias"] != "none":
        st["bias"] = rand(s // mult, h, n, m).to(TYPES[case["bias"]]).requires_grad_(grad)
    st["mask"] = torch.ones(s, m, device="cuda")
    for i in range(s):
        last = m - round(case["pad"] * m * (i + 1) / s)
        st["mask"][i, max(1, last):] = 0
    if s > 2 and case["pad"] >= 0.3:
        st["mask"][s - 1] = 0
    if case["pass"] != "forward":
        st["dout"] = (0.1 * rand(s, n, h * c)).to(t)
    if case["pass"] == "backward":
        if own:
            from boltz_mlx_amd import kernels as K

            st["out"], st["stats"] = K.attention(st["q"], st["k"], st["v"], h, g=st.get("g"), bias=st.get("bias"),
                                                 mask=st["mask"], multiplicity=mult)
        else:
            st["out"], st["stats"], _ = _forward(st)
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
    if op == "rel_bias":
        at = (st["own"]["buckets"], st["pos_q"], st["pos_k"], st["chain_q"], st["chain_k"])
        out = TYPES[case["t"]]
        if which == "forward":
            return {"bias": K.rel_bias(st["table"], *at, add=st.get("add"), out_dtype=out)}
        if which == "backward":
            return {"dtable": K.rel_bias_bwd(st["dy"], *at)}
        y = A.rel_bias(st["table"], *at, add=st.get("add"), out_dtype=out)
        d = torch.autograd.grad(y, [st[k] for k in ("table", "add") if k in st], st["dy"])
        return {"bias": y.detach(), **{"d" + k: v for k, v in zip(("table", "add"), d)}}
    if op == "qk_norm_rope":
        args = (st["q"], st["k"], st["wq"], st["wk"], case["h"], st["pos"])
        more = {"eps": EPS, "rotary": case["rotary"], "interleaved": case["interleaved"]}
        if which == "forward":
            q, k = K.qk_norm_rope(*args, **more, out_dtype=TYPES[case["y"]])
            return {"q": q, "k": k}
        if which == "backward":
            d = K.qk_norm_rope_bwd(st["dq"], st["dk"], *args, **more)
            return dict(zip(("dq", "dk", "dwq", "dwk"), d))
        q, k = A.qk_norm_rope(*args, **more, out_dtype=TYPES[case["y"]])
        d = torch.autograd.grad((q, k), args[:4], (st["dq"], st["dk"]))
        return {"q": q.detach(), "k": k.detach(), **dict(zip(("dq", "dk", "dwq", "dwk"), d))}
    more = {"g": st.get("g"), "bias": st.get("bias"), "mask": st["mask"], "multiplicity": case["mult"]}
    qkv = (st["q"], st["k"], st["v"])
    if which == "forward":
        out, stats = K.attention(*qkv, case["h"], **more)
        return {"out": out, "stats": stats}
    if which == "backward":
        d = K.attention_bwd(st["dout"], *qkv, case["h"], st["out"], st["stats"], **more)
        return {k: v for k, v in zip(("dq", "dk", "dv", "dg", "dbias"), d) if v is not None}
    out = A.attention(*qkv, case["h"], **more)
    names = [k for k in ("q", "k", "v", "g", "bias") if k in st]
    d = torch.autograd.grad(out, [st[k] for k in names], st["dout"])
    return {"out": out.detach(), **{"d" + k: v for k, v in zip(names, d)}}


# -------------------------------------------------------------------------------------------------- the plain forms

def _plain(st: dict):
    return {"rel_bias": _plain_bias, "qk_norm_rope": _plain_norms, "attention": _plain_attention}[st["case"]["op"]](st)


def _bucket(st: dict) -> torch.Tensor:
    """[b, n, m] buckets: how many borders lie at or below the distance, the last one for pairs of different chains."""
    d = st["pos_q"][:, :, None] - st["pos_k"][:, None, :]
    at = torch.bucketize(d, torch.tensor(st["edges"], device=d.device), right=True)
    if st["case"]["chains"] > 1:
        at = torch.where(st["chain_q"][:, :, None] == st["chain_k"][:, None, :], at, st["count"] - 1)
    return at


def _plain_bias(st: dict):
    case = st["case"]
    at, out = _bucket(st), {}
    if case["pass"] != "backward":
        y = st["table"].t()[:, at].transpose(0, 1)
        out["bias"] = (y + st["add"].float() if case["add"] else y).to(TYPES[case["t"]]).contiguous()
    if case["pass"] != "forward":
        # long sums: in 64 bits, of each query's row first
        dy = st["dy"].double().transpose(1, 2)  # [b, n, h, m]
        rows = torch.zeros(*dy.shape[:3], st["count"], dtype=torch.float64, device=dy.device)
        rows.scatter_add_(3, at[:, :, None, :].expand_as(dy), dy)
        out["dtable"] = rows.sum((0, 1)).t().float()
        if case["add"] and case["pass"] == "step":
            out["dadd"] = st["dy"]
    return out


def _turn(x: torch.Tensor, case: dict, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [b, n, heads, c] with its first `rotary` channels rotated."""
    r = case["rotary"]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
    a, b = a * cos - b * sin, a * sin + b * cos
    ab = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([ab, x[..., r:]], -1)


def _plain_norms(st: dict):
    case = st["case"]
    b, n, c, r = case["b"], case["n"], case["c"], case["rotary"]
    angle = st["pos"].double()[..., None] * 10000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / max(r, 1))
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    out = {}
    for name in ("q", "k"):
        x, w = st[name].float().reshape(b, n, -1, c), st["w" + name]
        rms = 1.0 / ((x * x).mean(-1, keepdim=True) + EPS).sqrt()
        xh = x * rms
        if case["pass"] != "backward":
            out[name] = _turn(xh * w, case, cos, sin).to(TYPES[case["y"]]).reshape(b, n, -1)
        if case["pass"] != "forward":
            g = _turn(st["d" + name].float().reshape(b, n, -1, c), case, cos, -sin)
            out["dw" + name] = (g * xh).sum((0, 1, 2))
            gw = g * w
            out["d" + name] = (rms * (gw - xh * (gw * xh).mean(-1, keepdim=True))).to(TYPES[case["x"]]).reshape(b, n, -1)
    return out


def _heads(x: torch.Tensor, h: int) -> torch.Tensor:
    """[s, n, h c] as [s, h, n, c] in 32 bits."""
    return x.float().unflatten(-1, (h, -1)).transpose(1, 2).contiguous()


def _rows(x: torch.Tensor, t) -> torch.Tensor:
    return x.transpose(1, 2).flatten(2).to(t)


def _forward(st: dict):
    """(out, stats, p) of the attention; stats are each row's largest logit and the sum of exp(logit - that)."""
    case = st["case"]
    h = case["h"]
    x = _heads(st["q"], h) @ _heads(st["k"], h).transpose(2, 3).contiguous()
    x *= case["c"] ** -0.5
    if "bias" in st:
        x = (x.unflatten(0, (-1, case["mult"])) + st["bias"].float()[:, None]).flatten(0, 1)
    keep = st["mask"] != 0
    keep = keep | ~keep.any(1, keepdim=True)  # a sample without keys runs without its mask
    x.masked_fill_(~keep[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - top).exp_()
    total = p.sum(-1, keepdim=True)
    p /= total
    o = p @ _heads(st["v"], h)
    if "g" in st:
        o = o * torch.sigmoid(_heads(st["g"], h))
    return _rows(o, TYPES[case["t"]]), torch.cat([top, total], -1), p


def _plain_attention(st: dict):
    case = st["case"]
    h, t = case["h"], TYPES[case["t"]]
    o, stats, p = _forward(st)
    if case["pass"] == "forward":
        return {"out": o, "stats": stats}
    out = {"out": o} if case["pass"] == "step" else {}
    v, do = _heads(st["v"], h), _heads(st["dout"], h)
    if "g" in st:
        gate = torch.sigmoid(_heads(st["g"], h))
        out["dg"] = _rows(do * (p @ v) * gate * (1 - gate), t)
        do = do * gate
    out["dv"] = _rows(p.transpose(2, 3).contiguous() @ do, t)
    dp = do @ v.transpose(2, 3).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    if "bias" in st:
        out["dbias"] = ds.unflatten(0, (-1, case["mult"])).sum(1).to(st["bias"].dtype)
    ds = ds * case["c"] ** -0.5
    out["dq"] = _rows(ds @ _heads(st["k"], h), t)
    out["dk"] = _rows(ds.transpose(2, 3).contiguous() @ _heads(st["q"], h), t)
    return out


# -------------------------------------------------------------------------------------------------- work and exact values

def work(case: dict) -> dict:
    which = case["pass"]
    fwd, bwd = which != "backward", which != "forward"
    if case["op"] == "rel_bias":
        n = case["b"] * case["h"] * case["n"] * case["m"]
        # the bias (and the pair bias) once; its gradient once
        return {"bytes": n * SIZE[case["t"]] * (fwd * (1 + case["add"]) + bwd) + 16 * case["b"] * (case["n"] + case["m"]),
                "flops": n * (fwd * (1 + case["add"]) + bwd)}
    if case["op"] == "qk_norm_rope":
        n = case["b"] * case["n"] * case["c"] * (case["h"] + case["hk"])
        sx, sy = SIZE[case["x"]], SIZE[case["y"]]
        return {"bytes": n * (sx + fwd * sy + bwd * (sx + sy)) + 8 * case["b"] * case["n"], "flops": n * (3 + 4 * fwd + 10 * bwd)}
    s, h, n, m, c = (case[k] for k in ("s", "h", "n", "m", "c"))
    e, gate = SIZE[case["t"]], case["gate"]
    bias = 0 if case["bias"] == "none" else SIZE[case["bias"]] * (s // case["mult"]) * h * n * m
    qo, kv = s * n * h * c * e, s * m * h * c * e
    # q, k, v, g and the bias once (a backward pass reads out and dout too); out; the gradients
    moved = (qo * (1 + gate) + 2 * kv + bias) + fwd * qo + bwd * ((1 + (which == "backward")) * qo + qo * (1 + gate) + 2 * kv + bias)
    return {"bytes": moved + 4 * s * m, "flops": s * h * n * m * c * (4 * fwd + 10 * bwd)}


def exact(case: dict, seed: int):
    global own
    kept, own = own, False
    try:
        st = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    finally:
        own = kept
    return {"rel_bias": _exact_bias, "qk_norm_rope": _exact_norms, "attention": _exact_attention}[case["op"]](case, st)


def _exact_bias(case, st):
    out, edges = {}, torch.tensor(st["edges"], device="cuda")
    fwd, bwd = case["pass"] != "backward", case["pass"] != "forward"
    bias, grad = [], torch.zeros(st["count"], case["h"], dtype=torch.float64, device="cuda")
    for b in range(case["b"]):
        at = torch.zeros(case["n"], case["m"], dtype=torch.int64, device="cuda")
        d = st["pos_q"][b].unsqueeze(1) - st["pos_k"][b].unsqueeze(0)
        for e in edges.tolist():
            at += d >= e
        if case["chains"] > 1:
            at[st["chain_q"][b].unsqueeze(1) != st["chain_k"][b].unsqueeze(0)] = st["count"] - 1
        if fwd:
            y = st["table"].double()[at].permute(2, 0, 1)
            bias.append(y + st["add"][b].double() if case["add"] else y)
        if bwd:
            for k in range(st["count"]):
                i, j = (at == k).nonzero(as_tuple=True)
                grad[k] += st["dy"][b][:, i, j].double().sum(1)
    if fwd:
        out["bias"] = torch.stack(bias)
    if bwd:
        out["dtable"] = grad
        if case["add"] and fwd:
            out["dadd"] = st["dy"].double()
    return out


def _exact_norms(case, st):
    b, n, c, r = case["b"], case["n"], case["c"], case["rotary"]
    p = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.ones(b, n, 1, r // 2, dtype=torch.float64, device="cuda"),
                       (st["pos"].double()[:, :, None] * torch.exp(-math.log(10000.0) * 2 * p / max(r, 1)))[:, :, None])

    def rotated(x, by):
        z = x[..., :r].unflatten(-1, (r // 2, 2) if case["interleaved"] else (2, r // 2))
        if not case["interleaved"]:
            z = z.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * by)
        z = z if case["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), x[..., r:]], -1)

    out = {}
    for name in ("q", "k"):
        x, w = st[name].double().unflatten(-1, (-1, c)), st["w" + name].double()
        size = torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
        if case["pass"] != "backward":
            out[name] = rotated(x / size * w, turn).flatten(2)
        if case["pass"] != "forward":
            g = rotated(st["d" + name].double().unflatten(-1, (-1, c)), turn.conj())
            out["dw" + name] = (g * x / size).sum((0, 1, 2))
            g = g * w
            out["d" + name] = (g / size - x * (g * x).mean(-1, keepdim=True) / size ** 3).flatten(2)
    return out


def _exact_attention(case, st):
    s, mult, h, c, n, m = (case[k] for k in ("s", "mult", "h", "c", "n", "m"))
    bwd = case["pass"] != "forward"
    parts = {}
    sums = torch.zeros(s // mult, h, n, m, dtype=torch.float64, device="cuda") if bwd and "bias" in st else None
    for i in range(s):
        sees = st["mask"][i].nonzero().flatten()
        if not len(sees):
            sees = torch.arange(m, device="cuda")
        for j in range(h):
            col = slice(j * c, (j + 1) * c)
            q, k, v = st["q"][i, :, col].double(), st["k"][i, sees, col].double(), st["v"][i, sees, col].double()
            x = torch.mm(q, k.t().contiguous()) / math.sqrt(c)
            if "bias" in st:
                x = x + st["bias"][i // mult, j][:, sees].double()
            top = x.max(1, keepdim=True).values
            total = torch.exp(x - top).sum(1, keepdim=True)
            p = torch.exp(x - top - torch.log(total))
            o = torch.mm(p, v)
            got = {"stats": torch.cat([top, total], 1)}
            gate = 1 / (1 + torch.exp(-st["g"][i, :, col].double())) if "g" in st else torch.ones_like(o)
            got["out"] = o * gate
            if bwd:
                do = st["dout"][i, :, col].double()
                if "g" in st:
                    got["dg"] = do * o * (gate - gate * gate)
                do = do * gate
                dp = torch.mm(do, v.t().contiguous())
                ds = p * dp - p * (do * o).sum(1, keepdim=True)
                if sums is not None:
                    sums[i // mult, j, :, sees] += ds
                got["dq"] = torch.mm(ds, k) / math.sqrt(c)
                for name, x, y in (("dk", ds, q / math.sqrt(c)), ("dv", p, do)):
                    got[name] = torch.zeros(m, c, dtype=torch.float64, device="cuda")
                    got[name][sees] = torch.mm(x.t().contiguous(), y)
            for name, x in got.items():
                parts.setdefault(name, {})[i, j] = x
    out = {name: torch.stack([torch.cat([of[i, j] for j in range(h)], 1) for i in range(s)])
           for name, of in parts.items() if name != "stats"}
    if not bwd:
        out["stats"] = torch.stack([torch.stack([parts["stats"][i, j] for j in range(h)]) for i in range(s)])
        return out
    if sums is not None:
        out["dbias"] = sums
    if case["pass"] == "backward":
        del out["out"]
    return out
