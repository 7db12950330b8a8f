"""What the speed of the block operators is judged by: the norm in front of an equivariant block (``IrrepsNorm``), the norm, gate,
scale and residual behind it (``GatedResidual``), and activations kept in 8 bits for the backward pass, by these two and by
``Linear``.  From one small molecule to the nodes of a million-edge training batch.

A case is a dict of plain values.  ``op`` names the operator:

* ``norm``      ``y = w x r(x)``, per row and irrep block ``r(x) = (mean of x^2 over the block + eps)^-1/2``;
* ``residual``  ``h = x + s act(g) y r(y)``; with ``norm_output`` also ``n = w h r(h)``, the norm in front of the next block;
* ``linear``    the equivariant linear layer that keeps its input in 8 bits for the weight gradient.

``saved = "int8"``: what the backward pass reads of an activation is, per row and irrep block, ``2^k rint(t 2^-k)`` with the
smallest ``k`` for which ``127 * 2^k`` holds the block's largest magnitude; ``r`` stays that of the exact values.

Sizes: 128 channels, lmax 3, 32,768 nodes, 64 / 96 channels are the ones of the benchmark configurations and of ``cases.py``; the
others are generic.
"""
from __future__ import annotations

import math
import re
from functools import lru_cache

import torch

own = False
DEVICE = "cuda"
EPS = 1e-5
DTYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16, "float16": torch.float16}
L3 = "128x0e+128x1o+128x2e+128x3o"


def listed():
    return [
        # One small molecule (21 atoms): a step of a few microseconds, all launches and host work.  Training.
        {"name": "norm_molecule", "op": "norm", "irreps": L3, "layout": "mul_ir", "rows": 21, "dtype": "float32", "train": True,
         "saved": "full"},
        # All nodes of the million-edge training batch (bench.py), in front of a block.
        {"name": "norm_batch", "op": "norm", "irreps": L3, "layout": "mul_ir", "rows": 32768, "dtype": "float32", "train": True,
         "saved": "full"},
        # A narrower model with odd counts in 16 bits, component-major, that keeps 8 bits of its activations.
        {"name": "norm_ragged_bf16", "op": "norm", "irreps": "96x0e+96x1o+96x2e", "layout": "ir_mul", "rows": 1999,
         "dtype": "bfloat16", "train": True, "saved": "int8"},
        # Molecular dynamics of the small molecule: between two blocks, forward only.
        {"name": "residual_molecule", "op": "residual", "irreps": L3, "layout": "mul_ir", "rows": 21, "dtype": "float32",
         "train": False, "gate": "sigmoid", "norm_output": True, "saved": "full"},
        # Behind a block of the training batch: activations kept as they are, ...
        {"name": "residual_batch", "op": "residual", "irreps": L3, "layout": "mul_ir", "rows": 32768, "dtype": "float32",
         "train": True, "gate": "sigmoid", "norm_output": False, "saved": "full"},
        # ... together with the norm in front of the next block, ...
        {"name": "residual_norm_batch", "op": "residual", "irreps": L3, "layout": "mul_ir", "rows": 32768, "dtype": "float32",
         "train": True, "gate": "sigmoid", "norm_output": True, "saved": "full"},
        # ... and kept in 8 bits.
        {"name": "residual_batch_int8", "op": "residual", "irreps": L3, "layout": "mul_ir", "rows": 32768, "dtype": "float32",
         "train": True, "gate": "sigmoid", "norm_output": False, "saved": "int8"},
        # Features on the edges of a batch in 16 bits: many short rows.
        {"name": "residual_edges_bf16", "op": "residual", "irreps": "64x0e+64x1o", "layout": "mul_ir", "rows": 262144,
         "dtype": "bfloat16", "train": True, "gate": "silu", "norm_output": False, "saved": "full"},
        # Double precision, as used to validate a model.
        {"name": "residual_norm_f64", "op": "residual", "irreps": "64x0e+64x1o+64x2e", "layout": "mul_ir", "rows": 4096,
         "dtype": "float64", "train": True, "gate": "silu", "norm_output": True, "saved": "full"},
        # The linear layer of the training batch, its input kept in 8 bits.
        {"name": "linear_batch_int8", "op": "linear", "irreps": L3, "layout": "mul_ir", "rows": 32768},
        # The same layer of a narrower model on a few hundred atoms.
        {"name": "linear_ragged_int8", "op": "linear", "irreps": "96x0e+64x1o+32x2e", "layout": "ir_mul", "rows": 421},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges; no drawn case moves more bytes than the largest listed ones of its kind."""
    op = rng.choice(["norm", "norm", "residual", "residual", "residual", "linear"])
    lmax = rng.randint(0, 3)
    layout = rng.choice(["mul_ir", "mul_ir", "ir_mul"])
    if op == "linear":
        muls = [rng.choice([32, 64, 96, 128])] * (lmax + 1) if rng.random() < 0.5 else [rng.choice([32, 64, 96, 128]) for _ in range(lmax + 1)]
    elif rng.random() < 0.6:
        muls = [rng.choice([16, 32, 48, 64, 96, 128, 128, 192, 256])] * (lmax + 1)
    else:
        muls = [_log_uniform(rng, 1, 256) for _ in range(lmax + 1)]
    irreps = "+".join(f"{m}x{l}{'eo'[l % 2]}" for l, m in enumerate(muls))  # noqa: E741
    dim = sum(m * (2 * l + 1) for l, m in enumerate(muls))  # noqa: E741
    if op == "linear":
        return {"op": op, "irreps": irreps, "layout": layout, "rows": _log_uniform(rng, 1, 32768)}
    dtype = rng.choice(["float32", "float32", "float32", "bfloat16", "bfloat16", "float16", "float64"])
    most = min(262144, 32768 * 2048 * 4 // (dim * (8 if dtype == "float64" else 4)))
    case = {"op": op, "irreps": irreps, "layout": layout, "rows": _log_uniform(rng, 1, most), "dtype": dtype,
            "train": rng.random() < 0.8, "saved": "int8" if dtype != "float64" and rng.random() < 0.4 else "full"}
    if op == "residual":
        case["gate"] = rng.choice(["sigmoid", "sigmoid", "silu", "none"])
        case["norm_output"] = case["saved"] == "full" and rng.random() < 0.5
    return case


# ---- the modules: a program builds each once and keeps it for all its inputs ----------------------------------------
@lru_cache(maxsize=None)
def _module(op, irreps, layout, saved, gate, norm_output):
    import cuequivariance_b200 as cb

    kw = dict(layout=getattr(cb, layout), internal_weights=False, saved_activations=saved)
    if op == "norm":
        return cb.IrrepsNorm(irreps, eps=EPS, **kw)
    if op == "residual":
        return cb.GatedResidual(irreps, eps=EPS, gate=None if gate == "none" else gate, norm_output=norm_output, **kw)
    return cb.Linear(irreps, irreps, shared_weights=True, **kw)


def _blocks(irreps):
    """[(mul, dim)] of a text like ``128x0e+128x1o``."""
    return [(int(m), 2 * int(l) + 1) for m, l in re.findall(r"(\d+)x(\d+)[eo]", irreps)]  # noqa: E741


# ---- prepare --------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    blocks = _blocks(case["irreps"])
    Z, dim, channels = case["rows"], sum(m * d for m, d in blocks), sum(m for m, _ in blocks)
    dt = DTYPES[case.get("dtype", "float32")]
    wide = torch.float64 if dt == torch.float64 else torch.float32

    def randn(*shape, scale=1.0, mean=0.0, dtype=dt):
        t = torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float64 if dtype == torch.float64 else torch.float32)
        return (t * scale + mean).to(dtype)

    def features(scale):
        """Rows of different magnitude, as nodes with few and many neighbours have; the rows of atoms without neighbours hold
        scalars only."""
        t = torch.randn(Z, dim, generator=gen, device=DEVICE, dtype=wide)
        t *= scale * torch.exp(0.5 * torch.randn(Z, 1, generator=gen, device=DEVICE, dtype=wide))
        n0 = sum(m * d for m, d in blocks if d == 1)
        if n0 < dim:
            alone = torch.rand(Z, generator=gen, device=DEVICE) < 0.01
            t[:, n0:].mul_((~alone).to(wide)[:, None])
        return t.to(dt)

    s = {"case": case, "blocks": blocks}
    if own:
        s["module"] = _module(case["op"], case["irreps"], case["layout"], case.get("saved", "int8"), case.get("gate", "none"),
                              case.get("norm_output", False))
    if case["op"] == "norm":
        s.update(x=features(1.0), w=randn(channels, scale=0.2, mean=1.0, dtype=wide))
        if case["train"]:
            s["cot"] = [randn(Z, dim)]
    elif case["op"] == "residual":
        s.update(x=features(1.0), y=features(2.0), s=randn(channels, scale=0.1, mean=0.5, dtype=wide))
        if case["gate"] != "none":
            s["g"] = randn(Z, channels, scale=1.5)
        if case["norm_output"]:
            s["w"] = randn(channels, scale=0.2, mean=1.0, dtype=wide)
        if case["train"]:
            s["cot"] = [randn(Z, dim) for _ in range(1 + case["norm_output"])]
    else:
        s.update(x=features(1.0), w=randn(1, sum(m * m for m, _ in blocks)), cot=[randn(Z, dim)])
    if own and "cot" in s:
        for k in ("x", "y", "g", "s", "w"):
            if k in s:
                s[k].requires_grad_(True)
    return s


# ---- run ------------------------------------------------------------------------------------------------------------
def run(s):
    if not own:
        return _plain(s)
    case, m, grad = s["case"], s["module"], torch.autograd.grad
    if case["op"] == "linear":
        out = m(s["x"], s["w"])
        return [out.detach(), *grad(out, (s["w"], s["x"]), s["cot"])]
    if case["op"] == "norm":
        call, leaves = (lambda: m(s["x"], weight=s["w"])), (s["x"], s["w"])
    else:
        call = lambda: m(s["x"], s["y"], gates=s.get("g"), scale=s["s"], weight=s.get("w"))  # noqa: E731
        leaves = tuple(s[k] for k in ("x", "y", "g", "s", "w") if k in s)
    if not case["train"]:
        with torch.no_grad():
            out = call()
        return list(out) if isinstance(out, tuple) else [out]
    out = call()
    out = list(out) if isinstance(out, tuple) else [out]
    return [*(o.detach() for o in out), *grad(out, leaves, s["cot"])]


def _split(t, blocks, layout):
    """A [rows, mul, dim] view per irrep block."""
    out, o = [], 0
    for m, d in blocks:
        b = t[:, o : o + m * d]
        out.append(b.reshape(-1, m, d) if layout == "mul_ir" else b.reshape(-1, d, m).transpose(1, 2))
        o += m * d
    return out


def _join(parts, layout):
    return torch.cat([(p if layout == "mul_ir" else p.transpose(1, 2)).reshape(p.shape[0], -1) for p in parts], dim=1)


def _kept(t, saved):
    """What the backward pass reads of the block ``t`` [rows, ...]."""
    if saved != "int8":
        return t
    amax = t.abs().flatten(1).amax(1).reshape(-1, *[1] * (t.dim() - 1))
    mantissa, k = torch.frexp(amax)
    k = torch.where(mantissa <= 127 / 128, k - 7, k - 6).clamp(min=-126)
    step = torch.ldexp(torch.ones_like(amax), k)
    return torch.round(t / step) * step


def _act(g, gate):
    """The gate's activation and its derivative."""
    if gate == "sigmoid":
        v = torch.sigmoid(g)
        return v, v * (1 - v)
    v = torch.sigmoid(g)
    return g * v, v * (1 + g * (1 - v))


def _plain(s):
    case, blocks = s["case"], s["blocks"]
    layout, saved, Z = case["layout"], case.get("saved", "int8"), case["rows"]
    math_dtype = torch.float64 if s["x"].dtype == torch.float64 else torch.float32
    data = s["x"].dtype
    split = lambda t: _split(t.to(math_dtype), blocks, layout)  # noqa: E731

    if case["op"] == "linear":
        out, gx, gw, o = [], [], [], 0
        for x, go, (m, _) in zip(split(s["x"]), split(s["cot"][0]), blocks):
            w, c = s["w"][0, o : o + m * m].reshape(m, m), m ** -0.5
            flat = lambda t: t.transpose(1, 2).reshape(-1, m)  # noqa: B023, E731  rows and components together
            back = lambda t: t.reshape(Z, -1, m).transpose(1, 2)  # noqa: B023, E731
            out.append(back(flat(x) @ w) * c)
            gx.append(back(flat(go) @ w.t()) * c)
            gw.append((flat(_kept(x, saved)).t() @ flat(go) * c).reshape(-1))
            o += m * m
        return [_join(out, layout), torch.cat(gw)[None], _join(gx, layout)]

    per_channel = lambda t: [b.reshape(1, -1, 1) for b in t.split([m for m, _ in blocks])]  # noqa: E731
    cots = [split(c) for c in s["cot"]] if case["train"] else []
    rms = lambda t: torch.rsqrt((t * t).flatten(1).mean(1) + EPS).reshape(-1, 1, 1)  # noqa: E731

    if case["op"] == "norm":
        xs, ws = split(s["x"]), per_channel(s["w"])
        rs = [rms(x) for x in xs]
        res = [_join([w * x * r for x, w, r in zip(xs, ws, rs)], layout).to(data)]
        if case["train"]:
            dx, dw = [], []
            for x, w, r, go in zip(xs, ws, rs, cots[0]):
                x = _kept(x, saved)
                p = (go * x).sum(2, keepdim=True)
                dw.append((r * p).sum(0).reshape(-1))
                mean = (w * p).sum(1, keepdim=True) / (x.shape[1] * x.shape[2])
                dx.append(r * (w * go - x * (r * r * mean)))
            res += [_join(dx, layout).to(data), torch.cat(dw)]
        return res

    xs, ys, ss = split(s["x"]), split(s["y"]), per_channel(s["s"])
    gs = [b[:, :, None] for b in s["g"].to(math_dtype).split([m for m, _ in blocks], dim=1)] if "g" in s else [None] * len(blocks)
    rs = [rms(y) for y in ys]
    hs = [x + sc * (y * r if g is None else _act(g, case["gate"])[0] * y * r) for x, y, sc, g, r in zip(xs, ys, ss, gs, rs)]
    res = [_join(hs, layout).to(data)]
    if case["norm_output"]:
        ws, rhs = per_channel(s["w"]), [rms(h) for h in hs]
        res.append(_join([w * h * r for h, w, r in zip(hs, ws, rhs)], layout).to(data))
    if not case["train"]:
        return res
    dxs, dys, dgs, dss, dws = [], [], [], [], []
    for b, go in enumerate(cots[0]):
        if case["norm_output"]:
            gn, h, w, r = cots[1][b], hs[b], ws[b], rhs[b]
            p = (gn * h).sum(2, keepdim=True)
            dws.append((r * p).sum(0).reshape(-1))
            mean = (w * p).sum(1, keepdim=True) / (h.shape[1] * h.shape[2])
            go = go + r * (w * gn - h * (r * r * mean))
        y, sc, r = _kept(ys[b], saved), ss[b], rs[b]
        p = (go * y).sum(2, keepdim=True)
        if gs[b] is None:
            a = sc
            dss.append((r * p).sum(0).reshape(-1))
        else:
            v, dv = _act(_kept(gs[b], saved), case["gate"])
            a = sc * v
            dss.append((v * r * p).sum(0).reshape(-1))
            dgs.append((sc * dv * r * p).reshape(Z, -1))
        mean = (a * p).sum(1, keepdim=True) / (y.shape[1] * y.shape[2])
        dxs.append(go)
        dys.append(r * (a * go - y * (r * r * mean)))
    res += [_join(dxs, layout).to(data), _join(dys, layout).to(data)]
    if "g" in s:
        res.append(torch.cat(dgs, dim=1).to(data))
    return res + [torch.cat(dss)] + ([torch.cat(dws)] if case["norm_output"] else [])


# ---- the definition in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    """Per irrep block, in 64 bits: Jacobian products of the normalised features ``t r(t)`` written out with einsum."""
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v)}
    cot = [c.double() for c in s.get("cot", [])]
    blocks, mul_ir, int8 = _blocks(case["irreps"]), case["layout"] == "mul_ir", case.get("saved", "int8") == "int8"
    Z = case["rows"]

    def quantised(t):
        top = t.abs().amax(dim=tuple(range(1, t.dim())), keepdim=True)
        k = torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / 127.0))
        k += (127.0 * torch.exp2(k) < top).double()           # log2 next to a power of two
        k -= (127.0 * torch.exp2(k - 1) >= top).double()
        k = k.clamp(min=-126.0)
        return torch.round(t * torch.exp2(-k)) * torch.exp2(k)

    def pull(grad, t, r):
        """The cotangent of ``t`` for the cotangent ``grad`` of ``t r(t)``, at the kept values ``t`` and the exact ``r``."""
        hat = t * r[:, None, None]
        along = torch.einsum("zui,zui->z", grad, hat) / (t.shape[1] * t.shape[2])
        return (grad - hat * along[:, None, None]) * r[:, None, None]

    def inverse_rms(t):
        return (torch.einsum("zui,zui->z", t, t) / (t.shape[1] * t.shape[2]) + EPS) ** -0.5

    parts, at, ch, wt = [], 0, 0, 0
    for m, dim in blocks:
        def cut(t):
            b = t[:, at : at + m * dim]  # noqa: B023
            return b.unflatten(1, (m, dim)) if mul_ir else b.unflatten(1, (dim, m)).mT  # noqa: B023

        def flat(t):
            return (t if mul_ir else t.mT).flatten(1)

        if case["op"] == "linear":
            x, go = cut(d["x"]), cut(cot[0])
            w = d["w"][0, wt : wt + m * m].unflatten(0, (m, m)) / math.sqrt(m)
            gw = torch.einsum("zui,zvi->uv", quantised(x), go) / math.sqrt(m)
            parts.append([flat(torch.einsum("zui,uv->zvi", x, w)), gw.flatten()[None], flat(torch.einsum("zvi,uv->zui", go, w))])
            wt += m * m
        elif case["op"] == "norm":
            x, w = cut(d["x"]), d["w"][ch : ch + m]
            r = inverse_rms(x)
            row = [flat(torch.einsum("zui,z,u->zui", x, r, w))]
            if cot:
                go, kept = cut(cot[0]), quantised(x) if int8 else x
                row += [flat(pull(torch.einsum("zui,u->zui", go, w), kept, r)), torch.einsum("zui,zui,z->u", go, kept, r)]
            parts.append(row)
        else:
            x, y, sc = cut(d["x"]), cut(d["y"]), d["s"][ch : ch + m]
            r = inverse_rms(y)

            def gate(g):
                if case["gate"] == "none":
                    return torch.ones(Z, m, dtype=torch.float64, device=DEVICE), None  # noqa: B023
                e = 1.0 / (1.0 + torch.exp(-g))
                return (e, e - e * e) if case["gate"] == "sigmoid" else (g * e, e + g * (e - e * e))

            g = d["g"][:, ch : ch + m] if "g" in d else None
            h = x + torch.einsum("zui,z,zu,u->zui", y, r, gate(g)[0], sc)
            row = [flat(h)]
            if case["norm_output"]:
                w, rh = d["w"][ch : ch + m], inverse_rms(h)
                row.append(flat(torch.einsum("zui,z,u->zui", h, rh, w)))
            if cot:
                gh = cut(cot[0])
                if case["norm_output"]:
                    gn = cut(cot[1])
                    gh = gh + pull(torch.einsum("zui,u->zui", gn, w), h, rh)
                kept, gk = (quantised(y) if int8 else y), (quantised(g) if int8 and g is not None else g)
                v, dv = gate(gk)
                p = torch.einsum("zui,zui,z->zu", gh, kept, r)
                row += [flat(gh), flat(pull(torch.einsum("zui,zu,u->zui", gh, v, sc), kept, r))]
                if g is not None:
                    row.append(p * dv * sc)
                row.append((p * v).sum(0))
                if case["norm_output"]:
                    row.append(torch.einsum("zui,zui,z->u", gn, h, rh))
            parts.append(row)
        at, ch = at + m * dim, ch + m
    res = [torch.cat(columns, dim=-1) for columns in zip(*parts)]
    return res


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    blocks, Z = _blocks(case["irreps"]), case["rows"]
    dim, channels = sum(m * d for m, d in blocks), sum(m for m, _ in blocks)
    size = {"float64": 8, "float32": 4}.get(case.get("dtype", "float32"), 2)
    param = 8 if size == 8 else 4
    if case["op"] == "linear":    # x, cotangent in, output and input gradient out; weights and their gradient
        return {"bytes": 4 * (4 * Z * dim + 2 * sum(m * m for m, _ in blocks)), "flops": 3 * 2 * Z * sum(m * m * d for m, d in blocks)}
    both = 2 if case["train"] else 1    # each input has a gradient, each output a cotangent
    if case["op"] == "norm":
        return {"bytes": both * (size * 2 * Z * dim + param * channels), "flops": Z * dim * (4 + (7 if case["train"] else 0))}
    gated, second = case["gate"] != "none", case["norm_output"]
    rows = size * Z * ((3 + second) * dim + gated * channels)
    return {"bytes": both * (rows + param * channels * (1 + second)),
            "flops": Z * dim * (5 + 3 * second + ((7 + 7 * second) if case["train"] else 0))}
