"""The norm in front of a block and the norm, gate and residual behind it in float64, with what an error bound needs: for every
result the same sums over the magnitudes of their terms.  Values kept in 8 bits are rounded as documented."""
import math

import torch


def blocks_of(irreps):
    return [(mul, ir.dim) for mul, ir in irreps if mul]


def split(t, blocks, mul_ir):
    out, o = [], 0
    for m, d in blocks:
        b = t[:, o : o + m * d]
        out.append(b.reshape(-1, m, d) if mul_ir else b.reshape(-1, d, m).transpose(1, 2))
        o += m * d
    return out


def join(parts, mul_ir):
    return torch.cat([(p if mul_ir else p.transpose(1, 2)).reshape(p.shape[0], -1) for p in parts], dim=1)


def step_of(t):
    """Per row of ``t`` [rows, ...]: the smallest power of two (at least 2^-126) of which 127 hold the largest magnitude."""
    out = []
    for top in t.abs().flatten(1).amax(1).tolist():
        if not math.isfinite(top):
            out.append(math.nan)
            continue
        k = -126
        while 127.0 * 2.0**k < top:
            k += 1
        out.append(2.0**k)
    return torch.tensor(out, dtype=torch.float64).reshape(-1, *[1] * (t.dim() - 1))


def kept(t, int8):
    if not int8:
        return t
    s = step_of(t)
    return torch.round(t / s) * s


def act(g, gate):
    """Activation, derivative, and the magnitude that the derivative's rounding errors scale with."""
    if gate is None:
        return torch.ones_like(g), torch.zeros_like(g), torch.zeros_like(g)
    e = torch.sigmoid(g)
    if gate == "sigmoid":
        return e, e * (1 - e), torch.ones_like(g)
    return g * e, e * (1 + g * (1 - e)), 1 + g.abs()


def reference(blocks, mul_ir, eps, gate, int8, x, y=None, g=None, s=None, w=None, go=None, gn=None):
    """``{name: (value, magnitude)}`` for out, norm, dx, dy, dg, ds, dw, as far as operands and cotangents are given."""
    d = lambda t: None if t is None else t.double()  # noqa: E731
    x, y, g, s, w, go, gn = map(d, (x, y, g, s, w, go, gn))
    sp = lambda t: [None] * len(blocks) if t is None else split(t, blocks, mul_ir)  # noqa: E731
    ch = lambda t: [None] * len(blocks) if t is None else t.split([m for m, _ in blocks], dim=-1)  # noqa: E731
    res = {}

    def put(name, value, mag, how):
        res.setdefault(name, ([], [], how))
        res[name][0].append(value)
        res[name][1].append(mag)

    rms = lambda t: ((t * t).flatten(1).mean(1) + eps).rsqrt().reshape(-1, 1, 1)  # noqa: E731
    for (m, dim), xb, yb, gb, sb, wb, gob, gnb in zip(blocks, sp(x), sp(y), ch(g), ch(s), ch(w), sp(go), sp(gn)):
        n = m * dim
        h, hmag = xb, xb.abs()
        if y is not None:
            r = rms(yb)
            gates = torch.zeros(x.shape[0], m, dtype=torch.float64) if gb is None else gb
            v = act(gates, gate)[0][:, :, None]
            sc = sb[None, :, None]
            h = xb + sc * v * yb * r
            hmag = xb.abs() + (sc * v * yb * r).abs()
            put("out", h, hmag, "rows")
        if w is not None:
            rh, wc = rms(h), wb[None, :, None]
            # an error of h moves its norm through h and, by at most as much again, through r
            put("norm", wc * h * rh, wc.abs() * rh * (hmag + h.abs() * rh**2 * (hmag * h.abs()).flatten(1).mean(1)[:, None, None]), "rows")
        if go is None and gn is None:
            continue
        cot = torch.zeros_like(xb) if gob is None else gob
        cmag = cot.abs()
        if gn is not None:
            hk = kept(h, int8)
            # h = x + branch is off by as much as its terms are, however small it is itself, and r(h) by the mean of that along h
            hm = (hk.abs() if y is None else hmag) * (1 + (rh**2 * (hmag * h.abs()).flatten(1).mean(1)[:, None, None] if y is not None else 0))
            p = (gnb * hk).sum(2, keepdim=True)
            pm = (gnb.abs() * hm).sum(2, keepdim=True)
            put("dw", (rh * p).sum((0, 2)), (rh * pm).sum((0, 2)), "channels")
            mean, mm = (wc * p).sum(1, keepdim=True) / n, (wc.abs() * pm).sum(1, keepdim=True) / n
            cot = cot + rh * (wc * gnb - hk * rh**2 * mean)
            cmag = cmag + rh * ((wc * gnb).abs() + hm * rh**2 * mm)
            put("dx", cot, cmag, "rows")
        elif y is not None:
            put("dx", cot, cmag, "rows")
        if y is None:
            continue
        yk, gk = kept(yb, int8), kept(gates, int8) if gb is not None else gates
        v, dv, dvm = (t[:, :, None] for t in act(gk, gate))
        p, pm = (cot * yk).sum(2, keepdim=True), (cmag * yk.abs()).sum(2, keepdim=True)
        a = sc * v
        mean, mm = (a * p).sum(1, keepdim=True) / n, (a.abs() * pm).sum(1, keepdim=True) / n
        put("dy", r * (a * cot - yk * r**2 * mean), r * (a.abs() * cmag + yk.abs() * r**2 * mm), "rows")
        put("ds", (v * r * p).sum((0, 2)), (v.abs() * r * pm).sum((0, 2)), "channels")
        if gb is not None:
            put("dg", (sc * dv * r * p)[:, :, 0], (sc.abs() * dvm * r * pm)[:, :, 0], "gates")
    joined = {}
    for name, (vals, mags, how) in res.items():
        j = (lambda t: join(t, mul_ir)) if how == "rows" else (lambda t: torch.cat(t, dim=-1))
        joined[name] = (j(vals), j(mags))
    return joined


def bound(name, mag, value, blocks, rows, dtype, both):
    """Largest error of a result.  Unit u = 2^-24 (2^-53 for float64).  A sum over an item is a chain of at most n / 32 + 10
    additions (a thread's share, 5 in a warp, 4 warps) of terms that are rounded themselves; r comes from one such sum, dot and a
    row's gradient from one more (two behind a branch with a norm); 40 covers the factors, expf and the reciprocals.  Sums over rows: a
    thread block's rows in a chain, then all thread blocks in 16 chains, at most rows + 40 additions.  Results of 16 bits are
    rounded once, by half a step; the norm's backward pass then reads h in these 16 bits, half a step off in both of its places."""
    u = 2.0**-53 if dtype == torch.float64 else 2.0**-24
    chain = max(m * d for m, d in blocks) / 32 + 10
    k = 40 + 3 * chain * (2 if both else 1) + (rows + 40 if name in ("ds", "dw") else 0)
    tol = k * u * mag + 1e-37
    if dtype in (torch.bfloat16, torch.float16):
        half = torch.finfo(dtype).eps / 2
        if name not in ("ds", "dw"):
            tol = tol + half * value.abs() * (1 + 2.0**-7) + (2.0**-25 if dtype == torch.float16 else 0)   # fp16: half of its smallest number
        if both and name not in ("out", "norm"):
            tol = tol + 2 * half * mag
    return tol
