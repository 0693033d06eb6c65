"""Plain 64-bit forms of the state space operators, token by token, for the tests.

Arrays are (tokens, channels); `spans` lists the half-open column range of every
sequence.  With ``mag`` every sum runs over the magnitudes of its terms: an error
that is relative to the terms is a multiple of that, so tolerances are too.
"""
import numpy as np

EPS = {"Float32": 2.0**-23, "Float16": 2.0**-10, "BFloat16": 2.0**-7}
TINY = {"Float32": 0.0, "Float16": 2.0**-25, "BFloat16": 0.0}  # half a step of Float16's smallest numbers


def sig(x):
    return 0.5 * (1.0 + np.tanh(0.5 * x))


def silu(x):
    return x * sig(x)


def dsilu(x):
    return sig(x) * (1.0 + x * (1.0 - sig(x)))


def dsilu_mag(x):
    """The terms of silu' = s + s x (1 - s) by magnitude: near x = -1.278 they cancel, and what is left of the
    derivative is smaller than the rounding of either."""
    return sig(x) * (1.0 + np.abs(x) * (1.0 - sig(x)))


def softplus(x):
    return np.maximum(x, 0.0) + np.log1p(np.exp(-np.abs(x)))


def close(got, ref, mag, eltype, k, what=""):
    """|got - ref| within half a step of the type and k units of 2^-24 of the terms' magnitudes."""
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    tol = EPS[eltype] / 2 * np.abs(ref) + TINY[eltype] + k * 2.0**-24 * np.asarray(mag) * (1 + EPS[eltype]) + 1e-37
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], ref[bad][:4], tol[bad][:4])


def spans_of(lens, lead=0):
    out, at = [], lead
    for n in lens:
        out.append((at, at + n))
        at += n
    return out


# ---- convolution ---------------------------------------------------------------------

def conv(x, w, bias, act, spans, init=None, dy=None, dlast=None, mag=False):
    """y, last[, dx, dw, dbias, dinit]; w is (W, D), states are (S, W-1, D)."""
    f = np.abs if mag else (lambda v: v)
    W, D = w.shape
    S = len(spans)
    y, last = np.zeros_like(x), np.zeros((S, W - 1, D))
    dx, dw, db, dinit = np.zeros_like(x), np.zeros((W, D)), np.zeros(D), np.zeros((S, W - 1, D))
    for s, (a, b) in enumerate(spans):
        h0 = init[s] if init is not None else np.zeros((W - 1, D))
        seen = np.concatenate([h0, x[a:b]])
        n = b - a
        true = sum(w[k] * seen[k:k + n] for k in range(W)) + bias
        pre = sum(f(w[k]) * f(seen[k:k + n]) for k in range(W)) + f(bias)
        y[a:b] = pre * (f(sig(true)) if act else 1.0)
        last[s] = f(seen[n:])
        if dy is not None:
            dp = f(dy[a:b]) * ((dsilu_mag(true) if mag else dsilu(true)) if act else 1.0)
            dp = dp + (f(dy[a:b]) * pre if mag and act else 0.0)  # act' moves with pre's own error
            dseen = np.zeros_like(seen)
            for k in range(W):
                dseen[k:k + n] += f(w[k]) * dp
                dw[k] += (dp * f(seen[k:k + n])).sum(0)
            db += dp.sum(0)
            if dlast is not None:
                dseen[n:] += f(dlast[s])
            dinit[s], dx[a:b] = dseen[:W - 1], dseen[W - 1:]
    return (y, last) if dy is None else (y, last, dx, dw, db, dinit)


# ---- scan ------------------------------------------------------------------------------

def scan(u, raw, A, B, C, skip, z, bias, soft, spans, init=None, dy=None, dlast=None, mag=False):
    """A (D, N), B and C (T, G, N), states (S, D, N).  y, last[, gradients as a dict]."""
    f = np.abs if mag else (lambda v: v)
    T, D = u.shape
    N, G, S = A.shape[1], B.shape[1], len(spans)
    grp = np.arange(D) // (D // G)
    x = raw + bias
    dt = softplus(x) if soft else x
    a = np.exp(dt[..., None] * A)
    fu, fB, fC, fd = f(u), f(B), f(C), f(skip)
    fdt = f(dt)
    gate, dgate = (f(silu(z)), dsilu_mag(z) if mag else dsilu(z)) if z is not None else (np.ones_like(u), None)
    y, h_all, before, last = np.zeros_like(u), np.zeros((T, D, N)), np.zeros((T, D, N)), np.zeros((S, D, N))
    for s, (lo, hi) in enumerate(spans):
        h = f(init[s]) if init is not None else np.zeros((D, N))
        for t in range(lo, hi):
            before[t] = h
            h = a[t] * h + (fdt[t] * fu[t])[:, None] * fB[t][grp]
            h_all[t] = h
        last[s] = h
    yp = np.zeros_like(u)
    for lo, hi in spans:
        yp[lo:hi] = (h_all[lo:hi] * fC[lo:hi][:, grp]).sum(-1) + fd * fu[lo:hi]
    y = yp * gate
    if dy is None:
        return y, last
    fdy = f(dy)
    dyp = fdy * gate
    g = {k: np.zeros_like(u) for k in ("u", "delta")}
    g.update(A=np.zeros((D, N)), B=np.zeros((T, G, N)), C=np.zeros((T, G, N)), D=np.zeros(D), bias=np.zeros(D),
             init=np.zeros((S, D, N)))
    g["z"] = fdy * yp * dgate if z is not None else None
    fA = f(A)
    for s, (lo, hi) in enumerate(spans):
        e = f(dlast[s]) if dlast is not None else np.zeros((D, N))
        for t in range(hi - 1, lo - 1, -1):
            gg = fC[t][grp] * dyp[t][:, None] + e
            q = gg * a[t] * before[t]
            g["A"] += q * fdt[t][:, None]
            gB = (gg * fB[t][grp]).sum(-1)
            ddt = (q * fA).sum(-1) + fu[t] * gB
            g["u"][t] = fdt[t] * gB + fd * dyp[t]
            g["delta"][t] = ddt * (sig(x[t]) if soft else 1.0)
            g["B"][t] = (gg * (fdt[t] * fu[t])[:, None]).reshape(G, D // G, N).sum(1)
            g["C"][t] = (h_all[t] * dyp[t][:, None]).reshape(G, D // G, N).sum(1)
            e = a[t] * gg
        g["init"][s] = e
        g["D"] += (dyp[lo:hi] * fu[lo:hi]).sum(0)
        g["bias"] += g["delta"][lo:hi].sum(0)
    return y, last, g


# ---- norms -----------------------------------------------------------------------------

def norm(r, w, h, hw, gate, act, scale, eps, dy=None, drout=None):
    """y, rout[, gradients as a dict]."""
    one = np.ones(r.shape[1])
    H = h if h is not None else np.zeros_like(r)
    i1 = 1.0 / np.sqrt((H**2).mean(-1, keepdims=True) + eps) if hw is not None else 1.0
    v = H * i1
    n = v * (hw if hw is not None else one)
    if gate is None:
        a, da = np.ones_like(r), np.zeros_like(r)
    elif act == "silu":
        a, da = silu(gate), dsilu(gate)
    else:
        a, da = sig(gate), sig(gate) * (1 - sig(gate))
    m = n * a
    sc = scale if scale is not None else one
    rout = r + sc * m
    i2 = 1.0 / np.sqrt((rout**2).mean(-1, keepdims=True) + eps)
    ww = w if w is not None else one
    y = rout * i2 * ww
    if dy is None and drout is None:
        return y, rout
    dro = drout if drout is not None else np.zeros_like(r)
    g = {"w": np.zeros(r.shape[1])}
    if dy is not None:
        xh, dx = rout * i2, dy * ww
        dro = dro + i2 * (dx - xh * (dx * xh).mean(-1, keepdims=True))
        g["w"] = (dy * xh).sum(0)
    dm = dro * sc
    dn = dm * a
    dv = dn * (hw if hw is not None else one)
    g.update(r=dro, scale=(dro * m).sum(0), gate=dm * n * da, hw=(dn * v).sum(0),
             h=i1 * (dv - v * (dv * v).mean(-1, keepdims=True)) if hw is not None else dv)
    return y, rout, g
