"""State space operators on the GPU against their plain 64-bit forms.

Tolerances count roundings: half a step of the output's type, plus k units of
2^-24 of the magnitudes of the summed terms.  For the scan k = 8 (L + 24) with L
the longest sequence: each of at most L decay factors is off by at most 2^-22
(the power of two) plus |dt A| 2^-23, which the factor itself outweighs, twice
over when the gradient walks back, and the elementwise functions add less than
24.  The convolution and the norms have a fixed number of operations: k = 64
covers W + 1 products, a sigmoid and a sum over the block's tokens in registers
and parts; sums over n tokens or channels add n / 8 (pairwise or walked by
several threads).
"""
import ctypes
import itertools

import numpy as np
import pytest
import torch

import cutilecpu_b200 as mk
import statespace_ref as ref

pytestmark = pytest.mark.gpu

TD = {"Float32": torch.float32, "Float16": torch.float16, "BFloat16": torch.bfloat16}
BE = mk.MLIRCUDABackend()


def gen(seed):
    return np.random.Generator(np.random.Philox(seed))


def dev(x, eltype="Float32"):
    """A device array of x (tokens first), and what it holds in 64 bits."""
    t = torch.from_numpy(np.ascontiguousarray(x)).to(torch.float32).to(TD[eltype]).cuda()
    return mk.MLIRArray(t.reshape(-1), dims=tuple(reversed(x.shape))), t.double().cpu().numpy()


def out(shape, eltype="Float32", fill=7.0):
    t = torch.full(shape, fill, dtype=TD[eltype], device="cuda")
    return mk.MLIRArray(t.reshape(-1), dims=tuple(reversed(shape)))


def host(a):
    """(tokens first) 64-bit copy of a device array."""
    return a.to_numpy().astype(np.float64).transpose(*reversed(range(len(a.dims))))


def ints(x):
    return mk.MLIRArray(np.asarray(x, np.int32))


def seqs_of(spans):
    return ints([a + 1 for a, _ in spans] + [spans[-1][1] + 1])


def inside(spans, T):
    m = np.zeros(T, bool)
    for a, b in spans:
        m[a:b] = True
    return m


# ---- convolution ---------------------------------------------------------------------

CONV = [  # lens, channels, taps, columns in front and behind, silu, bias, states
    ([1], 1, 2, 0, 0, True, True, False),
    ([5, 0, 1, 2, 33], 7, 4, 0, 0, True, True, True),
    ([64, 65, 63], 64, 4, 3, 5, True, False, True),
    ([200], 130, 3, 0, 0, False, True, False),
    ([0, 0, 3, 0], 16, 4, 0, 2, True, True, True),
    ([1, 1, 1, 1, 1, 1, 1, 1, 1, 300], 40, 2, 1, 1, True, True, True),
    ([777], 256, 4, 0, 0, True, True, False),
]


@pytest.mark.parametrize("eltype", list(TD))
@pytest.mark.parametrize("lens,D,W,lead,tail,silu,has_bias,states", CONV)
def test_conv(cuda, lens, D, W, lead, tail, silu, has_bias, states, eltype):
    r = gen(sum(lens) * 131 + D + W)
    spans = ref.spans_of(lens, lead)
    T, S = lead + sum(lens) + tail, len(lens)
    x, xv = dev(r.standard_normal((T, D)), eltype)
    w, wv = dev(r.standard_normal((W, D)))
    b, bv = dev(r.standard_normal(D)) if has_bias else (None, np.zeros(D))
    h0, h0v = dev(r.standard_normal((S, W - 1, D)), eltype) if states else (None, None)
    last = out((S, W - 1, D), eltype) if states else None
    y = out((T, D), eltype)
    mk.causal_conv(y, x, w, bias=b, silu=silu, seqs=seqs_of(spans), init=h0, last=last)
    mk.synchronize(BE)
    wy, wl = ref.conv(xv, wv, bv, silu, spans, h0v)
    my, _ = ref.conv(xv, wv, bv, silu, spans, h0v, mag=True)
    m = inside(spans, T)
    ref.close(host(y)[m], wy[m], my[m], eltype, 64, "y")
    assert (host(y)[~m] == 7.0).all()
    if states:
        np.testing.assert_array_equal(host(last), wl)

    dy, dyv = dev(r.standard_normal((T, D)), eltype)
    dl, dlv = dev(r.standard_normal((S, W - 1, D)), eltype) if states else (None, None)
    dx, dw, db = out((T, D), eltype), out((W, D)), out((D,)) if has_bias else None
    di = out((S, W - 1, D), eltype) if states else None
    mk.causal_conv_grad(dx, dw, dy, x, w, bias=b, dbias=db, silu=silu, seqs=seqs_of(spans), init=h0, dinit=di, dlast=dl)
    mk.synchronize(BE)
    want = ref.conv(xv, wv, bv, silu, spans, h0v, dyv, dlv)
    mag = ref.conv(xv, wv, bv, silu, spans, h0v, dyv, dlv, mag=True)
    ref.close(host(dx)[m], want[2][m], mag[2][m], eltype, 64, "dx")
    assert (host(dx)[~m] == 7.0).all()
    ref.close(host(dw), want[3], mag[3], "Float32", 64 + T / 8, "dw")
    if has_bias:
        ref.close(host(db), want[4], mag[4], "Float32", 64 + T / 8, "dbias")
    if states:
        ref.close(host(di), want[5], mag[5], eltype, 64, "dinit")


def test_conv_state_in_place_and_in_slots(cuda):
    r = gen(5)
    lens, D, W = [1, 40, 0, 2, 31], 24, 4
    spans = ref.spans_of(lens)
    x, xv = dev(r.standard_normal((sum(lens), D)), "BFloat16")
    w, wv = dev(r.standard_normal((W, D)))
    pool, pv = dev(r.standard_normal((9, W - 1, D)), "BFloat16")
    slots = [3, 9, 1, 0, 6]  # the fourth keeps no state
    y = out((sum(lens), D), "BFloat16")
    mk.causal_conv(y, x, w, seqs=seqs_of(spans), init=pool, last=pool, slots=ints(slots))
    mk.synchronize(BE)
    h0 = np.stack([pv[k - 1] if k > 0 else np.zeros((W - 1, D)) for k in slots])
    wy, wl = ref.conv(xv, wv, np.zeros(D), True, spans, h0)
    my, _ = ref.conv(xv, wv, np.zeros(D), True, spans, h0, mag=True)
    ref.close(host(y), wy, my, "BFloat16", 64)
    want = pv.copy()
    for s, k in enumerate(slots):
        if k > 0:
            want[k - 1] = wl[s]
    np.testing.assert_array_equal(host(pool), want)


@pytest.mark.parametrize("eltype", list(TD))
@pytest.mark.parametrize("B,D,W", [(1, 1, 2), (3, 33, 4), (64, 256, 4), (5, 516, 3)])
def test_conv_step(cuda, B, D, W, eltype):
    r = gen(B * 7 + D)
    x, xv = dev(r.standard_normal((B, D)), eltype)
    w, wv = dev(r.standard_normal((W, D)))
    b, bv = dev(r.standard_normal(D))
    st, sv = dev(r.standard_normal((B + 2, W - 1, D)), eltype)
    slots = np.arange(B + 2, 2, -1)
    slots[B // 2] = 0
    for inplace in (False, True):
        nxt = st if inplace else out((B + 2, W - 1, D), eltype)
        y = out((B, D), eltype)
        mk.causal_conv_step(y, nxt, st, x, w, bias=b, slots=ints(slots))
        mk.synchronize(BE)
        for e in range(B):
            if slots[e] == 0:
                assert (host(y)[e] == 7.0).all()
                continue
            wy, wl = ref.conv(xv[e:e + 1], wv, bv, True, [(0, 1)], sv[slots[e] - 1][None])
            my, _ = ref.conv(xv[e:e + 1], wv, bv, True, [(0, 1)], sv[slots[e] - 1][None], mag=True)
            ref.close(host(y)[e], wy[0], my[0], eltype, 64)
            np.testing.assert_array_equal(host(nxt)[slots[e] - 1], wl[0])
        untouched = [k for k in range(B + 2) if k + 1 not in slots]
        np.testing.assert_array_equal(host(nxt)[untouched], sv[untouched] if inplace else 7.0)


# ---- scan ------------------------------------------------------------------------------

SCAN = [  # lens, channels, states, groups, columns in front and behind, z, skip, bias, softplus, states
    ([1], 1, 1, 1, 0, 0, True, True, True, True, True),
    ([5, 0, 1, 2, 33], 7, 4, 1, 0, 0, True, True, True, True, True),
    ([64, 65, 63, 128], 64, 16, 1, 3, 5, True, True, True, True, True),
    ([150], 66, 16, 2, 0, 0, False, False, True, True, False),
    ([0, 0, 3, 0], 16, 8, 4, 0, 2, True, False, True, True, True),
    ([9, 200], 39, 11, 3, 1, 0, True, True, False, False, False),
    ([70, 31], 40, 24, 1, 0, 0, True, True, True, True, True),
    ([70, 1], 20, 64, 2, 0, 0, True, True, True, True, True),
    ([600], 33, 16, 1, 2, 1, True, True, True, True, True),     # cut into pieces
    ([700, 0, 513], 40, 5, 2, 0, 0, True, True, True, True, True),
    ([640], 8, 40, 1, 0, 0, False, True, True, True, True),
]


def scan_case(lens, D, N, G, lead, tail, has_z, has_skip, has_bias, soft, states, eltype, seed=0):
    r = gen(sum(lens) * 31 + D * 7 + N + seed)
    T, S = lead + sum(lens) + tail, len(lens)
    c = {"spans": ref.spans_of(lens, lead), "T": T, "S": S, "D": D, "N": N, "G": G, "soft": soft, "eltype": eltype}
    v = {}

    def put(name, x, t="Float32"):
        c[name], v[name] = dev(x, t)

    put("u", r.standard_normal((T, D)), eltype)
    put("delta", (0.5 * r.standard_normal((T, D)) - (0 if has_bias else -0.6)), eltype)
    put("A", -np.exp(0.5 * r.standard_normal((D, N))))
    put("B", r.standard_normal((T, G, N)), eltype)
    put("C", r.standard_normal((T, G, N)), eltype)
    put("z", r.standard_normal((T, D)), eltype)
    put("skip", r.standard_normal(D))
    put("bias", r.uniform(-5, 0, D))
    put("init", r.standard_normal((S, D, N)))
    put("dlast", r.standard_normal((S, D, N)))
    put("dy", r.standard_normal((T, D)), eltype)
    for name, has in (("z", has_z), ("skip", has_skip), ("bias", has_bias), ("init", states), ("dlast", states)):
        if not has:
            c[name] = v[name] = None
    c["v"] = v
    return c


def scan_ref(c, grad=False, mag=False):
    v, D = c["v"], c["D"]
    more = dict(dy=v["dy"], dlast=v["dlast"]) if grad else {}
    return ref.scan(v["u"], v["delta"], v["A"], v["B"], v["C"], v["skip"] if v["skip"] is not None else np.zeros(D),
                    v["z"], v["bias"] if v["bias"] is not None else np.zeros(D), c["soft"], c["spans"], v["init"],
                    mag=mag, **more)


def scan_forward(c, saved=None):
    y = out((c["T"], c["D"]), c["eltype"])
    last = out((c["S"], c["D"], c["N"])) if c["init"] is not None else None
    mk.selective_scan(y, c["u"], c["delta"], c["A"], c["B"], c["C"], D=c["skip"], z=c["z"], bias=c["bias"],
                      softplus=c["soft"], seqs=seqs_of(c["spans"]), init=c["init"], last=last, saved=saved)
    return y, last


def scan_grad(c, saved):
    t = c["eltype"]
    g = {"u": out((c["T"], c["D"]), t), "delta": out((c["T"], c["D"]), t), "A": out((c["D"], c["N"])),
         "B": out((c["T"], c["G"], c["N"]), t), "C": out((c["T"], c["G"], c["N"]), t),
         "D": out((c["D"],)) if c["skip"] is not None else None,
         "z": out((c["T"], c["D"]), t) if c["z"] is not None else None,
         "bias": out((c["D"],)) if c["bias"] is not None else None,
         "init": out((c["S"], c["D"], c["N"])) if c["init"] is not None else None}
    mk.selective_scan_grad(g["u"], g["delta"], g["A"], g["B"], g["C"], c["dy"], c["u"], c["delta"], c["A"], c["B"],
                           c["C"], saved, D=c["skip"], dD=g["D"], z=c["z"], dz=g["z"], bias=c["bias"], dbias=g["bias"],
                           softplus=c["soft"], seqs=seqs_of(c["spans"]), dinit=g["init"], dlast=c["dlast"])
    return g


def k_scan(c):
    return 8 * (max(b - a for a, b in c["spans"]) + 24)


@pytest.mark.parametrize("eltype", list(TD))
@pytest.mark.parametrize("args", SCAN)
def test_scan_and_gradients(cuda, args, eltype):
    c = scan_case(*args, eltype)
    saved = mk.selective_scan_saved(c["u"], c["A"], seqs=seqs_of(c["spans"]))
    y, last = scan_forward(c, saved)
    mk.synchronize(BE)
    wy, wl = scan_ref(c)
    my, ml = scan_ref(c, mag=True)
    m, k = inside(c["spans"], c["T"]), k_scan(c)
    ref.close(host(y)[m], wy[m], my[m], eltype, k, "y")
    assert (host(y)[~m] == 7.0).all()
    if last is not None:
        ref.close(host(last), wl, ml, "Float32", k, "last")

    g = scan_grad(c, saved)
    mk.synchronize(BE)
    want, mag = scan_ref(c, grad=True)[2], scan_ref(c, grad=True, mag=True)[2]
    for name in ("u", "delta", "z"):
        if g[name] is not None:
            ref.close(host(g[name])[m], want[name][m], mag[name][m], eltype, k, "d" + name)
            assert (host(g[name])[~m] == 7.0).all()
    for name in ("B", "C"):
        ref.close(host(g[name])[m], want[name][m], mag[name][m], eltype, k, "d" + name)
        assert (host(g[name])[~m] == 7.0).all()
    for name in ("A", "D", "bias", "init"):
        if g[name] is not None:
            ref.close(host(g[name]), want[name], mag[name], "Float32", k + c["T"] / 8, "d" + name)


def test_scan_gradient_against_differences(cuda):
    """The kernel's gradient along a direction, against differences of the 64-bit form.  Central differences with
    step 1e-5 err by 1e-10 of the third derivative, far below the gradient's own 32-bit error."""
    c = scan_case([70, 9], 12, 6, 2, 0, 0, True, True, True, True, True, "Float32")
    saved = mk.selective_scan_saved(c["u"], c["A"], seqs=seqs_of(c["spans"]))
    scan_forward(c, saved)
    g = scan_grad(c, saved)
    mk.synchronize(BE)
    v, r = c["v"], gen(1)
    names = {"u": "u", "delta": "delta", "A": "A", "B": "B", "C": "C", "z": "z", "D": "skip", "bias": "bias",
             "init": "init"}

    def value():
        y, last = scan_ref(c)
        return (y * v["dy"]).sum() + (last * v["dlast"]).sum()

    mags = scan_ref(c, grad=True, mag=True)[2]
    for gname, vname in names.items():
        d = r.standard_normal(v[vname].shape)
        kept = v[vname]
        v[vname] = kept + 1e-5 * d
        up = value()
        v[vname] = kept - 1e-5 * d
        down = value()
        v[vname] = kept
        want = (up - down) / 2e-5
        got = (host(g[gname]) * d).sum()
        tol = (2.0**-23 + (k_scan(c) + 20) * 2.0**-24) * (mags[gname] * np.abs(d)).sum() + 1e-5 * abs(want)
        assert abs(got - want) <= tol, gname


def test_scan_state_in_place_in_slots_and_in_pieces(cuda):
    for lens, D in (([300, 0, 2, 77], 300), ([900, 0, 600], 24)):  # whole sequences; pieces
        c = scan_case(lens, D, 16, 1, 0, 0, True, True, True, True, False, "BFloat16")
        pool, pv = dev(gen(2).standard_normal((8, D, 16)))
        slots = [5, 8, 0, 2][:len(lens)]
        h0 = np.stack([pv[k - 1] if k else np.zeros((D, 16)) for k in slots])
        y = out((c["T"], D), "BFloat16")
        mk.selective_scan(y, c["u"], c["delta"], c["A"], c["B"], c["C"], D=c["skip"], z=c["z"], bias=c["bias"],
                          seqs=seqs_of(c["spans"]), init=pool, last=pool, slots=ints(slots))
        mk.synchronize(BE)
        c["v"]["init"] = h0
        wy, wl = scan_ref(c)
        my, ml = scan_ref(c, mag=True)
        ref.close(host(y), wy, my, "BFloat16", k_scan(c))
        for s, k in enumerate(slots):
            if k:
                ref.close(host(pool)[k - 1], wl[s], ml[s], "Float32", k_scan(c))
        rest = [k for k in range(8) if k + 1 not in slots]
        np.testing.assert_array_equal(host(pool)[rest], pv[rest])


def test_scan_equal_lengths_in_place_output(cuda):
    """Sequences of equal length without offsets; y written over u."""
    r = gen(3)
    L, S, D, N = 37, 3, 50, 16
    u, uv = dev(r.standard_normal((S, L, D)), "Float16")
    dl, dv = dev(r.standard_normal((S, L, D)), "Float16")
    A, Av = dev(-np.exp(r.standard_normal((D, N))))
    B, Bv = dev(r.standard_normal((S, L, N)), "Float16")
    C, Cv = dev(r.standard_normal((S, L, N)), "Float16")
    mk.selective_scan(u, u, dl, A, B, C)
    mk.synchronize(BE)
    f = lambda x, n: x.reshape(S * L, *n)  # noqa: E731
    a = (f(uv, (D,)), f(dv, (D,)), Av, f(Bv, (1, N)), f(Cv, (1, N)), np.zeros(D), None, np.zeros(D), True,
         ref.spans_of([L] * S))
    wy, my = ref.scan(*a)[0], ref.scan(*a, mag=True)[0]
    ref.close(host(u).reshape(S * L, D), wy, my, "Float16", 8 * (L + 24))


@pytest.mark.parametrize("eltype", list(TD))
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 1), (3, 33, 16, 1), (40, 128, 16, 2), (2, 30, 5, 3), (2, 24, 64, 1),
                                     (3, 20, 24, 2), (3, 20, 7, 1)])
def test_scan_step(cuda, B, D, N, G, eltype):
    c = scan_case([1] * B, D, N, G, 0, 0, True, True, True, True, False, eltype)
    pool, pv = dev(gen(B).standard_normal((B + 2, D, N)))
    slots = np.arange(B + 2, 2, -1)
    slots[B // 2] = 0 if B > 1 else slots[0]
    for inplace in (False, True):
        nxt = pool if inplace else out((B + 2, D, N))
        y = out((B, D), eltype)
        mk.selective_scan_step(y, nxt, pool, c["u"], c["delta"], c["A"], c["B"], c["C"], D=c["skip"], z=c["z"],
                               bias=c["bias"], slots=ints(slots))
        mk.synchronize(BE)
        c["v"]["init"] = np.stack([pv[k - 1] for k in slots])
        (wy, wl), (my, ml) = scan_ref(c), scan_ref(c, mag=True)
        on = slots > 0
        ref.close(host(y)[on], wy[on], my[on], eltype, k_scan(c))
        assert (host(y)[~on] == 7.0).all()
        ref.close(host(nxt)[slots[on] - 1], wl[on], ml[on], "Float32", k_scan(c))


def test_scan_long_memory_and_extreme_steps(cuda):
    """Decay near one over many tokens, and steps so large that nothing is left of the state."""
    T, D, N = 2000, 4, 16
    r = gen(9)
    u, uv = dev(r.standard_normal((T, D)))
    raw = np.full((T, D), -9.0)
    raw[::97] = 60.0
    dl, dv = dev(raw)
    A, Av = dev(-np.linspace(0.01, 40, D * N).reshape(D, N))
    B, Bv = dev(r.standard_normal((T, 1, N)))
    C, Cv = dev(r.standard_normal((T, 1, N)))
    y = out((T, D))
    mk.selective_scan(y, u, dl, A, B, C)
    mk.synchronize(BE)
    a = (uv, dv, Av, Bv, Cv, np.zeros(D), None, np.zeros(D), True, [(0, T)])
    ref.close(host(y), ref.scan(*a)[0], ref.scan(*a, mag=True)[0], "Float32", 8 * (T + 24))


def test_scan_infinite_rate(cuda):
    """A state that forgets at once (A = -inf): nothing but the last token is in it, at every length of a tile's rest."""
    r = gen(15)
    for T in (1, 3, 8, 33, 700):
        u, uv = dev(r.standard_normal((T, 4)))
        dl, dv = dev(r.standard_normal((T, 4)))
        Av = -np.exp(r.standard_normal((4, 6)))
        Av[:, ::2] = -np.inf
        A, Av = dev(Av)
        B, Bv = dev(r.standard_normal((T, 1, 6)))
        y, last, h0 = out((T, 4)), out((1, 4, 6)), r.standard_normal((1, 4, 6))
        init, h0 = dev(h0)
        mk.selective_scan(y, u, dl, A, B, B, init=init, last=last)
        mk.synchronize(BE)
        a = (uv, dv, Av, Bv, Bv, np.zeros(4), None, np.zeros(4), True, [(0, T)], h0)
        (wy, wl), (my, ml) = ref.scan(*a), ref.scan(*a, mag=True)
        ref.close(host(y), wy, my, "Float32", 8 * (T + 24))
        ref.close(host(last), wl, ml, "Float32", 8 * (T + 24))


# ---- norms -----------------------------------------------------------------------------

NORM = [(1, 1), (3, 7), (5, 64), (2, 100), (33, 256), (3, 1000), (4, 1030), (2, 4096), (3, 4100), (1, 8200), (2, 16384),
        (1, 16383)]


@pytest.mark.parametrize("eltype,rtype", [("Float32", "Float32"), ("BFloat16", "Float32"), ("BFloat16", "BFloat16"),
                                          ("Float16", "Float32"), ("Float16", "Float16")])
@pytest.mark.parametrize("T,D", NORM)
def test_norm(cuda, T, D, eltype, rtype):
    r = gen(T * 1000 + D)
    eps = 1e-5
    R, Rv = dev(2 * r.standard_normal((T, D)), rtype)
    h, hv = dev(r.standard_normal((T, D)), eltype)
    gt, gv = dev(2 * r.standard_normal((T, D)), eltype)
    w, wv = dev(1 + 0.1 * r.standard_normal(D))
    hw, hwv = dev(1 + 0.1 * r.standard_normal(D))
    sc, scv = dev(r.standard_normal(D))
    dy, dyv = dev(r.standard_normal((T, D)), eltype)
    dro, drov = dev(r.standard_normal((T, D)), rtype)
    # which of (h, hw, gate, scale, y, rout) take part
    forms = [(1, 1, 1, 1, 1, 1), (0, 0, 0, 0, 1, 0), (1, 0, 1, 0, 1, 1), (1, 1, 0, 1, 0, 1), (1, 1, 1, 0, 1, 0)]
    for act, (uh, uhw, ug, us, uy, uro) in itertools.product(("silu", "sigmoid"), forms):
        if act == "sigmoid" and not ug:
            continue
        on = lambda c, x: x if c else None  # noqa: E731
        y, ro = on(uy, out((T, D), eltype)), on(uro, out((T, D), rtype))
        mk.block_norm(y, ro, R, on(uy, w), h=on(uh, h), hw=on(uhw, hw), gate=on(ug, gt), act=act, scale=on(us, sc),
                      eps=eps)
        a = (Rv, on(uy, wv), on(uh, hv), on(uhw, hwv), on(ug, gv), act, on(us, scv), eps)
        wy, wro = ref.norm(*a)
        # magnitudes: rout is a difference, so its error is relative to its terms
        term = np.abs(Rv) + np.abs(wro - Rv)
        k = 64 + D / 64
        if uy:
            rms = 1 / np.sqrt((wro**2).mean(-1, keepdims=True) + eps)
            ref.close(host(y), wy, term * rms * np.abs(wv) + np.abs(wy) * (1 + (term**2).mean(-1, keepdims=True) * rms**2),
                      eltype, k, "y")
        if uro:
            ref.close(host(ro), wro, term, rtype, 64, "rout")
        g = {"r": out((T, D), rtype), "w": on(uy, out((D,))), "h": on(uh, out((T, D), eltype)),
             "hw": on(uhw, out((D,))), "gate": on(ug, out((T, D), eltype)), "scale": on(us, out((D,)))}
        mk.block_norm_grad(g["r"], g["w"], on(uy, dy), R, on(uy, w), drout=on(uro, dro), h=on(uh, h), dh=g["h"],
                           hw=on(uhw, hw), dhw=g["hw"], gate=on(ug, gt), dgate=g["gate"], act=act, scale=on(us, sc),
                           dscale=g["scale"], eps=eps)
        mk.synchronize(BE)
        want = ref.norm(*a, dy=on(uy, dyv), drout=on(uro, drov))[2]
        # every gradient is a product of a few factors with one subtraction of a column's mean: errors are
        # relative to the largest value of the column (or, for sums over tokens, of the whole)
        for name, x in g.items():
            if x is None:
                continue
            ww = want[name]
            top = (np.abs(ww).max(-1, keepdims=True) + 1.0) * np.ones_like(ww)
            token = name in ("r", "h", "gate")
            ref.close(host(x), ww, top * (1 + np.abs(Rv).max()), rtype if name == "r" else eltype if token else "Float32",
                      (64 + D / 64) * (1 if token else 1 + T / 8), (act, "d" + name))


@pytest.mark.parametrize("eltype,rtype", [("Float32", "Float32"), ("BFloat16", "Float32"), ("Float16", "Float16")])
@pytest.mark.parametrize("T,D", [(6001, 24), (3001, 72), (1500, 520), (700, 2048), (500, 4096), (900, 1001),
                                 (301, 4104), (300, 8184), (160, 6001)])
def test_norm_many_columns(cuda, T, D, eltype, rtype):
    """More columns than walk at once."""
    test_norm(cuda, T, D, eltype, rtype)


def test_norm_in_place(cuda):
    r = gen(4)
    R, Rv = dev(r.standard_normal((6, 96)))
    h, hv = dev(r.standard_normal((6, 96)), "BFloat16")
    mk.block_norm(None, R, R, None, h=h)
    mk.synchronize(BE)
    ref.close(host(R), Rv + hv, np.abs(Rv) + np.abs(hv), "Float32", 4)


# ---- layouts, streams, graphs, errors -----------------------------------------------------

def test_rows_of_a_projection(cuda):
    """x, z, delta, B, C as rows of one matrix, at offsets that no vector divides."""
    r = gen(6)
    T, D, N, W = 70, 36, 8, 4
    H = 3 * D + 2 * N + 3
    P, Pv = dev(r.standard_normal((T, H)), "BFloat16")
    at = {"x": (1, D), "z": (D + 1, 2 * D), "delta": (2 * D + 2, 3 * D + 1), "B": (3 * D + 3, 3 * D + 2 + N),
          "C": (3 * D + 3 + N, 3 * D + 2 + 2 * N)}
    R = {k: mk.rows(P, lo, hi) for k, (lo, hi) in at.items()}
    V = {k: Pv[:, lo - 1:hi] for k, (lo, hi) in at.items()}
    w, wv = dev(r.standard_normal((W, D)))
    A, Av = dev(-np.exp(r.standard_normal((D, N))))
    x = out((T, D), "BFloat16")
    mk.causal_conv(x, R["x"], w)
    mk.synchronize(BE)
    spans = [(0, T)]
    wx, mx = ref.conv(V["x"], wv, np.zeros(D), True, spans)[0], ref.conv(V["x"], wv, np.zeros(D), True, spans, mag=True)[0]
    ref.close(host(x), wx, mx, "BFloat16", 64)
    xv = host(x)
    Y = out((T, 2 * D + 1), "BFloat16")
    mk.selective_scan(mk.rows(Y, 2, D + 1), x, R["delta"], A, R["B"], R["C"], z=R["z"])
    mk.synchronize(BE)
    a = (xv, V["delta"], Av, V["B"][:, None], V["C"][:, None], np.zeros(D), V["z"], np.zeros(D), True, spans)
    ref.close(host(Y)[:, 1:D + 1], ref.scan(*a)[0], ref.scan(*a, mag=True)[0], "BFloat16", 8 * (T + 24))
    assert (host(Y)[:, 0] == 7.0).all() and (host(Y)[:, D + 1:] == 7.0).all()
    n = out((T, D), "BFloat16")
    one, _ = dev(np.ones(D))
    mk.block_norm(n, None, R["z"], one)
    mk.synchronize(BE)
    wn = ref.norm(V["z"], np.ones(D), None, None, None, "silu", None, 1e-5)[0]
    ref.close(host(n), wn, np.abs(wn), "BFloat16", 64)


def test_prompt_then_single_tokens_equal_the_whole_prompt(cuda):
    """A block as a model runs it: norm, projection, convolution, projections, scan, projection, norm with gate and
    residual; a prompt of 20 tokens and five single ones against one prompt of 25, both in Float32."""
    r = gen(7)
    M, D, N, W, T, K = 48, 64, 16, 4, 25, 20
    f = lambda *s: dev(r.standard_normal(s) / np.sqrt(s[-1]))[0]  # noqa: E731
    # projections: mul!(C, A, B) with A (out, in)
    Win, Wdt, WB, WC, Wout = (mk.MLIRArray((r.standard_normal((o, i)) / np.sqrt(i)).astype(np.float32))
                              for o, i in ((2 * D, M), (D, D), (N, D), (N, D), (M, D)))
    cw, cb, A = f(W, D), f(D), dev(-np.exp(r.standard_normal((D, N))))[0]
    skip, bias, w1, w2, hw, sc = f(D), dev(r.uniform(-4, 0, D))[0], f(M), f(M), f(M), f(M)
    X = r.standard_normal((T, M))
    G = r.standard_normal((T, M))

    def mul(Wm, x):
        y = mk.zeros(BE, "Float32", (Wm.dims[0],) + tuple(x.dims[1:]))
        mk.mul(y, Wm, x)
        return y

    def block(x, gate, n, conv, scan):
        x, gate = dev(x)[0], dev(gate)[0]
        a = out((n, M))
        mk.block_norm(a, None, x, w1)
        p = mul(Win, a)
        xs, z = mk.rows(p, 1, D), mk.rows(p, D + 1, 2 * D)
        c = out((n, D))
        conv(c, xs)
        y = out((n, D))
        scan(y, c, mul(Wdt, c), mul(WB, c), mul(WC, c), z)
        ro, nx = out((n, M)), out((n, M))
        mk.block_norm(nx, ro, x, w2, h=mul(Wout, y), hw=hw, gate=gate, scale=sc)
        mk.synchronize(BE)
        return host(ro), host(nx)

    cs, ss = out((1, W - 1, D), fill=0.0), out((1, D, N), fill=0.0)

    def prompt(keep):
        return (lambda c, x: mk.causal_conv(c, x, cw, bias=cb, last=cs if keep else None),
                lambda y, c, d, B, C, z: mk.selective_scan(y, c, d, A, B, C, D=skip, z=z, bias=bias,
                                                           last=ss if keep else None))

    single = (lambda c, x: mk.causal_conv_step(c, cs, cs, x, cw, bias=cb),
              lambda y, c, d, B, C, z: mk.selective_scan_step(y, ss, ss, c, d, A, B, C, D=skip, z=z, bias=bias))
    whole = block(X, G, T, *prompt(False))
    first = block(X[:K], G[:K], K, *prompt(True))
    for a, b in zip(whole, first):
        np.testing.assert_allclose(b, a[:K], rtol=1e-4, atol=1e-4)
    for t in range(K, T):
        step = block(X[t:t + 1], G[t:t + 1], 1, *single)
        for a, b in zip(whole, step):
            # the projections' 3xTF32 products differ by 2e-6 relative with the number of columns; chains of
            # five operators on values of order one stay two orders below this
            np.testing.assert_allclose(b[0], a[t], rtol=1e-4, atol=1e-4)


def test_two_streams_and_a_replayed_graph(cuda):
    """The same training pass eagerly, on another stream, and captured and replayed: bit for bit the same."""
    c = scan_case([600, 200], 24, 16, 1, 0, 0, True, True, True, True, True, "BFloat16")
    seqs = seqs_of(c["spans"])

    def pass_():
        saved = mk.selective_scan_saved(c["u"], c["A"], seqs=seqs)
        y, last = scan_forward(c, saved)
        g = scan_grad(c, saved)
        return [y, last] + [x for x in g.values() if x is not None]

    want = [host(x) for x in pass_()]
    mk.synchronize(BE)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = pass_()
    s.synchronize()
    for a, b in zip(want, other):
        np.testing.assert_array_equal(a, host(b))
    saved = mk.selective_scan_saved(c["u"], c["A"], seqs=seqs)
    t = c["eltype"]
    y, last = out((c["T"], c["D"]), t), out((c["S"], c["D"], c["N"]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mk.selective_scan(y, c["u"], c["delta"], c["A"], c["B"], c["C"], D=c["skip"], z=c["z"], bias=c["bias"],
                          seqs=seqs, init=c["init"], last=last, saved=saved)
        du = out((c["T"], c["D"]), t)
        g = [out(s_, t_) for s_, t_ in (((c["T"], c["D"]), t), ((c["D"], c["N"]), "Float32"),
                                        ((c["T"], 1, c["N"]), t), ((c["T"], 1, c["N"]), t), ((c["T"], c["D"]), t),
                                        ((c["D"],), "Float32"), ((c["D"],), "Float32"),
                                        ((c["S"], c["D"], c["N"]), "Float32"))]
        mk.selective_scan_grad(du, g[0], g[1], g[2], g[3], c["dy"], c["u"], c["delta"], c["A"], c["B"], c["C"], saved,
                               D=c["skip"], dD=g[5], z=c["z"], dz=g[4], bias=c["bias"], dbias=g[6], seqs=seqs,
                               dinit=g[7], dlast=c["dlast"])
    for _ in range(2):
        graph.replay()
    mk.synchronize(BE)
    got = [y, last, du, g[0], g[1], g[2], g[3], g[5], g[4], g[6], g[7]]
    for a, b in zip(want, got):
        np.testing.assert_array_equal(a, host(b))


@pytest.mark.parametrize("offsets", [[1, 40, 20, 65], [0, 10, 20, 65], [1, 10, 20, 67]])
def test_bad_offsets_are_reported_and_stay_in_bounds(cuda, offsets):
    c = scan_case([64], 20, 16, 1, 0, 0, True, True, True, True, False, "Float32")
    w, _ = dev(gen(1).standard_normal((4, 20)))
    y, bad = out((64, 20)), ints(offsets)
    mk.selective_scan(y, c["u"], c["delta"], c["A"], c["B"], c["C"], seqs=bad)
    with pytest.raises(mk.KernelException, match="offsets"):
        mk.synchronize(BE)
    mk.causal_conv(y, c["u"], w, seqs=bad)
    with pytest.raises(mk.KernelException, match="offsets"):
        mk.synchronize(BE)
    mk.synchronize(BE)


@pytest.mark.parametrize("slots", [[1, 4], [2, 2]])
def test_bad_slots_are_reported(cuda, slots):
    c = scan_case([1, 1], 20, 16, 1, 0, 0, True, True, True, True, False, "Float32")
    w, _ = dev(gen(1).standard_normal((4, 20)))
    ss, cs, y = out((3, 20, 16)), out((3, 3, 20)), out((2, 20))
    calls = [lambda: mk.selective_scan_step(y, ss, ss, c["u"], c["delta"], c["A"], c["B"], c["C"], slots=ints(slots)),
             lambda: mk.causal_conv_step(y, cs, cs, c["u"], w, slots=ints(slots)),
             lambda: mk.selective_scan(y, c["u"], c["delta"], c["A"], c["B"], c["C"], seqs=ints([1, 2, 3]), last=ss,
                                       slots=ints(slots)),
             lambda: mk.causal_conv(y, c["u"], w, seqs=ints([1, 2, 3]), last=cs, slots=ints(slots))]
    for call in calls:
        call()
        with pytest.raises(mk.KernelException, match="slot"):
            mk.synchronize(BE)


def test_columns_outside_the_sequences_are_never_read(cuda):
    """NaN in front of, between batches' ends and behind the sequences, and in states that no sequence uses."""
    lens, D, N, W, lead, tail = [37, 0, 50], 40, 16, 4, 5, 9
    c = scan_case(lens, D, N, 1, lead, tail, True, True, True, True, True, "BFloat16")
    m = torch.from_numpy(inside(c["spans"], c["T"])).cuda()

    def poison(a):
        a.storage.view(c["T"], -1)[~m] = float("nan")

    seqs = seqs_of(c["spans"])
    w, _ = dev(gen(3).standard_normal((W, D)))
    h0, _ = dev(gen(4).standard_normal((3, W - 1, D)), "BFloat16")

    def everything():
        saved = mk.selective_scan_saved(c["u"], c["A"], seqs=seqs)
        y, last = scan_forward(c, saved)
        g = scan_grad(c, saved)
        t = "BFloat16"
        cy, dx, dw = out((c["T"], D), t), out((c["T"], D), t), out((W, D))
        cl, di = out((3, W - 1, D), t), out((3, W - 1, D), t)
        mk.causal_conv(cy, c["u"], w, seqs=seqs, init=h0, last=cl)
        mk.causal_conv_grad(dx, dw, c["dy"], c["u"], w, seqs=seqs, init=h0, dinit=di, dlast=h0)
        mk.synchronize(BE)
        return [host(x) for x in [y, last, cy, dx, dw, cl, di] + [x for x in g.values() if x is not None]]

    want = everything()
    for k in ("u", "delta", "z", "B", "C", "dy"):
        poison(c[k])
    for a, b in zip(want, everything()):
        assert np.isfinite(b).all()
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("N", [16, 7])
def test_many_channels_in_pieces(cuda, N):
    """Enough tokens and channels for two channels per lane in pieces; the first and the last group are compared."""
    D, G = 2048, 32
    c = scan_case([2600, 0, 2000, 437], D, N, G, 0, 0, True, True, True, True, True, "BFloat16")
    saved = mk.selective_scan_saved(c["u"], c["A"], seqs=seqs_of(c["spans"]))
    y, last = scan_forward(c, saved)
    g = scan_grad(c, saved)
    mk.synchronize(BE)
    ch, gr = np.r_[:D // G, D - D // G:D], [0, G - 1]
    v = c["v"]
    sub = dict(c, D=2 * (D // G), v={k: v[k][:, ch] for k in ("u", "delta", "z", "dy", "init", "dlast")}
               | {k: v[k][ch] for k in ("A", "skip", "bias")} | {k: v[k][:, gr] for k in ("B", "C")})
    (wy, wl, wg), (my, ml, mg) = scan_ref(sub, True), scan_ref(sub, True, True)
    ref.close(host(y)[:, ch], wy, my, "BFloat16", k_scan(c))
    ref.close(host(last)[:, ch], wl, ml, "Float32", k_scan(c))
    for name in ("u", "delta", "z"):
        ref.close(host(g[name])[:, ch], wg[name], mg[name], "BFloat16", k_scan(c), name)
    for name in ("B", "C"):
        ref.close(host(g[name])[:, gr], wg[name], mg[name], "BFloat16", k_scan(c), name)
    for name in ("A", "D", "bias"):
        ref.close(host(g[name])[ch], wg[name], mg[name], "Float32", k_scan(c) + c["T"] / 8, name)
    ref.close(host(g["init"])[:, ch], wg["init"], mg["init"], "Float32", k_scan(c) + c["T"] / 8, "init")


def test_pieces_behind_columns_of_no_sequence(cuda):
    """Sequences cut into pieces behind more uncovered columns than a piece has (NaN there): they stay as they were."""
    c = scan_case([600, 0, 90], 33, 16, 1, 270, 130, True, True, True, True, True, "Float32")
    m = inside(c["spans"], c["T"])
    for k in ("u", "delta", "z", "B", "C", "dy"):
        c[k].storage.view(c["T"], -1)[~torch.from_numpy(m).cuda()] = float("nan")
    saved = mk.selective_scan_saved(c["u"], c["A"], seqs=seqs_of(c["spans"]))
    y, last = scan_forward(c, saved)
    g = scan_grad(c, saved)
    mk.synchronize(BE)
    (wy, wl, wg), (my, ml, mg) = scan_ref(c, True), scan_ref(c, True, True)
    ref.close(host(y)[m], wy[m], my[m], "Float32", k_scan(c))
    ref.close(host(last), wl, ml, "Float32", k_scan(c))
    assert (host(y)[~m] == 7.0).all()
    for name in ("u", "delta", "z", "B", "C"):
        ref.close(host(g[name])[m], wg[name][m], mg[name][m], "Float32", k_scan(c), name)
        assert (host(g[name])[~m] == 7.0).all(), name
    for name in ("A", "D", "bias", "init"):
        ref.close(host(g[name]), wg[name], mg[name], "Float32", k_scan(c) + c["T"] / 8, name)


def test_columns_beyond_two_to_the_31_elements(cuda):
    """Rows of a matrix of 2.2e9 elements: the last columns against the same columns on their own."""
    D, T, ld = 64, 2100, 1 << 20
    parent = mk.MLIRArray(torch.zeros(ld * T, dtype=torch.bfloat16, device="cuda"), dims=(ld, T))
    x = mk.rows(parent, ld - D + 1, ld)
    view = parent.storage.view(T, ld)[:, ld - D:]
    r = gen(12)
    xs, _ = dev(r.standard_normal((T, D)), "BFloat16")
    view.copy_(xs.storage.view(T, D))
    w, _ = dev(r.standard_normal((4, D)))
    A, _ = dev(-np.exp(r.standard_normal((D, 4))))
    B, _ = dev(r.standard_normal((T, 4)), "BFloat16")
    one, _ = dev(np.ones(D))
    for call in (lambda y, a: mk.causal_conv(y, a, w), lambda y, a: mk.selective_scan(y, a, a, A, B, B, z=a),
                 lambda y, a: mk.block_norm(y, None, a, one)):
        far, near = out((T, D), "BFloat16"), out((T, D), "BFloat16")
        call(far, x)
        call(near, xs)
        mk.synchronize(BE)
        np.testing.assert_array_equal(host(far), host(near))


def test_many_short_sequences(cuda):
    """More sequences than a warp looks over at once, most of them short or empty."""
    r = gen(13)
    lens = list(r.integers(0, 4, 1500)) + [70] + list(r.integers(0, 2, 300))
    c = scan_case([int(n) for n in lens], 16, 4, 1, 1, 2, True, True, True, True, True, "Float32")
    saved = mk.selective_scan_saved(c["u"], c["A"], seqs=seqs_of(c["spans"]))
    y, last = scan_forward(c, saved)
    g = scan_grad(c, saved)
    w, wv = dev(r.standard_normal((4, 16)))
    x, xv = c["u"], c["v"]["u"]
    cy, dx, dw = out((c["T"], 16)), out((c["T"], 16)), out((4, 16))
    mk.causal_conv(cy, x, w, seqs=seqs_of(c["spans"]))
    mk.causal_conv_grad(dx, dw, c["dy"], x, w, seqs=seqs_of(c["spans"]))
    mk.synchronize(BE)
    m = inside(c["spans"], c["T"])
    (wy, wl, wg), (my, ml, mg) = scan_ref(c, True), scan_ref(c, True, True)
    ref.close(host(y)[m], wy[m], my[m], "Float32", k_scan(c))
    ref.close(host(last), wl, ml, "Float32", k_scan(c))
    for name in ("u", "delta", "z", "B", "C"):
        ref.close(host(g[name])[m], wg[name][m], mg[name][m], "Float32", k_scan(c), name)
    for name in ("A", "D", "bias", "init"):
        ref.close(host(g[name]), wg[name], mg[name], "Float32", k_scan(c) + c["T"] / 8, name)
    a = (xv, wv, np.zeros(16), True, c["spans"], None, c["v"]["dy"])
    want, mag = ref.conv(*a), ref.conv(*a, mag=True)
    ref.close(host(cy)[m], want[0][m], mag[0][m], "Float32", 64)
    ref.close(host(dx)[m], want[2][m], mag[2][m], "Float32", 64)
    ref.close(host(dw), want[3], mag[3], "Float32", 64 + c["T"] / 8)


def test_nothing_to_do(cuda):
    """No tokens, no sequences, no batch entries."""
    A, _ = dev(-np.ones((8, 16)))
    w, _ = dev(np.ones((4, 8)))
    e = lambda *s: out(s)  # noqa: E731
    mk.causal_conv(e(0, 8), e(0, 8), w, seqs=ints([1]))
    mk.selective_scan(e(0, 8), e(0, 8), e(0, 8), A, e(0, 16), e(0, 16), seqs=ints([1]))
    mk.causal_conv_step(e(0, 8), e(0, 3, 8), e(0, 3, 8), e(0, 8), w)
    mk.selective_scan_step(e(0, 8), e(0, 8, 16), e(0, 8, 16), e(0, 8), e(0, 8), A, e(0, 16), e(0, 16))
    g1, g2 = e(8), e(4, 8)
    mk.block_norm_grad(e(0, 8), g1, e(0, 8), e(0, 8), dev(np.ones(8))[0])
    mk.causal_conv_grad(e(0, 8), g2, e(0, 8), e(0, 8), w, seqs=ints([1]))
    dA = e(8, 16)
    saved = mk.selective_scan_saved(e(0, 8), A, seqs=ints([1]))
    mk.selective_scan_grad(e(0, 8), e(0, 8), dA, e(0, 16), e(0, 16), e(0, 8), e(0, 8), e(0, 8), A, e(0, 16), e(0, 16),
                           saved, seqs=ints([1]))
    last = out((2, 8, 16))
    mk.selective_scan(e(0, 8), e(0, 8), e(0, 8), A, e(0, 16), e(0, 16), seqs=ints([1, 1, 1]), last=last)
    mk.synchronize(BE)
    assert (host(g1) == 0).all() and (host(g2) == 0).all() and (host(dA) == 0).all() and (host(last) == 0).all()


def test_half_types_of_arrays(cuda):
    """Float16 and BFloat16 arrays: made, copied, pooled, rounded to the nearest."""
    x = np.array([1.0, 1.00390625, -2.5, 3.0e38], np.float32)
    b = mk.MLIRArray(x, eltype="BFloat16")
    np.testing.assert_array_equal(mk.Array(b), torch.from_numpy(x).to(torch.bfloat16).float().numpy())
    assert mk.ones(BE, "Float16", 3).to_numpy().dtype == np.float16
    p = mk.pool_allocate("BFloat16", (2, 3))
    mk.copyto(BE, p, np.arange(6, dtype=np.float32).reshape(2, 3))
    np.testing.assert_array_equal(mk.Array(p), np.arange(6, dtype=np.float32).reshape(2, 3))


# ---- far gates, rates and offsets ------------------------------------------------------------

# A sigmoid below the smallest normal number counts as zero: 2^-126, times a gate of at most 110 and factors below
# 1e5, is less than this.
FLUSH = 1e-30


@pytest.fixture
def far_sig(monkeypatch):
    """The sigmoid with full relative precision far below zero, where 1 + tanh(x / 2) has none left."""
    def sig(x):
        e = np.exp(-np.abs(x))
        return np.where(x < 0, e, 1.0) / (1.0 + e)
    monkeypatch.setattr(ref, "sig", sig)


def near(got, want, mag, eltype, k, what=""):
    """`close`, and FLUSH beside it."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    ok = np.abs(got - want) <= FLUSH
    ref.close(np.where(ok, want, got), want, mag, eltype, k, what)


@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("eltype", ["Float32", "BFloat16"])
@pytest.mark.parametrize("D", [1000, 1001, 4400])
def test_norm_far_gates(cuda, far_sig, D, eltype, act):
    """Gates from -110 to 110 (e^110 is beyond Float32), infinite ones where the activation is finite."""
    r, T = gen(D), 16
    gate = r.permutation(np.linspace(-110, 110, T * D)).reshape(T, D)
    if act == "sigmoid":
        gate[3, 5:9] = [np.inf, -np.inf, np.inf, -np.inf]
    gt, gv = dev(gate, eltype)
    R, Rv = dev(r.standard_normal((T, D)))
    h, hv = dev(r.standard_normal((T, D)), eltype)
    w, wv = dev(1 + 0.1 * r.standard_normal(D))
    hw, hwv = dev(1 + 0.1 * r.standard_normal(D))
    dy, dyv = dev(r.standard_normal((T, D)), eltype)
    dro, drov = dev(r.standard_normal((T, D)))
    y, ro = out((T, D), eltype), out((T, D))
    mk.block_norm(y, ro, R, w, h=h, hw=hw, gate=gt, act=act)
    g = {"r": out((T, D)), "w": out((D,)), "h": out((T, D), eltype), "hw": out((D,)), "gate": out((T, D), eltype)}
    mk.block_norm_grad(g["r"], g["w"], dy, R, w, drout=dro, h=h, dh=g["h"], hw=hw, dhw=g["hw"], gate=gt,
                       dgate=g["gate"], act=act)
    mk.synchronize(BE)
    wy, wro, want = ref.norm(Rv, wv, hv, hwv, gv, act, None, 1e-5, dy=dyv, drout=drov)
    term, k = np.abs(Rv) + np.abs(wro - Rv), 64 + D / 64
    # 16-bit gates: the exponent's rounding adds 110 units
    k += 110 if eltype != "Float32" else 0
    rms = 1 / np.sqrt((wro**2).mean(-1, keepdims=True) + 1e-5)
    near(host(ro), wro, term, "Float32", k, "rout")
    near(host(y), wy, term * rms * np.abs(wv) + np.abs(wy) * (1 + (term**2).mean(-1, keepdims=True) * rms**2), eltype,
         k, "y")
    for name, x in g.items():  # errors are relative to a column's largest value, as in test_norm; rout reaches 110 |n|
        top = (np.abs(want[name]).max(-1, keepdims=True) + 1.0) * np.ones_like(want[name])
        token = name in ("r", "h", "gate")
        near(host(x), want[name], top * (1 + np.abs(term).max()), "Float32" if name == "r" or not token else eltype,
             k * (1 if token else 1 + T / 8), (act, "d" + name))


@pytest.mark.parametrize("eltype", ["Float32", "BFloat16"])
@pytest.mark.parametrize("D", [64, 33])
def test_conv_far_inputs(cuda, far_sig, D, eltype):
    """Values in front of the silu from -110 to 110.  Their own W + 1 roundings move it by up to 111 times as much."""
    r, T, W = gen(D), 200, 2
    x, xv = dev(r.permutation(np.linspace(-88, 88, T * D)).reshape(T, D), eltype)
    w, wv = dev(np.stack([np.full(D, 0.25), np.ones(D)]))
    dy, dyv = dev(r.standard_normal((T, D)), eltype)
    y, dx, dw = out((T, D), eltype), out((T, D), eltype), out((W, D))
    mk.causal_conv(y, x, w)
    mk.causal_conv_grad(dx, dw, dy, x, w)
    st, y1 = out((T, W - 1, D), eltype, 0.0), out((T, D), eltype)
    mk.causal_conv_step(y1, st, st, x, w)
    mk.synchronize(BE)
    a = (xv, wv, np.zeros(D), True, [(0, T)], None, dyv)
    want, mag, k = ref.conv(*a), ref.conv(*a, mag=True), 64 + 3 * 111 + 110
    near(host(y), want[0], mag[0], eltype, k, "y")
    near(host(dx), want[2], mag[2], eltype, k, "dx")
    near(host(dw), want[3], mag[3], "Float32", k + T / 8, "dw")
    a = (xv, wv, np.zeros(D), True, ref.spans_of([1] * T))
    near(host(y1), ref.conv(*a)[0], ref.conv(*a, mag=True)[0], eltype, k, "step")


@pytest.mark.parametrize("eltype", ["Float32", "BFloat16"])
@pytest.mark.parametrize("D", [64, 33])
def test_scan_far_gates(cuda, far_sig, D, eltype):
    """Gates from -110 to 110, in whole sequences, pieces and single tokens."""
    for lens in ([40] * 5, [640]):
        c = scan_case(lens, D, 16, 1, 0, 0, True, True, True, True, True, eltype)
        c["z"], c["v"]["z"] = dev(gen(D).permutation(np.linspace(-110, 110, c["T"] * D)).reshape(c["T"], D), eltype)
        saved = mk.selective_scan_saved(c["u"], c["A"], seqs=seqs_of(c["spans"]))
        y, _ = scan_forward(c, saved)
        g = scan_grad(c, saved)
        mk.synchronize(BE)
        (wy, _, want), (my, _, mag) = scan_ref(c, True), scan_ref(c, True, True)
        k = k_scan(c) + 110
        near(host(y), wy, my, eltype, k, "y")
        for name in ("u", "delta", "z", "B", "C"):
            near(host(g[name]), want[name], mag[name], eltype, k, "d" + name)
        for name in ("A", "D", "bias", "init"):
            near(host(g[name]), want[name], mag[name], "Float32", k + c["T"] / 8, "d" + name)
    c = scan_case([1] * 60, D, 16, 1, 0, 0, True, True, True, True, True, eltype)
    c["z"], c["v"]["z"] = dev(gen(D).permutation(np.linspace(-110, 110, 60 * D)).reshape(60, D), eltype)
    y, nxt = out((60, D), eltype), out((60, D, 16))
    mk.selective_scan_step(y, nxt, c["init"], c["u"], c["delta"], c["A"], c["B"], c["C"], D=c["skip"], z=c["z"],
                           bias=c["bias"])
    mk.synchronize(BE)
    near(host(y), scan_ref(c)[0], scan_ref(c, mag=True)[0], eltype, k_scan(c) + 110, "step")


@pytest.mark.parametrize("offsets", [[1, 501, 101, 1025], [1, 1001, 20, 30, 1025], [1, 2000, 700, 1025],
                                     [-5, 300, 200, 1025]])
def test_bad_offsets_are_reported_in_pieces(cuda, offsets):
    """The same where sequences are cut: every offset is looked at, whichever sequence a piece is taken for."""
    c = scan_case([1024], 20, 16, 1, 0, 0, True, True, True, True, False, "Float32")
    bad, S = ints(offsets), len(offsets) - 1
    saved = mk.selective_scan_saved(c["u"], c["A"], seqs=bad)
    saved.storage.zero_()
    y, last = out((1024, 20)), out((S, 20, 16))
    mk.selective_scan(y, c["u"], c["delta"], c["A"], c["B"], c["C"], seqs=bad, last=last, saved=saved)
    with pytest.raises(mk.KernelException, match="offsets"):
        mk.synchronize(BE)
    du, dd, dA, dB, dC = (out(s) for s in ((1024, 20), (1024, 20), (20, 16), (1024, 16), (1024, 16)))
    mk.selective_scan_grad(du, dd, dA, dB, dC, c["dy"], c["u"], c["delta"], c["A"], c["B"], c["C"], saved, seqs=bad)
    with pytest.raises(mk.KernelException, match="offsets"):
        mk.synchronize(BE)
    mk.synchronize(BE)


@pytest.mark.parametrize("eltype,D", [("Float32", 33), ("Float32", 96), ("BFloat16", 96), ("BFloat16", 33),
                                      ("BFloat16", 4104), ("Float32", 4104), ("BFloat16", 8200)])
def test_norm_gradient_of_absent_parts(cuda, D, eltype):
    """Without dy the norm of rout takes no part: infinite and undefined values of r stay out of the gradients.
    Without hw that of h does not: neither do infinite values of h."""
    r, T = gen(D), 5
    Rv = r.standard_normal((T, D))
    Rv[1, ::7], Rv[2, ::5], Rv[3, 0] = np.inf, -np.inf, np.nan
    R, _ = dev(Rv)
    h, hv = dev(r.standard_normal((T, D)), eltype)
    gt, gv = dev(r.standard_normal((T, D)), eltype)
    hw, hwv = dev(1 + 0.1 * r.standard_normal(D))
    sc, scv = dev(r.standard_normal(D))
    dro, drov = dev(r.standard_normal((T, D)))
    dr = out((T, D))
    mk.block_norm_grad(dr, None, None, R, None, drout=dro)
    mk.synchronize(BE)
    np.testing.assert_array_equal(host(dr), drov)
    dr, dh, dhw, dg, ds = out((T, D)), out((T, D), eltype), out((D,)), out((T, D), eltype), out((D,))
    mk.block_norm_grad(dr, None, None, R, None, drout=dro, h=h, dh=dh, hw=hw, dhw=dhw, gate=gt, dgate=dg, scale=sc,
                       dscale=ds)
    mk.synchronize(BE)
    np.testing.assert_array_equal(host(dr), drov)
    want = ref.norm(np.zeros((T, D)), None, hv, hwv, gv, "silu", scv, 1e-5, drout=drov)[2]
    for name, x in (("h", dh), ("hw", dhw), ("gate", dg), ("scale", ds)):
        top = (np.abs(want[name]).max(-1, keepdims=True) + 1.0) * np.ones_like(want[name])
        ref.close(host(x), want[name], top, eltype if name in ("h", "gate") else "Float32", (64 + D / 64) * (1 + T / 8),
                  name)
    hv[0, ::3], hv[4, -1] = np.inf, -np.inf
    h, _ = dev(hv, eltype)
    dr, dh = out((T, D)), out((T, D), eltype)
    mk.block_norm_grad(dr, None, None, R, None, drout=dro, h=h, dh=dh)
    mk.synchronize(BE)
    np.testing.assert_array_equal(host(dr), drov)
    ref.close(host(dh), drov, np.abs(drov), eltype, 4, "dh without hw")


@pytest.mark.parametrize("eltype", list(TD))
@pytest.mark.parametrize("B,D,N,G", [(80, 516, 16, 1), (60, 700, 8, 1), (75, 520, 7, 2), (100, 390, 24, 3),
                                     (60, 660, 13, 1), (60, 520, 64, 1), (70, 640, 3, 1)])
def test_scan_step_of_a_serving_batch(cuda, B, D, N, G, eltype):
    """Enough entries and channels for several channels per thread, the last of a tile beyond the group's end."""
    test_scan_step(cuda, B, D, N, G, eltype)


@pytest.mark.parametrize("D,N,G,eltype", [(4096, 16, 32, "BFloat16"), (4096, 7, 32, "Float16"), (4096, 24, 32, "BFloat16"),
                                          (4096, 16, 32, "Float32"), (4096, 7, 32, "Float32"),
                                          (4095, 16, 35, "BFloat16"), (2048, 64, 16, "Float16")])
def test_gradients_of_many_sequences(cuda, D, N, G, eltype):
    """Several sequences for each block of the gradient, two channels per lane or one; the first and the last group
    are compared."""
    lens = [int(n) for n in gen(D + N).integers(0, 40, 80)]
    c = scan_case(lens, D, N, G, 1, 2, True, True, True, True, True, eltype)
    saved = mk.selective_scan_saved(c["u"], c["A"], seqs=seqs_of(c["spans"]))
    y, last = scan_forward(c, saved)
    g = scan_grad(c, saved)
    mk.synchronize(BE)
    ch, gr, m = np.r_[:D // G, D - D // G:D], [0, G - 1], inside(c["spans"], c["T"])
    v = c["v"]
    sub = dict(c, D=2 * (D // G), v={k: v[k][:, ch] for k in ("u", "delta", "z", "dy", "init", "dlast")}
               | {k: v[k][ch] for k in ("A", "skip", "bias")} | {k: v[k][:, gr] for k in ("B", "C")})
    (wy, wl, wg), (my, ml, mg) = scan_ref(sub, True), scan_ref(sub, True, True)
    ref.close(host(y)[m][:, ch], wy[m], my[m], eltype, k_scan(c))
    ref.close(host(last)[:, ch], wl, ml, "Float32", k_scan(c))
    for name in ("u", "delta", "z"):
        ref.close(host(g[name])[m][:, ch], wg[name][m], mg[name][m], eltype, k_scan(c), name)
    for name in ("B", "C"):
        ref.close(host(g[name])[m][:, gr], wg[name][m], mg[name][m], eltype, k_scan(c), name)
    for name in ("A", "D", "bias"):
        ref.close(host(g[name])[ch], wg[name], mg[name], "Float32", k_scan(c) + c["T"] / 8, name)
    ref.close(host(g["init"])[:, ch], wg["init"], mg["init"], "Float32", k_scan(c) + c["T"] / 8, "init")


def test_scan_gradient_workspace(cuda):
    """The sums of dB and dC for every tile of channels: 8 bytes per token, row of B and tile of 32 channels (64 with
    two per lane, 16 beyond 32 states), a few MB of parts beside them.  Only the size is asked for."""
    p = 1 << 20  # never followed
    for T, D, N, G, tile in ((8192, 4096, 16, 1, 64), (8192, 4096, 24, 1, 32), (8192, 4096, 64, 1, 16),
                             (1 << 20, 8192, 16, 8, 64)):
        a = mk._lib.ScanArgs(type=2, softplus=1, D=D, N=N, G=G, T=T, nseq=8, len=T // 8, u=p, ldu=D, delta=p, lddelta=D,
                             dy=p, lddy=D, du=p, lddu=D, ddelta=p, ldddelta=D)
        n = ctypes.c_size_t()
        mk._lib.check(mk._lib.lib().mk_selective_scan_grad_workspace(a, n), "workspace")
        sums = 8 * T * G * N * (D // G // tile)
        assert sums <= n.value <= sums + 8 * D * (N + 2) * 4 + 1024, (T, D, N, G)
