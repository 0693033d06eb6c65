"""State space operators, what needs no GPU: the argument structs against the header, and the calls that the C entry
points and the Python layer refuse before anything is launched (the pointers below are never followed)."""
import ctypes as C
import subprocess

import numpy as np
import pytest
import torch

import cutilecpu_b200 as mk
import statespace_ref as ref
from conftest import ROOT
from cutilecpu_b200 import _lib

P = 1 << 20  # a pointer that is aligned and never followed
STRUCTS = {"mk_conv_args": _lib.ConvArgs, "mk_conv_step_args": _lib.ConvStepArgs, "mk_scan_args": _lib.ScanArgs,
           "mk_scan_step_args": _lib.ScanStepArgs, "mk_norm_args": _lib.NormArgs}


def test_structs_match_the_header(tmp_path):
    lines = []
    for name, s in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in s._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mk_kernels.h"\nint main(void) {%s return 0;}'
                   % "\n".join(lines))
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True,
                                                       text=True).stdout.splitlines())
    for name, s in STRUCTS.items():
        assert int(got[name]) == C.sizeof(s)
        for f, _ in s._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(s, f).offset, (name, f)


def conv(**more):
    a = dict(type=2, width=4, D=8, T=16, nseq=1, len=16, x=P, ldx=8, y=2 * P, ldy=8, w=P, dy=P, lddy=8, dx=3 * P,
             lddx=8, dw=P)
    return _lib.ConvArgs(**{**a, **more})


def scan(**more):
    a = dict(type=1, D=8, N=16, G=2, T=16, nseq=2, len=8, u=P, ldu=8, delta=P, lddelta=8, B=P, ldb=32, C=P, ldc=32, A=P,
             y=2 * P, ldy=8, saved=P, dy=P, lddy=8, du=P, lddu=8, ddelta=P, ldddelta=8, dB=P, lddb=32, dC=P, lddc=32,
             dA=P)
    return _lib.ScanArgs(**{**a, **more})


def norm(**more):
    a = dict(type=2, rtype=0, D=8, T=4, eps=1e-5, r=P, ldr=8, y=P, ldy=8, w=P, dy=P, lddy=8, dr=P, lddr=8, dw=P)
    return _lib.NormArgs(**{**a, **more})


CASES = [
    ("mk_causal_conv", conv(type=3), "element type"),
    ("mk_causal_conv", conv(width=1), "2 to 4 taps"),
    ("mk_causal_conv", conv(width=5), "2 to 4 taps"),
    ("mk_causal_conv", conv(D=0), "no channels"),
    ("mk_causal_conv", conv(T=-1), "negative"),
    ("mk_causal_conv", conv(len=15), "nseq \\* len"),
    ("mk_causal_conv", conv(T=0, nseq=4, len=1 << 62), "nseq \\* len"),  # the product passes 64 bits
    ("mk_causal_conv", conv(slots=P, nslots=4, seqs=P, nseq=(1 << 20) + 1), "2\\^20 entries"),
    ("mk_causal_conv", conv(x=None), "x is null"),
    ("mk_causal_conv", conv(ldx=7), "leading dimension"),
    ("mk_causal_conv", conv(x=P + 1), "element-aligned"),
    ("mk_causal_conv", conv(w=None), "w is null"),
    ("mk_causal_conv", conv(y=P), "y must not be x"),
    ("mk_causal_conv", conv(slots=P, nslots=-1), "slots"),
    ("mk_causal_conv", conv(D=(1 << 20) + 1, ldx=1 << 21, ldy=1 << 21), "2\\^20 channels"),
    ("mk_causal_conv_grad", conv(dx=P), "dx must not be"),
    ("mk_causal_conv_grad", conv(dw=None), "dw is null"),
    ("mk_causal_conv_grad", conv(slots=P), "slots are for serving"),
    ("mk_causal_conv_step", _lib.ConvStepArgs(type=0, width=4, D=4, B=1, x=P, ldx=4, y=P, ldy=4, w=P, next=P), "state"),
    ("mk_causal_conv_step", _lib.ConvStepArgs(type=0, width=4, D=4, B=(1 << 20) + 1, x=P, ldx=4, y=P, ldy=4, w=P, next=P,
                                              state=P, slots=P, nslots=4), "2\\^20 entries"),
    ("mk_selective_scan", scan(T=0, nseq=4, len=1 << 62), "nseq \\* len"),
    ("mk_selective_scan", scan(slots=P, nslots=4, seqs=P, nseq=(1 << 20) + 1), "2\\^20 entries"),
    ("mk_selective_scan", scan(N=0), "1 to 64 states"),
    ("mk_selective_scan", scan(N=65), "1 to 64 states"),
    ("mk_selective_scan", scan(G=3), "groups"),
    ("mk_selective_scan", scan(ldb=31), "leading dimension"),
    ("mk_selective_scan", scan(A=None), "A is null"),
    ("mk_selective_scan", scan(A=P + 4), "16-byte aligned"),
    ("mk_selective_scan", scan(init=P + 8), "16-byte aligned"),
    ("mk_selective_scan", scan(y=None), "y is null"),
    ("mk_selective_scan", scan(z=P, ldz=4), "leading dimension"),
    ("mk_selective_scan", scan(len=9), "nseq \\* len"),
    ("mk_selective_scan_grad", scan(saved=None), "saved is null"),
    ("mk_selective_scan_grad", scan(z=P, ldz=8), "dz is needed"),
    ("mk_selective_scan_grad", scan(bias=P), "dbias"),
    ("mk_selective_scan_grad", scan(slots=P), "slots are for serving"),
    ("mk_selective_scan_step", _lib.ScanStepArgs(type=0, D=4, N=4, G=1, B=1), "u is null"),
    ("mk_block_norm", norm(type=1, rtype=2), "Float32 or of the type"),
    ("mk_block_norm", norm(D=16385, ldr=16385), "16384"),
    ("mk_block_norm", norm(eps=-1.0), "eps"),
    ("mk_block_norm", norm(eps=float("nan")), "eps"),
    ("mk_block_norm", norm(act=2), "activation"),
    ("mk_block_norm", norm(gate=P, ldgate=8), "belong to h"),
    ("mk_block_norm", norm(w=None), "given together"),
    ("mk_block_norm", norm(y=None, w=None), "neither"),
    ("mk_block_norm_grad", norm(dy=None, w=None, dw=None), "neither"),
    ("mk_block_norm_grad", norm(dw=None), "dw, dhw"),
    ("mk_block_norm_grad", norm(h=P, ldh=8), "dh and dgate"),
]


@pytest.mark.parametrize("entry,args,msg", CASES)
def test_c_entry_refuses(entry, args, msg):
    L = _lib.lib()
    assert getattr(L, entry)(args, None) == _lib.MK_ERR_INVALID
    with pytest.raises(mk.MLIRKernelsError, match=msg):
        _lib.check(_lib.MK_ERR_INVALID, entry)


def test_null_arguments_are_refused():
    L = _lib.lib()
    for entry in ("mk_causal_conv", "mk_causal_conv_grad", "mk_causal_conv_step", "mk_selective_scan",
                  "mk_selective_scan_grad", "mk_selective_scan_step", "mk_block_norm", "mk_block_norm_grad"):
        assert getattr(L, entry)(None, None) == _lib.MK_ERR_INVALID
    n = C.c_size_t()
    for entry in ("mk_causal_conv_grad_workspace", "mk_selective_scan_workspace", "mk_selective_scan_grad_workspace",
                  "mk_block_norm_grad_workspace"):
        assert getattr(L, entry)(None, n) == _lib.MK_ERR_INVALID


def fake(dims, eltype="Float32"):
    """An array in host memory: enough for the checks in front of a launch."""
    a = mk.MLIRArray.__new__(mk.MLIRArray)
    a.dims, a.eltype = tuple(dims), eltype
    a.storage = torch.zeros(int(np.prod(dims)), dtype={"Float32": torch.float32, "Int32": torch.int32,
                                                       "BFloat16": torch.bfloat16, "Float64": torch.float64}[eltype])
    return a


def test_python_layer_refuses():
    x, y, w, A, B = fake((8, 16)), fake((8, 16)), fake((8, 4)), fake((16, 8)), fake((16, 16))
    bad = [
        (lambda: mk.causal_conv(y, np.zeros((8, 16)), w), "must be an MLIRArray"),
        (lambda: mk.causal_conv(y, fake((8, 16), "Float64"), w), "element type Float64"),
        (lambda: mk.causal_conv(fake((8, 16), "BFloat16"), x, w), "expected Float32"),
        (lambda: mk.causal_conv(fake((8, 15)), x, w), "expected 8 x 16"),
        (lambda: mk.causal_conv(y, x, fake((4, 8))), "`w` must be"),
        (lambda: mk.causal_conv(y, x, w, bias=fake((7,))), "`bias` has 7"),
        (lambda: mk.causal_conv(y, x, w, seqs=fake((2,))), "`seqs` has element type"),
        (lambda: mk.causal_conv(y, x, w, seqs=fake((0,), "Int32")), "no entries"),
        (lambda: mk.causal_conv(y, x, w, init=fake((8, 3, 2))), "`init` has 48"),
        (lambda: mk.causal_conv(y, x, w, init=fake((8, 3, 2)), last=fake((8, 3, 4)), slots=fake((1,), "Int32")),
         "different numbers"),
        (lambda: mk.causal_conv(y, x, w, slots=fake((2,), "Int32")), "`slots` has 2"),
        (lambda: mk.selective_scan(y, x, x, fake((16, 7)), B, B), "`A` must be"),
        (lambda: mk.selective_scan(y, x, x, A, fake((15, 16)), B), "`B` has dims"),
        (lambda: mk.selective_scan(y, x, x, A, B, fake((32, 16))), "`C` has dims"),
        (lambda: mk.selective_scan(y, x, x, A, B, B, saved=fake((16, 8, 2))), "`saved` has"),
        (lambda: mk.selective_scan_grad(y, y, A, B, B, y, x, x, A, B, B, A, z=x), "`dz` is needed"),
        (lambda: mk.selective_scan_step(y, fake((16, 8, 16)), fake((16, 8, 15)), x, x, A, B, B), "`state` has"),
        (lambda: mk.block_norm(None, None, x, None), "neither"),
        (lambda: mk.block_norm(y, None, x, None), "given together"),
        (lambda: mk.block_norm(y, None, x, fake((8,)), gate=x), "belong to `h`"),
        (lambda: mk.block_norm(y, None, x, fake((8,)), h=x, act="relu"), "no gate activation"),
        (lambda: mk.block_norm(fake((8, 16)), None, fake((8, 16), "BFloat16"), fake((8,))), "`r` has element type"),
        (lambda: mk.block_norm_grad(y, None, None, x, None, drout=x, h=x), "`dh` is needed"),
    ]
    for call, msg in bad:
        with pytest.raises(mk.MLIRKernelsError, match=msg):
            call()


def test_rows_view_bounds():
    a = fake((8, 16))
    v = mk.rows(a, 3, 6)
    assert (v.dims, v.ld, v.pointer() - a.pointer()) == ((4, 16), 8, 8)
    assert mk.rows(a, 9, 8).length == 0
    for lo, hi in ((0, 3), (2, 9), (5, 3)):
        with pytest.raises(IndexError):
            mk.rows(a, lo, hi)
    with pytest.raises(TypeError):
        mk.rows(fake((8,)), 1, 2)


def test_plain_gradients_against_differences():
    """The 64-bit forms that the GPU tests compare with: their gradients against their own differences."""
    r = np.random.Generator(np.random.Philox(1))
    spans, T, D, N, G, W = [(1, 6), (6, 6), (6, 9)], 10, 6, 3, 2, 3
    f = r.standard_normal
    v = {"u": f((T, D)), "delta": f((T, D)), "A": -np.exp(f((D, N))), "B": f((T, G, N)), "C": f((T, G, N)), "D": f(D),
         "z": f((T, D)), "bias": f(D), "init": f((3, D, N))}
    dy, dl = f((T, D)), f((3, D, N))

    def run(grad=False):
        a = (v["u"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], True, spans, v["init"])
        return ref.scan(*a, dy=dy, dlast=dl)[2] if grad else sum(
            (x * g).sum() for x, g in zip(ref.scan(*a), (dy, dl)))

    def check(v, run):
        grads = run(True)
        for k in v:
            d, kept = f(v[k].shape), v[k]
            v[k] = kept + 1e-5 * d
            up = run()
            v[k] = kept - 1e-5 * d
            down = run()
            v[k] = kept
            assert (up - down) / 2e-5 == pytest.approx((grads[k] * d).sum(), rel=1e-6, abs=1e-7), k

    check(v, run)
    c = {"x": f((T, D)), "w": f((W, D)), "bias": f(D), "init": f((3, W - 1, D))}
    cl = f((3, W - 1, D))

    def run_conv(grad=False):
        a = (c["x"], c["w"], c["bias"], True, spans, c["init"])
        if grad:
            return dict(zip(("x", "w", "bias", "init"), ref.conv(*a, dy=dy, dlast=cl)[2:]))
        return sum((x * g).sum() for x, g in zip(ref.conv(*a), (dy, cl)))

    check(c, run_conv)
    n = {"r": f((T, D)), "w": f(D), "h": f((T, D)), "hw": f(D), "gate": f((T, D)), "scale": f(D)}
    dro = f((T, D))
    for act in ("silu", "sigmoid"):
        def run_norm(grad=False):
            a = (n["r"], n["w"], n["h"], n["hw"], n["gate"], act, n["scale"], 1e-5)
            return ref.norm(*a, dy=dy, drout=dro)[2] if grad else sum(
                (x * g).sum() for x, g in zip(ref.norm(*a), (dy, dro)))
        check(n, run_norm)


def refused(monkeypatch, cases):
    """Every call raises with its message, and none comes as far as a launch."""
    launched = []
    monkeypatch.setattr(mk.statespace, "launch", lambda *a: launched.append(a[3]))
    for call, msg in cases:
        with pytest.raises(mk.MLIRKernelsError, match=msg):
            call()
    assert not launched


def test_norm_arrays_of_other_sizes_are_refused(monkeypatch):
    """Arrays that agree with one another, but not with r."""
    y, h, g, w = fake((8, 16)), fake((8, 16)), fake((8, 16)), fake((8,))
    longer, wider = fake((8, 32)), fake((16, 16))
    refused(monkeypatch, [
        (lambda: mk.block_norm(y, None, longer, w, h=h), "expected 8 x 16"),
        (lambda: mk.block_norm(y, None, longer, w), "expected 8 x 16"),
        (lambda: mk.block_norm(None, fake((8, 32)), longer, None, h=h), "expected 8 x 16"),
        (lambda: mk.block_norm(None, y, longer, None), "expected 8 x 32"),
        (lambda: mk.block_norm(None, y, longer, None, h=h), "expected 8 x 16"),
        (lambda: mk.block_norm(None, longer, y, None, h=h), "expected 8 x 16"),
        (lambda: mk.block_norm(None, fake((16, 16)), wider, None, h=h), "expected 8 x 16"),
        (lambda: mk.block_norm(y, None, wider, fake((16,)), h=h), "expected 8 x 16"),
        (lambda: mk.block_norm(y, None, longer, w, h=longer, gate=g), "expected 8 x 32"),
        (lambda: mk.block_norm(y, None, mk.rows(fake((9, 32)), 1, 8), w, h=h), "expected 8 x 16"),
        (lambda: mk.block_norm(mk.rows(fake((9, 16)), 1, 8), None, longer, w), "expected 8 x 16"),
        (lambda: mk.block_norm(fake((8,)), None, y, w), "expected 8 x 1"),
        (lambda: mk.block_norm_grad(longer, w, y, longer, w), "expected 8 x 16"),
        (lambda: mk.block_norm_grad(longer, w, y, longer, w, h=h, dh=g), "expected 8 x 16"),
        (lambda: mk.block_norm_grad(longer, w, longer, longer, w, h=h, dh=g), "expected 8 x 16"),
        (lambda: mk.block_norm_grad(y, w, y, y, w, h=h, dh=longer), "expected 8 x 16"),
        (lambda: mk.block_norm_grad(longer, w, y, y, w, h=h, dh=g), "expected 8 x 16"),
        (lambda: mk.block_norm_grad(longer, None, None, longer, None, drout=y), "expected 8 x 32"),
        (lambda: mk.block_norm_grad(longer, None, None, longer, None, drout=longer, h=h, dh=g), "expected 8 x 16"),
        (lambda: mk.block_norm_grad(fake((16, 16)), None, None, wider, None, drout=fake((16, 16)), h=h, dh=g),
         "expected 8 x 16"),
    ])


def test_scan_matrices_of_other_rows_are_refused(monkeypatch):
    """B, C and their gradients with as many rows as u has channels, where the call needs another number."""
    u, x, A, B = fake((8, 16)), fake((8, 16)), fake((4, 8)), fake((4, 16))
    saved = fake((4, 8, 1))
    refused(monkeypatch, [
        (lambda: mk.selective_scan(x, u, u, A, B, u), "`C` has dims"),
        (lambda: mk.selective_scan(x, u, u, A, u, B), "`C` has dims"),
        (lambda: mk.selective_scan(x, u, u, fake((3, 8)), u, u), "`B` has dims"),
        (lambda: mk.selective_scan(x, u, u, fake((16, 8)), fake((16, 16)), u), "`C` has dims"),
        (lambda: mk.selective_scan(x, u, u, A, fake((6, 16)), fake((6, 16))), "`B` has dims"),
        (lambda: mk.selective_scan(x, u, u, A, fake((4, 17)), fake((4, 17))), "`B` has dims"),
        (lambda: mk.selective_scan_step(x, fake((4, 8, 16)), fake((4, 8, 16)), u, u, A, B, u), "`C` has dims"),
        (lambda: mk.selective_scan_step(x, fake((3, 8, 16)), fake((3, 8, 16)), u, u, fake((3, 8)), u, u),
         "`B` has dims"),
        (lambda: mk.selective_scan_grad(x, x, A, x, B, u, u, u, A, B, B, saved), "`dB` has dims"),
        (lambda: mk.selective_scan_grad(x, x, A, B, x, u, u, u, A, B, B, saved), "`dC` has dims"),
        (lambda: mk.selective_scan_grad(x, x, A, fake((8, 16)), fake((8, 16)), u, u, u, A, B, B, saved), "`dB` has"),
    ])


def test_scan_matrices_of_as_many_rows_as_channels(monkeypatch):
    """The same number of rows where it is the right one: N states, or groups of them."""
    seen = []
    monkeypatch.setattr(mk.statespace, "launch", lambda entry, args, arrays, what: seen.append(args))
    u, x = fake((8, 16)), fake((8, 16))
    for A, G in ((fake((8, 8)), 1), (fake((4, 8)), 2), (fake((2, 8)), 4)):
        mk.selective_scan(x, u, u, A, fake((8, 16)), u)
        mk.selective_scan(x, u, u, A, mk.rows(fake((9, 16)), 2, 9), fake((8 // G, G, 16)))
        assert [(a.N, a.G, a.ldb, a.ldc) for a in seen[-2:]] == [(8 // G, G, 8, 8), (8 // G, G, 9, 8)]


def test_one_token_without_a_second_dimension(monkeypatch):
    """u of one dimension is one token; the others are compared with it, not with the first matrix that follows."""
    u, A, B, st = fake((8,)), fake((4, 8)), fake((4, 1)), fake((4, 8, 1))
    refused(monkeypatch, [
        (lambda: mk.selective_scan_step(fake((4, 1)), st, st, u, u, A, B, B), "`y` has dims"),
        (lambda: mk.selective_scan_step(u, st, st, u, fake((4, 1)), A, B, B), "`delta` has dims"),
        (lambda: mk.selective_scan(fake((4, 1)), u, u, A, B, B), "`y` has dims"),
        (lambda: mk.selective_scan_grad(fake((4, 1)), u, A, B, B, u, u, u, A, B, B, st), "`du` has dims"),
        (lambda: mk.causal_conv(fake((4, 1)), u, fake((8, 4))), "`y` has dims"),
    ])
    seen = []
    monkeypatch.setattr(mk.statespace, "launch", lambda entry, args, arrays, what: seen.append(args))
    mk.selective_scan_step(u, st, st, u, fake((8, 1)), A, B, fake((4, 1, 1)), z=u)
    mk.causal_conv_step(u, fake((8, 3, 1)), fake((8, 3, 1)), u, fake((8, 4)))
    mk.block_norm(u, None, fake((8, 1)), fake((8,)), h=u)
    assert [(a.D, a.T if hasattr(a, "T") else a.B) for a in seen] == [(8, 1)] * 3


def test_slots_without_a_pool_are_refused(monkeypatch):
    x, A, B, one = fake((8, 16)), fake((4, 8)), fake((4, 16)), fake((1,), "Int32")
    refused(monkeypatch, [
        (lambda: mk.causal_conv(fake((8, 16)), x, fake((8, 4)), slots=one), "`slots` without"),
        (lambda: mk.selective_scan(fake((8, 16)), x, x, A, B, B, slots=one), "`slots` without"),
    ])


def test_no_tokens_with_groups_as_rows(monkeypatch):
    """No tokens: B and C as rows of a wider matrix have the rows of all groups, as they have with tokens."""
    seen = []
    monkeypatch.setattr(mk.statespace, "launch", lambda entry, args, arrays, what: seen.append(args))
    u, A = fake((8, 0)), fake((4, 8))
    for B in (fake((8, 0)), mk.rows(fake((9, 0)), 2, 9), fake((4, 2, 0)), fake((4, 0))):
        mk.selective_scan(fake((8, 0)), u, u, A, B, B, seqs=fake((1,), "Int32"))
        mk.selective_scan_step(fake((8, 0)), fake((4, 8, 0)), fake((4, 8, 0)), u, u, A, B, B)
    assert [(a.G, a.N) for a in seen] == [(2, 4)] * 6 + [(1, 4)] * 2
    refused(monkeypatch, [
        (lambda: mk.selective_scan(fake((8, 0)), u, u, A, fake((6, 0)), fake((6, 0))), "`B` has dims"),
        (lambda: mk.selective_scan(fake((8, 0)), u, u, A, fake((8, 0)), fake((4, 0))), "`C` has dims"),
        (lambda: mk.selective_scan(fake((8, 0)), u, u, A, None, fake((4, 0))), "`B` "),
    ])


def every_call():
    """The calls with all of their arrays, by name: (call, arrays)."""
    f, i = (lambda *s: fake(s)), (lambda *s: fake(s, "Int32"))
    D, T, S, N, G, W, P, t = 8, 16, 2, 4, 2, 3, 5, (8, 16)
    conv = dict(x=f(*t), w=f(D, W), bias=f(D), seqs=i(S + 1))
    scan = dict(u=f(*t), delta=f(*t), A=f(N, D), B=f(N, G, T), C=f(N, G, T), D=f(D), z=f(*t), bias=f(D), seqs=i(S + 1))
    step = {k: v for k, v in scan.items() if k != "seqs"}
    norm = dict(r=f(*t), w=f(D), h=f(*t), hw=f(D), gate=f(*t), scale=f(D))
    saved = f(N, D, T // 32 + S)
    return {
        "causal_conv": (mk.causal_conv, dict(y=f(*t), **conv, init=f(D, W - 1, S), last=f(D, W - 1, S))),
        "causal_conv_slots": (mk.causal_conv, dict(y=f(*t), **conv, init=f(D, W - 1, P), last=f(D, W - 1, P), slots=i(S))),
        "causal_conv_grad": (mk.causal_conv_grad, dict(
            dx=f(*t), dw=f(D, W), dy=f(*t), dbias=f(D), **conv, init=f(D, W - 1, S), dinit=f(D, W - 1, S),
            dlast=f(D, W - 1, S))),
        "causal_conv_step": (mk.causal_conv_step, dict(
            y=f(*t), next=f(D, W - 1, T), state=f(D, W - 1, T), x=f(*t), w=f(D, W), bias=f(D))),
        "selective_scan": (mk.selective_scan, dict(y=f(*t), **scan, init=f(N, D, S), last=f(N, D, S), saved=saved)),
        "selective_scan_slots": (mk.selective_scan, dict(y=f(*t), **scan, init=f(N, D, P), last=f(N, D, P), slots=i(S))),
        "selective_scan_grad": (mk.selective_scan_grad, dict(
            du=f(*t), ddelta=f(*t), dA=f(N, D), dB=f(N, G, T), dC=f(N, G, T), dy=f(*t), **scan, saved=saved, dD=f(D),
            dz=f(*t), dbias=f(D), dinit=f(N, D, S), dlast=f(N, D, S))),
        "selective_scan_step": (mk.selective_scan_step, dict(y=f(*t), next=f(N, D, T), state=f(N, D, T), **step)),
        "block_norm": (mk.block_norm, dict(y=f(*t), rout=f(*t), **norm)),
        "block_norm_grad": (mk.block_norm_grad, dict(
            dr=f(*t), dw=f(D), dy=f(*t), drout=f(*t), **norm, dh=f(*t), dhw=f(D), dgate=f(*t), dscale=f(D))),
    }


@pytest.mark.parametrize("name", list(every_call()))
def test_every_array_of_another_size_is_refused(monkeypatch, name):
    """One array at a time, larger or smaller in one dimension, or with dims that another array of the call has."""
    call, arrays = every_call()[name]
    launched = []
    monkeypatch.setattr(mk.statespace, "launch", lambda *a: launched.append(a[3]))
    call(**arrays)
    assert len(launched) == 1
    others = {a.dims for a in arrays.values() if a.eltype == "Float32"}
    for k, a in arrays.items():
        wrong = {a.dims[:j] + (a.dims[j] + d,) + a.dims[j + 1:] for j in range(len(a.dims)) for d in (-1, 1, a.dims[j])}
        wrong |= {d for d in others if np.prod(d) != np.prod(a.dims)} if a.eltype == "Float32" else set()
        if (name, k) == ("causal_conv_slots", "w"):
            continue  # a pool is taken by its elements: it holds another number of states of other taps
        for dims in wrong:
            with pytest.raises(mk.MLIRKernelsError):
                call(**dict(arrays, **{k: fake(dims, a.eltype)}))
    assert len(launched) == 1
