"""State space operators: causal convolution, selective scan, block norms.

They work on (channels, tokens) arrays, a token's channels contiguous, beside
``accumulate`` (a scan with a fixed operator) and ``mapreducedim`` (a reduction
of one dimension), and like ``mul``'s Julia counterpart ``mul!`` they write into
the arrays given first.  Token arrays are Float32, Float16 or BFloat16, all of
one call alike, as an ``MLIRArray`` or as neighbouring rows of one (``rows``);
parameters, their gradients and scan states are Float32; sums are kept in
Float32.  Each call is asynchronous on torch's current stream of the arrays'
device.

Sequences.  Without ``seqs`` an array (D, L, S) holds S sequences of L tokens
and (D, T) one.  With ``seqs`` (Int32, S + 1 entries, 1-based, ascending)
sequence s has the columns ``seqs[s] : seqs[s+1]-1``; columns outside all
sequences are left as they were.  Sequences may be empty.

Slots.  With ``slots`` (Int32, 1-based, one per sequence or batch entry) states
are taken from and put into that column of a pool; entries <= 0 have no state
(a prompt starts from zero and leaves none, a step leaves its output alone).

Offsets and slots are read on the device.  Bad ones (offsets that descend or
leave the array, slots above the pool or used twice) raise ``KernelException``
at the next ``synchronize``.

A gradient overwrites the arrays given for it.  Workspaces come from torch's
allocator, so a call may be captured into a CUDA graph; two graphs do not share
one.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .array import MLIRArray, MLIRCUDABackend, MLIRRows, allocate, current_stream_handle, on_device

_FLOATS = ("Float32", "Float16", "BFloat16")


def _fail(what: str, msg: str):
    raise _lib.MLIRKernelsError(f"MLIRCUDABackend: {what}: {msg}")


class _Call:
    """Checks the arrays of one call and collects what the C entry point takes."""

    def __init__(self, what: str):
        self.what, self.arrays, self.eltype = what, [], None

    def tokens(self, a, name: str, rows: int | None = None, cols: int | None = None, eltype: str | None = None):
        """A token array as (pointer, ld); its element type is the call's unless given."""
        if not isinstance(a, (MLIRArray, MLIRRows)):
            _fail(self.what, f"`{name}` must be an MLIRArray or rows of one, got {type(a).__name__}")
        if a.eltype not in _FLOATS:
            _fail(self.what, f"`{name}` has element type {a.eltype}, expected {' or '.join(_FLOATS)}")
        if eltype is None:
            if self.eltype is None:
                self.eltype = a.eltype
            eltype = self.eltype
        if a.eltype != eltype:
            _fail(self.what, f"`{name}` has element type {a.eltype}, expected {eltype}")
        r, n = a.dims[0] if a.dims else 1, math.prod(a.dims[1:])
        if rows is not None:
            # (N, G, T) arrays: the leading dimensions of a token together
            if r != rows and isinstance(a, MLIRArray) and len(a.dims) > 1 and r * a.dims[1] == rows:
                r, n = rows, math.prod(a.dims[2:])
            if r != rows or n != cols:
                _fail(self.what, f"`{name}` has dims {a.dims}, expected {rows} x {cols} tokens")
        self.arrays.append(a)
        return a.pointer(), a.ld if isinstance(a, MLIRRows) else r

    def dense(self, a, name: str, length: int, eltypes=("Float32",)):
        """A dense array of `length` elements (None: any), as a pointer."""
        if a is None:
            return None
        if not isinstance(a, MLIRArray):
            _fail(self.what, f"`{name}` must be an MLIRArray, got {type(a).__name__}")
        if a.eltype not in eltypes:
            _fail(self.what, f"`{name}` has element type {a.eltype}, expected {' or '.join(eltypes)}")
        if length is not None and a.length != length:
            _fail(self.what, f"`{name}` has {a.length} elements, expected {length}")
        self.arrays.append(a)
        return a.pointer()

    def sequences(self, x, seqs):
        """(T, nseq, len, pointer of seqs) of the token array x."""
        dims = x.dims if len(x.dims) > 1 else tuple(x.dims) + (1,)
        T = math.prod(dims[1:])
        if seqs is None:
            return T, math.prod(dims[2:]), dims[1], None
        p = self.dense(seqs, "seqs", None, ("Int32",))
        if seqs.length < 1:
            _fail(self.what, "`seqs` has no entries, expected one more than sequences")
        return T, seqs.length - 1, 0, p

    def pool(self, name: str, a, slots, one: int, count: int, eltypes=("Float32",)):
        """A state array of `count` states of `one` elements, or a pool of any number with slots."""
        if a is None:
            return None, 0
        if slots is None:
            return self.dense(a, name, one * count, eltypes), count
        p = self.dense(a, name, None, eltypes)
        if a.length % one:
            _fail(self.what, f"`{name}` has {a.length} elements, not a number of states of {one}")
        return p, a.length // one

    def slots(self, slots, count: int, *pools):
        """(pointer, number of slots) for the pools given as (name, size or None)."""
        if slots is None:
            return None, 0
        p = self.dense(slots, "slots", count, ("Int32",))
        sizes = {n for n in pools if n is not None}
        if len(sizes) > 1:
            _fail(self.what, f"the state pools hold different numbers of states: {sorted(sizes)}")
        return p, sizes.pop() if sizes else 0

    def run(self, entry: str, args, workspace: str | None = None):
        L = _lib.lib()
        with on_device(*self.arrays):
            if workspace is not None:
                n = C.c_size_t()
                _lib.check(getattr(L, workspace)(args, n), self.what)
                if n.value:
                    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
                    args.workspace, args.workspace_bytes = ws.data_ptr(), n.value
            _lib.check(getattr(L, entry)(args, current_stream_handle()), self.what)


# ---- causal convolution ----------------------------------------------------------

def _conv(call: _Call, x, w, bias, silu, seqs):
    px, ldx = call.tokens(x, "x")
    T, nseq, ln, pseqs = call.sequences(x, seqs)
    D = x.dims[0]
    pw = call.dense(w, "w", None)
    if w is None or len(w.dims) != 2 or w.dims[0] != D:
        _fail(call.what, f"`w` must be ({D}, taps)")
    return _lib.ConvArgs(type=_lib.MK_T[call.eltype], width=w.dims[1], silu=int(bool(silu)), D=D, T=T, nseq=nseq,
                         len=ln, seqs=pseqs, x=px, ldx=ldx, w=pw, bias=call.dense(bias, "bias", D))


def causal_conv(y, x, w, *, bias=None, silu=True, seqs=None, init=None, last=None, slots=None):
    """``y[d,t] = act(bias[d] + sum_k w[d,k] x[d,t-W+k])``, k = 1..W: each channel's
    tokens filtered with W = 2 to 4 taps, ``w`` (D, W).  Tokens before a sequence
    are its state in ``init`` (D, W-1, S), the oldest first, or zero; ``last``
    receives the state behind it and may be ``init``.  ``y`` must not be ``x``."""
    c = _Call("causal_conv")
    a = _conv(c, x, w, bias, silu, seqs)
    a.y, a.ldy = c.tokens(y, "y", a.D, a.T)
    one = a.D * (a.width - 1)
    a.init, ni = c.pool("init", init, slots, one, a.nseq, (c.eltype,))
    a.last, nl = c.pool("last", last, slots, one, a.nseq, (c.eltype,))
    a.slots, a.nslots = c.slots(slots, a.nseq, ni if init is not None else None, nl if last is not None else None)
    c.run("mk_causal_conv", a)
    return y


def causal_conv_grad(dx, dw, dy, x, w, *, bias=None, dbias=None, silu=True, seqs=None, init=None, dinit=None,
                     dlast=None):
    """Gradients of ``causal_conv`` for ``dy`` (and ``dlast``, that of ``last``):
    ``dx``, ``dw`` and, where given, ``dbias`` and ``dinit``.  The forward pass's
    intermediate values are computed again; nothing of it has to be kept."""
    c = _Call("causal_conv_grad")
    a = _conv(c, x, w, bias, silu, seqs)
    a.dy, a.lddy = c.tokens(dy, "dy", a.D, a.T)
    a.dx, a.lddx = c.tokens(dx, "dx", a.D, a.T)
    one = a.D * (a.width - 1)
    a.init = c.dense(init, "init", one * a.nseq, (c.eltype,))
    a.dinit = c.dense(dinit, "dinit", one * a.nseq, (c.eltype,))
    a.dlast = c.dense(dlast, "dlast", one * a.nseq, (c.eltype,))
    a.dw = c.dense(dw, "dw", a.D * a.width)
    a.dbias = c.dense(dbias, "dbias", a.D)
    c.run("mk_causal_conv_grad", a, "mk_causal_conv_grad_workspace")
    return dx


def causal_conv_step(y, next, state, x, w, *, bias=None, silu=True, slots=None):
    """One token per batch entry: ``y`` and ``x`` are (D, B), ``state`` (D, W-1, B)
    or a pool with ``slots``; ``next`` receives the state moved on by ``x`` and may
    be ``state``.  Pool columns that no entry uses are left as they were."""
    c = _Call("causal_conv_step")
    px, ldx = c.tokens(x, "x")
    D, B = x.dims[0], math.prod(x.dims[1:])
    pw = c.dense(w, "w", None)
    if w is None or len(w.dims) != 2 or w.dims[0] != D:
        _fail(c.what, f"`w` must be ({D}, taps)")
    W = w.dims[1]
    py, ldy = c.tokens(y, "y", D, B)
    ps, ns = c.pool("state", state, slots, max(1, D * (W - 1)), B, (c.eltype,))
    pn, nn = c.pool("next", next, slots, max(1, D * (W - 1)), B, (c.eltype,))
    pslots, nslots = c.slots(slots, B, ns, nn)
    c.run("mk_causal_conv_step", _lib.ConvStepArgs(
        type=_lib.MK_T[c.eltype], width=W, silu=int(bool(silu)), D=D, B=B, slots=pslots, nslots=nslots, x=px, ldx=ldx,
        y=py, ldy=ldy, state=ps, next=pn, w=pw, bias=c.dense(bias, "bias", D)))
    return y


# ---- selective scan --------------------------------------------------------------

def _states(call: _Call, A, B, D: int, T: int):
    """(pointer of A, N, G): A is (N, D), B has G * N rows."""
    p = call.dense(A, "A", None)
    if A is None or len(A.dims) != 2 or A.dims[1] != D:
        _fail(call.what, f"`A` must be (states, {D})")
    N = A.dims[0]
    rows = B.length // T if isinstance(B, (MLIRArray, MLIRRows)) and T else N
    G = rows // N if N else 0
    if G < 1 or D % G:
        _fail(call.what, f"`B` has dims {getattr(B, 'dims', None)}: not (groups of) {N} rows for {T} tokens")
    return p, N, G


def _scan(call: _Call, u, delta, A, B, Cm, D, z, bias, softplus, seqs):
    pu, ldu = call.tokens(u, "u")
    T, nseq, ln, pseqs = call.sequences(u, seqs)
    n = u.dims[0]
    pd, ldd = call.tokens(delta, "delta", n, T)
    pA, N, G = _states(call, A, B, n, T)
    pB, ldb = call.tokens(B, "B", G * N, T)
    pC, ldc = call.tokens(Cm, "C", G * N, T)
    pz, ldz = call.tokens(z, "z", n, T) if z is not None else (None, 0)
    return _lib.ScanArgs(type=_lib.MK_T[call.eltype], softplus=int(bool(softplus)), D=n, N=N, G=G, T=T, nseq=nseq,
                         len=ln, seqs=pseqs, u=pu, delta=pd, z=pz, B=pB, C=pC, ldu=ldu, lddelta=ldd, ldz=ldz, ldb=ldb,
                         ldc=ldc, A=pA, Dskip=call.dense(D, "D", n), bias=call.dense(bias, "bias", n))


def _saved_length(u, A, T: int, nseq: int) -> int:
    return A.dims[0] * u.dims[0] * (T // _lib.MK_SCAN_PIECE + nseq)


def selective_scan_saved(u, A, *, seqs=None) -> MLIRArray:
    """An array for the states that ``selective_scan`` leaves for its gradient: one
    per 32 tokens of a sequence, N floats per channel."""
    c = _Call("selective_scan_saved")
    T, nseq, _, _ = c.sequences(u, seqs)
    with on_device(u, A):
        return allocate(MLIRCUDABackend(), "Float32", (A.dims[0], u.dims[0], T // _lib.MK_SCAN_PIECE + nseq))


def selective_scan(y, u, delta, A, B, C, *, D=None, z=None, bias=None, softplus=True, seqs=None, init=None, last=None,
                   slots=None, saved=None):
    """Per channel d and state n, along the tokens t of a sequence::

        dt = softplus(delta + bias)            (delta + bias without softplus)
        h[n] = exp(dt * A[n,d]) * h[n] + dt * u * B[n,g,t]
        y = (sum_n C[n,g,t] * h[n] + D[d] * u) * silu(z)

    ``u``, ``delta``, ``z``, ``y`` are (D, T) or (D, L, S); ``A`` is (N, D), N <= 64;
    ``B`` and ``C`` are (N, T), or (N, G, T) with groups of D/G neighbouring channels
    (also as rows of a wider matrix, N * G of them).  ``h`` starts at ``init``
    (N, D, S) or zero; ``last`` receives it behind the sequence and may be ``init``.
    ``saved`` (``selective_scan_saved``) keeps what the gradient needs.  ``y`` may be
    ``u``, ``delta`` or ``z``."""
    c = _Call("selective_scan")
    a = _scan(c, u, delta, A, B, C, D, z, bias, softplus, seqs)
    a.y, a.ldy = c.tokens(y, "y", a.D, a.T)
    a.init, ni = c.pool("init", init, slots, a.N * a.D, a.nseq)
    a.last, nl = c.pool("last", last, slots, a.N * a.D, a.nseq)
    a.slots, a.nslots = c.slots(slots, a.nseq, ni if init is not None else None, nl if last is not None else None)
    if saved is not None:
        a.saved = c.dense(saved, "saved", _saved_length(u, A, a.T, a.nseq))
    c.run("mk_selective_scan", a, "mk_selective_scan_workspace")
    return y


def selective_scan_grad(du, ddelta, dA, dB, dC, dy, u, delta, A, B, C, saved, *, D=None, dD=None, z=None, dz=None,
                        bias=None, dbias=None, softplus=True, seqs=None, dinit=None, dlast=None):
    """Gradients of ``selective_scan`` for ``dy`` (and ``dlast``, that of ``last``).
    ``dB`` and ``dC`` are summed over the channels of a group, ``dA``, ``dD`` and
    ``dbias`` over all tokens.  ``saved`` is what the forward pass left, for the same
    inputs (an ``init`` is in it); ``dD``, ``dz``, ``dbias`` go with ``D``, ``z``, ``bias``."""
    c = _Call("selective_scan_grad")
    a = _scan(c, u, delta, A, B, C, D, z, bias, softplus, seqs)
    GN = a.G * a.N
    a.dy, a.lddy = c.tokens(dy, "dy", a.D, a.T)
    a.du, a.lddu = c.tokens(du, "du", a.D, a.T)
    a.ddelta, a.ldddelta = c.tokens(ddelta, "ddelta", a.D, a.T)
    a.dB, a.lddb = c.tokens(dB, "dB", GN, a.T)
    a.dC, a.lddc = c.tokens(dC, "dC", GN, a.T)
    for name, given, grad in (("D", D, dD), ("z", z, dz), ("bias", bias, dbias)):
        if (given is None) != (grad is None):
            _fail(c.what, f"`d{name}` is needed exactly when `{name}` is given")
    if z is not None:
        a.dz, a.lddz = c.tokens(dz, "dz", a.D, a.T)
    a.dA = c.dense(dA, "dA", a.N * a.D)
    a.dDskip = c.dense(dD, "dD", a.D)
    a.dbias = c.dense(dbias, "dbias", a.D)
    a.saved = c.dense(saved, "saved", _saved_length(u, A, a.T, a.nseq))
    a.dinit = c.dense(dinit, "dinit", a.N * a.D * a.nseq)
    a.dlast = c.dense(dlast, "dlast", a.N * a.D * a.nseq)
    c.run("mk_selective_scan_grad", a, "mk_selective_scan_grad_workspace")
    return du


def selective_scan_step(y, next, state, u, delta, A, B, C, *, D=None, z=None, bias=None, softplus=True, slots=None):
    """One token per batch entry: ``u``, ``delta``, ``z``, ``y`` are (D, B), ``B`` and ``C``
    (N, B) or (N, G, B), ``state`` (N, D, B) or a pool with ``slots``; ``next`` receives
    the state moved on and may be ``state``.  Pool columns that no entry uses are left
    as they were."""
    c = _Call("selective_scan_step")
    pu, ldu = c.tokens(u, "u")
    n, batch = u.dims[0], math.prod(u.dims[1:])
    pd, ldd = c.tokens(delta, "delta", n, batch)
    pA, N, G = _states(c, A, B, n, batch)
    pB, ldb = c.tokens(B, "B", G * N, batch)
    pC, ldc = c.tokens(C, "C", G * N, batch)
    pz, ldz = c.tokens(z, "z", n, batch) if z is not None else (None, 0)
    py, ldy = c.tokens(y, "y", n, batch)
    ps, ns = c.pool("state", state, slots, N * n, batch)
    pn, nn = c.pool("next", next, slots, N * n, batch)
    pslots, nslots = c.slots(slots, batch, ns, nn)
    c.run("mk_selective_scan_step", _lib.ScanStepArgs(
        type=_lib.MK_T[c.eltype], softplus=int(bool(softplus)), D=n, N=N, G=G, B=batch, slots=pslots, nslots=nslots,
        u=pu, delta=pd, z=pz, Bmat=pB, Cmat=pC, ldu=ldu, lddelta=ldd, ldz=ldz, ldb=ldb, ldc=ldc, A=pA,
        Dskip=c.dense(D, "D", n), bias=c.dense(bias, "bias", n), state=ps, next=pn, y=py, ldy=ldy))
    return y


# ---- norms around a block ----------------------------------------------------------

def _norm(call: _Call, r, w, h, hw, gate, scale, act, eps, lead):
    if act not in _lib.MK_ACT:
        _fail(call.what, f"no gate activation {act!r} (supported: silu, sigmoid)")
    call.tokens(lead, "h" if lead is h else "y")  # sets the call's element type
    if not isinstance(r, (MLIRArray, MLIRRows)):
        _fail(call.what, f"`r` must be an MLIRArray or rows of one, got {type(r).__name__}")
    rt = r.eltype
    if rt not in ("Float32", call.eltype):
        _fail(call.what, f"`r` has element type {rt}, expected Float32 or {call.eltype}")
    pr, ldr = call.tokens(r, "r", eltype=rt)
    D, T = r.dims[0], math.prod(r.dims[1:])
    if h is None and not (gate is None and hw is None and scale is None):
        _fail(call.what, "`gate`, `hw` and `scale` belong to `h`")
    a = _lib.NormArgs(type=_lib.MK_T[call.eltype], rtype=_lib.MK_T[rt], act=_lib.MK_ACT[act], eps=eps, D=D, T=T, r=pr,
                      ldr=ldr, hw=call.dense(hw, "hw", D), scale=call.dense(scale, "scale", D),
                      w=call.dense(w, "w", D))
    if h is not None:
        a.h, a.ldh = call.tokens(h, "h", D, T)
    if gate is not None:
        a.gate, a.ldgate = call.tokens(gate, "gate", D, T)
    return a


def block_norm(y, rout, r, w, *, h=None, hw=None, gate=None, act="silu", scale=None, eps=1e-5):
    """The norms behind and before a block with its gate and residual, per token::

        n = h / sqrt(mean(h^2) + eps) * hw        (h without hw)
        m = n * act(gate)                         (n without gate; "silu" or "sigmoid")
        rout = r + scale * m                      (r without h, r + m without scale)
        y = rout / sqrt(mean(rout^2) + eps) * w

    ``r`` is the residual stream, Float32 or of ``h``'s type, ``rout`` the new one (it
    may be ``r``, or None), ``y`` what the next block takes (``y`` and ``w`` None: no
    norm).  ``y`` is computed from ``rout`` before it is rounded.  At most 16384
    channels."""
    c = _Call("block_norm")
    if y is None and rout is None:
        _fail(c.what, "neither `y` nor `rout` is given")
    if (y is None) != (w is None):
        _fail(c.what, "`y` and `w` are given together")
    a = _norm(c, r, w, h, hw, gate, scale, act, eps, h if h is not None else y if y is not None else r)
    if y is not None:
        a.y, a.ldy = c.tokens(y, "y", a.D, a.T)
    if rout is not None:
        a.rout, a.ldrout = c.tokens(rout, "rout", a.D, a.T, eltype=r.eltype)
    c.run("mk_block_norm", a)
    return y if y is not None else rout


def block_norm_grad(dr, dw, dy, r, w, *, drout=None, h=None, dh=None, hw=None, dhw=None, gate=None, dgate=None,
                    act="silu", scale=None, dscale=None, eps=1e-5):
    """Gradients of ``block_norm`` for ``dy`` and ``drout`` (either may be None, ``dy``
    with ``w`` and ``dw``): ``dr`` (may be ``drout``) and those of ``h``, ``gate``,
    ``hw``, ``scale`` and ``w``, each needed exactly when the input is given.  The
    forward values are computed again from ``r``, ``h`` and ``gate``."""
    c = _Call("block_norm_grad")
    if dy is None and drout is None:
        _fail(c.what, "neither `dy` nor `drout` is given")
    if (dy is None) != (w is None):
        _fail(c.what, "`dy` and `w` are given together")
    for name, given, grad in (("w", w, dw), ("h", h, dh), ("hw", hw, dhw), ("gate", gate, dgate),
                              ("scale", scale, dscale)):
        if (given is None) != (grad is None):
            _fail(c.what, f"`d{name}` is needed exactly when `{name}` is given")
    a = _norm(c, r, w, h, hw, gate, scale, act, eps, h if h is not None else dy if dy is not None else r)
    a.dr, a.lddr = c.tokens(dr, "dr", a.D, a.T, eltype=r.eltype)
    if dy is not None:
        a.dy, a.lddy = c.tokens(dy, "dy", a.D, a.T)
    if drout is not None:
        a.drout, a.lddrout = c.tokens(drout, "drout", a.D, a.T, eltype=r.eltype)
    if h is not None:
        a.dh, a.lddh = c.tokens(dh, "dh", a.D, a.T)
    if gate is not None:
        a.dgate, a.lddgate = c.tokens(dgate, "dgate", a.D, a.T)
    a.dw, a.dhw, a.dscale = c.dense(dw, "dw", a.D), c.dense(dhw, "dhw", a.D), c.dense(dscale, "dscale", a.D)
    c.run("mk_block_norm_grad", a, "mk_block_norm_grad_workspace")
    return dr
