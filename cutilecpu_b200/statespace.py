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
at the next ``synchronize``; results of such a call are not to be used.

A gradient overwrites the arrays given for it.  Arrays that a call writes must
not overlap its others unless it says so.  Workspaces come from torch's
allocator, so a call may be captured into a CUDA graph; two graphs do not share
one.

Speed.  The scan and the norms take 16 bytes at a time where the channels (of a
group), leading dimensions and first rows are multiples of that, and single
elements otherwise, which takes 1.1 to 1.3 (scan) and 1.8 times (norms) as long:
parts of a projection are best laid out at such multiples.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .array import MLIRArray, MLIRCUDABackend, MLIRRows, allocate, launch, on_device

_FLOATS = ("Float32", "Float16", "BFloat16")


def _fail(what: str, msg: str):
    raise _lib.MLIRKernelsError(f"MLIRCUDABackend: {what}: {msg}")


class _Call:
    """Checks the arrays of one call and collects what the C entry point takes."""

    __slots__ = ("what", "arrays", "eltype", "lead")

    def __init__(self, what: str):
        self.what, self.arrays, self.eltype, self.lead = what, [], None, None

    def tokens(self, a, name: str, rows: int | None = None, cols: int | None = None, eltype: str | None = None):
        """A token array as (pointer, ld); its element type is the call's unless given."""
        dims = self.lead
        if (type(a) is MLIRArray and a.dims == dims and (rows is None or rows == dims[0])
                and a.eltype == (eltype or self.eltype)):
            self.arrays.append(a)  # like the call's first array, whose tokens all others have
            return a.storage.data_ptr(), dims[0]
        if not isinstance(a, (MLIRArray, MLIRRows)):
            _fail(self.what, f"`{name}` must be an MLIRArray or rows of one, got {type(a).__name__}")
        if a.eltype not in _FLOATS:
            _fail(self.what, f"`{name}` has element type {a.eltype}, expected {' or '.join(_FLOATS)}")
        dims = a.dims
        if self.eltype is None:
            self.eltype = a.eltype
        if self.lead is None:
            self.lead = dims
        if a.eltype != (eltype or self.eltype):
            _fail(self.what, f"`{name}` has element type {a.eltype}, expected {eltype or self.eltype}")
        r = dims[0] if dims else 1
        if rows is not None:
            n = math.prod(dims[1:])
            # (N, G, T) arrays: the leading dimensions of a token together
            if r != rows and len(dims) > 1 and r * dims[1] == rows and isinstance(a, MLIRArray):
                r, n = rows, math.prod(dims[2:])
            if r != rows or n != cols:
                _fail(self.what, f"`{name}` has dims {dims}, expected {rows} x {cols} tokens")
        self.arrays.append(a)
        return a.storage.data_ptr(), a.ld if isinstance(a, MLIRRows) else r

    def like(self, names: str, rows: int, cols: int, *arrays):
        """The pointers of several token arrays of the call's lead, then their leading dimensions (None, 0: no array)."""
        lead, eltype, ptrs, lds = self.lead, self.eltype, [], []
        for i, a in enumerate(arrays):
            if a is None:
                ptrs.append(None)
                lds.append(0)
            elif type(a) is MLIRArray and a.dims == lead and a.eltype == eltype:
                self.arrays.append(a)
                ptrs.append(a.storage.data_ptr())
                lds.append(rows)
            else:
                p, ld = self.tokens(a, names.split()[i], rows, cols)
                ptrs.append(p)
                lds.append(ld)
        return ptrs + lds

    def floats(self, names: str, length: int, *arrays):
        """The pointers of several Float32 arrays of `length` elements (None: no array)."""
        out = []
        for i, a in enumerate(arrays):
            if a is None:
                out.append(None)
            elif type(a) is MLIRArray and a.eltype == "Float32" and a.storage.numel() == length:
                self.arrays.append(a)
                out.append(a.storage.data_ptr())
            else:
                out.append(self.dense(a, names.split()[i], length))
        return out

    def dense(self, a, name: str, length: int | None, eltype: str = "Float32"):
        """A dense array of `length` elements (None: any), as a pointer."""
        if a is None:
            return None
        if type(a) is not MLIRArray:
            _fail(self.what, f"`{name}` must be an MLIRArray, got {type(a).__name__}")
        if a.eltype != eltype:
            _fail(self.what, f"`{name}` has element type {a.eltype}, expected {eltype}")
        if length is not None and a.storage.numel() != length:
            _fail(self.what, f"`{name}` has {a.length} elements, expected {length}")
        self.arrays.append(a)
        return a.storage.data_ptr()

    def sequences(self, x, seqs):
        """(T, nseq, len, pointer of seqs) of the token array x."""
        dims = x.dims if len(x.dims) > 1 else tuple(x.dims) + (1,)
        T = math.prod(dims[1:])
        if seqs is None:
            return T, math.prod(dims[2:]), dims[1], None
        p = self.dense(seqs, "seqs", None, "Int32")
        if seqs.length < 1:
            _fail(self.what, "`seqs` has no entries, expected one more than sequences")
        return T, seqs.length - 1, 0, p

    def pool(self, name: str, a, slots, one: int, count: int, eltype: str = "Float32"):
        """A state array of `count` states of `one` elements, or a pool of any number with slots."""
        if a is None:
            return None, 0
        if slots is None:
            return self.dense(a, name, one * count, eltype), count
        p = self.dense(a, name, None, eltype)
        n, rest = divmod(a.storage.numel(), one)
        if rest:
            _fail(self.what, f"`{name}` has {a.length} elements, not a number of states of {one}")
        return p, n

    def slots(self, slots, count: int, first: int | None, second: int | None):
        """(pointer, number of slots) for the sizes of the two pools (None: no such pool)."""
        if slots is None:
            return None, 0
        if first is not None and second is not None and first != second:
            _fail(self.what, f"the state pools hold different numbers of states: {sorted((first, second))}")
        p = self.dense(slots, "slots", count, "Int32")
        if first is None and second is None:
            _fail(self.what, "`slots` without `init` or `last`, whose columns they choose")
        return p, second if first is None else first

    def run(self, entry: str, args, workspace: str | None = None):
        L = _lib.lib()
        if workspace is None:
            launch(getattr(L, entry), args, self.arrays, self.what)
            return
        query, call, n = getattr(L, workspace), getattr(L, entry), C.c_size_t()

        def both(args, stream):
            rc = query(args, n)
            if rc or not n.value:
                return rc or call(args, stream)
            ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
            args.workspace, args.workspace_bytes = ws.data_ptr(), n.value
            return call(args, stream)

        launch(both, args, self.arrays, self.what)


# ---- causal convolution ----------------------------------------------------------

def _conv(call: _Call, x, w, silu, seqs):
    """The first fields of ConvArgs up to seqs, and (D, T, nseq, W, x's pointer and ld, w's pointer)."""
    px, ldx = call.tokens(x, "x")
    T, nseq, ln, pseqs = call.sequences(x, seqs)
    D = x.dims[0]
    pw = call.dense(w, "w", None)
    if w is None or len(w.dims) != 2 or w.dims[0] != D:
        _fail(call.what, f"`w` must be ({D}, taps)")
    W = w.dims[1]
    return (_lib.MK_T[call.eltype], W, 1 if silu else 0, D, T, nseq, ln, pseqs), (D, T, nseq, W, px, ldx, pw)


def causal_conv(y, x, w, *, bias=None, silu=True, seqs=None, init=None, last=None, slots=None):
    """``y[d,t] = act(bias[d] + sum_k w[d,k] x[d,t-W+k])``, k = 1..W: each channel's
    tokens filtered with W = 2 to 4 taps, ``w`` (D, W).  Tokens before a sequence
    are its state in ``init`` (D, W-1, S), the oldest first, or zero; ``last``
    receives the state behind it and may be ``init``.  ``y`` must not be ``x``."""
    c = _Call("causal_conv")
    head, (D, T, nseq, W, px, ldx, pw) = _conv(c, x, w, silu, seqs)
    py, ldy = c.like("y", D, T, y)
    one = D * (W - 1)
    pi, ni = c.pool("init", init, slots, one, nseq, c.eltype)
    pl, nl = c.pool("last", last, slots, one, nseq, c.eltype)
    pslots, nslots = c.slots(slots, nseq, None if init is None else ni, None if last is None else nl)
    pb, = c.floats("bias", D, bias)
    c.run("mk_causal_conv", _lib.ConvArgs(*head, pslots, nslots, px, ldx, py, ldy, pw, pb, pi, pl))
    return y


def causal_conv_grad(dx, dw, dy, x, w, *, bias=None, dbias=None, silu=True, seqs=None, init=None, dinit=None,
                     dlast=None):
    """Gradients of ``causal_conv`` for ``dy`` (and ``dlast``, that of ``last``):
    ``dx``, ``dw`` and, where given, ``dbias`` and ``dinit``.  The forward pass's
    intermediate values are computed again; nothing of it has to be kept."""
    c = _Call("causal_conv_grad")
    head, (D, T, nseq, W, px, ldx, pw) = _conv(c, x, w, silu, seqs)
    pdy, pdx, lddy, lddx = c.like("dy dx", D, T, dy, dx)
    one = D * (W - 1) * nseq
    pi, pdl, pdi = (c.dense(a, n, one, c.eltype) for n, a in (("init", init), ("dlast", dlast), ("dinit", dinit)))
    pdw = c.dense(dw, "dw", D * W)
    pb, pdb = c.floats("bias dbias", D, bias, dbias)
    c.run("mk_causal_conv_grad", _lib.ConvArgs(*head, None, 0, px, ldx, None, 0, pw, pb, pi, None, pdy, lddy, pdl, pdx,
                                               lddx, pdw, pdb, pdi), "mk_causal_conv_grad_workspace")
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
    ps, ns = c.pool("state", state, slots, max(1, D * (W - 1)), B, c.eltype)
    pn, nn = c.pool("next", next, slots, max(1, D * (W - 1)), B, c.eltype)
    pslots, nslots = c.slots(slots, B, ns, nn)
    # fields in the struct's order
    c.run("mk_causal_conv_step", _lib.ConvStepArgs(
        _lib.MK_T[c.eltype], W, 1 if silu else 0, D, B, pslots, nslots, px, ldx, py, ldy, ps, pn, pw,
        c.dense(bias, "bias", D)))
    return y


# ---- selective scan --------------------------------------------------------------

def _states(call: _Call, A, B, D: int, T: int):
    """(pointer of A, N, G): A is (N, D), B has G * N rows."""
    p = call.dense(A, "A", None)
    if A is None or len(A.dims) != 2 or A.dims[1] != D:
        _fail(call.what, f"`A` must be (states, {D})")
    N = A.dims[0]
    rows, rest = N, 0
    if isinstance(B, (MLIRArray, MLIRRows)) and B.dims:
        if T:
            rows, rest = divmod(math.prod(B.dims), T)
        else:  # (N, G, no tokens) has one dimension more than u
            rows = math.prod(B.dims[:2 if len(B.dims) > len(call.lead) else 1])
    G = rows // N if N else 0
    if G < 1 or D % G or rest or rows % N:
        _fail(call.what, f"`B` has dims {getattr(B, 'dims', None)}: not (groups of) {N} rows for {T} tokens")
    return p, N, G


def _scan(call: _Call, u, delta, A, B, Cm, z, softplus, seqs):
    """(D, T, N, G, nseq) and the fields of ScanArgs: up to seqs, and from u to A."""
    pu, ldu = call.tokens(u, "u")
    T, nseq, ln, pseqs = call.sequences(u, seqs)
    n = u.dims[0]
    pA, N, G = _states(call, A, B, n, T)
    pd, pz, ldd, ldz = call.like("delta z", n, T, delta, z)
    pB, ldb = call.tokens(B, "B", G * N, T)
    pC, ldc = call.tokens(Cm, "C", G * N, T)
    return ((n, T, N, G, nseq), (_lib.MK_T[call.eltype], 1 if softplus else 0, n, N, G, T, nseq, ln, pseqs),
            (pu, pd, pz, pB, pC, ldu, ldd, ldz, ldb, ldc, pA))


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
    (n, T, N, _, nseq), head, inputs = _scan(c, u, delta, A, B, C, z, softplus, seqs)
    py, ldy = c.like("y", n, T, y)
    pi, ni = c.pool("init", init, slots, N * n, nseq)
    pl, nl = c.pool("last", last, slots, N * n, nseq)
    pslots, nslots = c.slots(slots, nseq, None if init is None else ni, None if last is None else nl)
    pD, pb = c.floats("D bias", n, D, bias)
    ps = c.dense(saved, "saved", _saved_length(u, A, T, nseq))
    c.run("mk_selective_scan", _lib.ScanArgs(*head, pslots, nslots, *inputs, pD, pb, pi, py, ldy, pl, ps),
          "mk_selective_scan_workspace")
    return y


def selective_scan_grad(du, ddelta, dA, dB, dC, dy, u, delta, A, B, C, saved, *, D=None, dD=None, z=None, dz=None,
                        bias=None, dbias=None, softplus=True, seqs=None, dinit=None, dlast=None):
    """Gradients of ``selective_scan`` for ``dy`` (and ``dlast``, that of ``last``).
    ``dB`` and ``dC`` are summed over the channels of a group, ``dA``, ``dD`` and
    ``dbias`` over all tokens.  ``saved`` is what the forward pass left, for the same
    inputs (an ``init`` is in it); ``dD``, ``dz``, ``dbias`` go with ``D``, ``z``, ``bias``.
    The workspace is 8 bytes per token, row of B and tile of 16 to 64 channels (67 MB
    for 8192 tokens of 4096 channels with 16 states, 1.07 GB with 64)."""
    c = _Call("selective_scan_grad")
    for name, given, grad in (("D", D, dD), ("z", z, dz), ("bias", bias, dbias)):
        if (given is None) != (grad is None):
            _fail(c.what, f"`d{name}` is needed exactly when `{name}` is given")
    (n, T, N, G, nseq), head, inputs = _scan(c, u, delta, A, B, C, z, softplus, seqs)
    pdy, pdu, pdd, pdz, lddy, lddu, lddd, lddz = c.like("dy du ddelta dz", n, T, dy, du, ddelta, dz)
    pdB, lddb = c.tokens(dB, "dB", G * N, T)
    pdC, lddc = c.tokens(dC, "dC", G * N, T)
    pD, pb, pdD, pdb = c.floats("D bias dD dbias", n, D, bias, dD, dbias)
    pdA = c.dense(dA, "dA", N * n)
    ps = c.dense(saved, "saved", _saved_length(u, A, T, nseq))
    pdl, pdi = c.floats("dlast dinit", N * n * nseq, dlast, dinit)
    # fields in the struct's order
    c.run("mk_selective_scan_grad", _lib.ScanArgs(
        *head, None, 0, *inputs, pD, pb, None, None, 0, None, ps, pdy, lddy, pdl, pdu, pdd, pdz, pdB, pdC, lddu, lddd,
        lddz, lddb, lddc, pdA, pdD, pdb, pdi), "mk_selective_scan_grad_workspace")
    return du


def selective_scan_step(y, next, state, u, delta, A, B, C, *, D=None, z=None, bias=None, softplus=True, slots=None):
    """One token per batch entry: ``u``, ``delta``, ``z``, ``y`` are (D, B), ``B`` and ``C``
    (N, B) or (N, G, B), ``state`` (N, D, B) or a pool with ``slots``; ``next`` receives
    the state moved on and may be ``state``.  Pool columns that no entry uses are left
    as they were."""
    c = _Call("selective_scan_step")
    pu, ldu = c.tokens(u, "u")
    dims = u.dims
    n, batch = dims[0], dims[1] if len(dims) == 2 else math.prod(dims[1:])
    pA, N, G = _states(c, A, B, n, batch)
    pB, ldb = c.tokens(B, "B", G * N, batch)
    pC, ldc = c.tokens(C, "C", G * N, batch)
    pd, pz, py, ldd, ldz, ldy = c.like("delta z y", n, batch, delta, z, y)
    ps, ns = c.pool("state", state, slots, N * n, batch)
    pn, nn = c.pool("next", next, slots, N * n, batch)
    pslots, nslots = c.slots(slots, batch, ns, nn)
    pD, pbias = c.floats("D bias", n, D, bias)
    # fields in the struct's order
    c.run("mk_selective_scan_step", _lib.ScanStepArgs(
        _lib.MK_T[c.eltype], 1 if softplus else 0, n, N, G, batch, pslots, nslots, pu, pd, pz, pB, pC, ldu, ldd, ldz,
        ldb, ldc, pA, pD, pbias, ps, pn, py, ldy))
    return y


# ---- norms around a block ----------------------------------------------------------

def _norm(call: _Call, r, w, h, hw, gate, scale, act, eps, lead):
    """NormArgs with the inputs filled in."""
    if act not in _lib.MK_ACT:
        _fail(call.what, f"no gate activation {act!r} (supported: silu, sigmoid)")
    call.tokens(lead, "h" if lead is h else "y")  # sets the call's element type
    if not isinstance(r, (MLIRArray, MLIRRows)):
        _fail(call.what, f"`r` must be an MLIRArray or rows of one, got {type(r).__name__}")
    rt = r.eltype
    if rt not in ("Float32", call.eltype):
        _fail(call.what, f"`r` has element type {rt}, expected Float32 or {call.eltype}")
    if h is None and not (gate is None and hw is None and scale is None):
        _fail(call.what, "`gate`, `hw` and `scale` belong to `h`")
    # the sizes of the call are those of its first array, which the others are compared with
    dims = lead.dims
    D, T = dims[0], dims[1] if len(dims) == 2 else math.prod(dims[1:])
    pr, ldr = call.tokens(r, "r", D, T, eltype=rt)
    ph, pg, ldh, ldg = call.like("h gate", D, T, h, gate)
    phw, psc, pw = call.floats("hw scale w", D, hw, scale, w)
    # fields in the struct's order, up to ldgate
    return _lib.NormArgs(_lib.MK_T[call.eltype], _lib.MK_T[rt], _lib.MK_ACT[act], eps, D, T, pr, ph, pg, phw, psc, pw,
                         None, None, ldr, ldh, ldg)


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
    D, T = a.D, a.T
    a.dr, a.lddr = c.tokens(dr, "dr", D, T, eltype=r.eltype)
    a.dy, a.dh, a.dgate, a.lddy, a.lddh, a.lddgate = c.like("dy dh dgate", D, T, dy, dh, dgate)
    if drout is not None:
        a.drout, a.lddrout = c.tokens(drout, "drout", D, T, eltype=r.eltype)
    a.dw, a.dhw, a.dscale = c.floats("dw dhw dscale", D, dw, dhw, dscale)
    c.run("mk_block_norm_grad", a, "mk_block_norm_grad_workspace")
    return dr
