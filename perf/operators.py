"""The state space operators of this library, as cases that can be timed and compared.

A case names one operator with its sizes.  `run` makes one pass through it: in its plain form
(elementary torch operations in 32 bits) or, where `own` is true, by the calls that a user makes
of `cutilecpu_b200`.  Tensors here are row-major (tokens, channels): the memory of the library's
column-major (channels, tokens) arrays.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CHUNK = 64  # steps of the plain recurrence that are combined by doubling


def listed():
    return [
        # one request that decodes: the latency of a call that moves half a megabyte
        {"name": "step-one", "op": "scan_step", "type": "bf16", "B": 1, "D": 1024, "N": 16, "G": 1, "pad": 0},
        # a serving batch with padded entries: bound by the state that it reads and writes
        {"name": "step-batch", "op": "scan_step", "type": "bf16", "B": 192, "D": 4096, "N": 16, "G": 1, "pad": 7},
        # prompts of several requests in one packed batch, their states kept in slots
        {"name": "prompt-ragged", "op": "scan_prompt", "type": "bf16", "lens": "1031,1,517,0,2048,96,1300,7,1000",
         "D": 2048, "N": 16, "G": 1, "state": True},
        # one long document on few channels: hardly any rows to spread over the card
        {"name": "prompt-long", "op": "scan_prompt", "type": "f16", "lens": "24577", "D": 640, "N": 16, "G": 2,
         "state": False},
        # a training step's layer
        {"name": "scan-train", "op": "scan_train", "type": "bf16", "lens": "2048,2048,2048,2048", "D": 4096, "N": 16,
         "G": 1},
        # a small model in 32 bits, odd in every size
        {"name": "scan-train-odd", "op": "scan_train", "type": "f32", "lens": "1001,3,1237,760", "D": 333, "N": 11,
         "G": 3},
        # the convolution before the scan, for packed prompts and for training
        {"name": "conv-prompt", "op": "conv_prompt", "type": "bf16", "lens": "4099,1,2500,0,8192,33,1559", "D": 4096,
         "W": 4},
        {"name": "conv-train", "op": "conv_train", "type": "bf16", "lens": "2048,2048,2048,2048", "D": 4096, "W": 4},
        {"name": "conv-step", "op": "conv_step", "type": "f32", "B": 192, "D": 4099, "W": 3, "pad": 5},
        # norms around a block: one decoded token, a training step, an odd width in 16 bits throughout
        {"name": "norm-one", "op": "norm", "type": "bf16", "res": "f32", "T": 1, "D": 2048},
        {"name": "norm-train", "op": "norm_train", "type": "bf16", "res": "f32", "T": 8192, "D": 4096},
        {"name": "norm-train-odd", "op": "norm_train", "type": "f16", "res": "f16", "T": 1027, "D": 1999},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _odd(rng, n):
    """`n`, or a neighbour that no vector width divides."""
    return n if rng.random() < 0.5 else max(1, n - n % 64 + rng.randrange(1, 64))


def _lens(rng, total):
    """Lengths of packed sequences, equal or ragged, some of them short or empty, `total` tokens at most."""
    count = _log(rng, 1, 16)
    if rng.random() < 0.4:
        return ",".join([str(max(1, total // count))] * count)
    cuts = sorted(rng.randrange(total + 1) for _ in range(count - 1))
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))


def draw(rng):
    op = rng.choice(["scan_step", "scan_prompt", "scan_prompt", "scan_train", "scan_train", "conv_prompt",
                     "conv_train", "conv_step", "norm", "norm_train"])
    case = {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op in ("scan_step", "conv_step"):
        case["D"] = _odd(rng, 16 * _log(rng, 4, 256))
        case["B"] = _log(rng, 1, 192)
        case["pad"] = rng.randrange(0, 1 + case["B"] // 4)
    if op in ("scan_prompt", "scan_train"):
        case["D"] = _odd(rng, 16 * _log(rng, 4, 256))
        most = 8192 if op == "scan_train" else 16384
        case["lens"] = _lens(rng, _log(rng, 1, max(1, min(most, (1 << 25) // case["D"]))))
    if op in ("scan_step", "scan_prompt", "scan_train"):
        case["N"] = rng.choice([16, 16, 16, 8, 5, 16])
        case["G"] = rng.choice([g for g in (1, 1, 2, 3, 4) if case["D"] % g == 0])
    if op == "scan_prompt":
        case["state"] = rng.random() < 0.5
    if op in ("conv_prompt", "conv_train"):
        case["D"] = _odd(rng, 16 * _log(rng, 4, 256))
        case["lens"] = _lens(rng, _log(rng, 1, 8192))
    if op in ("conv_prompt", "conv_train", "conv_step"):
        case["W"] = rng.choice([4, 4, 3, 2])
    if op in ("norm", "norm_train"):
        case["D"] = _odd(rng, 16 * _log(rng, 4, 256))
        case["T"] = _log(rng, 1, 8192)
        case["res"] = rng.choice(["f32", case["type"]])
    return case


# ---- inputs -----------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    dt = TYPES[case["type"]]
    s = {"op": case["op"], "dt": dt}

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(shape, generator=g, device="cuda")

    op, D = case["op"], case["D"]
    if "lens" in case:
        lens = [int(x) for x in case["lens"].split(",")]
        T, S = sum(lens), len(lens)
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        s.update(lens=lens, starts=starts, T=T, S=S)
        s["seqs"] = torch.tensor(starts, dtype=torch.int32, device="cuda") + 1
        rows = T
    else:
        rows = case.get("B", case.get("T"))
    if op.startswith("scan"):
        N, G = case["N"], case["G"]
        s.update(N=N, G=G, D=D, rows=rows)
        s["u"] = torch.nn.functional.silu(normal(rows, D)).to(dt)
        s["delta"] = (0.5 * normal(rows, D)).to(dt)
        step = torch.exp(uniform(math.log(1e-3), math.log(0.1), D))
        s["bias"] = step + torch.log(-torch.expm1(-step))  # softplus(bias) is a step of 0.001 to 0.1
        s["A"] = -(torch.arange(1, N + 1, device="cuda", dtype=torch.float32)[None, :] * torch.exp(0.1 * normal(D, N)))
        s["B"] = normal(rows, G, N).to(dt)
        s["C"] = normal(rows, G, N).to(dt)
        s["skip"] = 1.0 + 0.1 * normal(D)
        s["z"] = normal(rows, D).to(dt)
        s["y"] = torch.empty(rows, D, dtype=dt, device="cuda")
    elif op.startswith("conv"):
        W = case["W"]
        s.update(W=W, D=D, rows=rows)
        s["x"] = normal(rows, D).to(dt)
        s["w"] = uniform(-1, 1, W, D) / math.sqrt(W)
        s["bias"] = uniform(-0.5, 0.5, D)
        s["y"] = torch.empty(rows, D, dtype=dt, device="cuda")
    else:
        rt = TYPES[case["res"]]
        s.update(D=D, rows=rows, rt=rt, eps=1e-5)
        s["r"] = (2.0 * normal(rows, D)).to(rt)
        s["h"] = normal(rows, D).to(dt)
        s["gate"] = normal(rows, D).to(dt)
        s["hw"] = 1.0 + 0.1 * normal(D)
        s["w"] = 1.0 + 0.1 * normal(D)
        s["scale"] = 0.5 + 0.1 * normal(D)
        s["y"] = torch.empty(rows, D, dtype=dt, device="cuda")
        s["rout"] = torch.empty(rows, D, dtype=rt, device="cuda")
    if op.endswith("step"):
        pool = rows + 5
        slots = torch.randperm(pool, generator=g, device="cuda")[:rows] + 1
        slots[rows - case["pad"]:] = 0  # padded entries of the batch
        s["slots"] = slots.to(torch.int32)
        s["state"] = normal(pool, D, case["N"]) if op == "scan_step" else normal(pool, case["W"] - 1, D).to(dt)
        s["next"] = s["state"].clone()
        s["y"].zero_()
    elif op in ("scan_prompt", "conv_prompt"):
        pool = s["S"] + 3
        s["slots"] = (torch.randperm(pool, generator=g, device="cuda")[:s["S"]] + 1).to(torch.int32)
        shape = (pool, D, case["N"]) if op == "scan_prompt" else (pool, case["W"] - 1, D)
        s["last"] = torch.zeros(shape, dtype=torch.float32 if op == "scan_prompt" else dt, device="cuda")
        has = case.get("state", True)
        s["init"] = normal(*shape).to(s["last"].dtype) if has else None
    elif op.endswith("train"):
        s["dy"] = (normal(rows, D)).to(dt)
        if op == "norm_train":
            s["drout"] = normal(rows, D).to(s["rt"])
    if own:
        _prepare_own(s)
    return s


def _prepare_own(s):
    import cutilecpu_b200 as mk
    be = mk.MLIRCUDABackend()
    a = {}
    for k, v in s.items():
        if isinstance(v, torch.Tensor):
            a[k] = mk.MLIRArray(v.view(-1), dims=tuple(reversed(v.shape)))

    def grad(name, like, dt=None):
        s[name] = torch.empty(s[like].shape, dtype=dt or s[like].dtype, device="cuda")
        a[name] = mk.MLIRArray(s[name].view(-1), dims=tuple(reversed(s[name].shape)))

    f32 = torch.float32
    if s["op"] == "scan_train":
        for k in ("u", "delta", "z", "B", "C", "A", "skip", "bias"):
            grad("d" + k, k)
        a["saved"] = mk.selective_scan_saved(a["u"], a["A"], seqs=a["seqs"])
    elif s["op"] == "conv_train":
        for k in ("x", "w", "bias"):
            grad("d" + k, k)
    elif s["op"] == "norm_train":
        for k in ("r", "h", "gate"):
            grad("d" + k, k)
        for k in ("hw", "w", "scale"):
            grad("d" + k, k, f32)
    s["mk"], s["be"], s["a"] = mk, be, a


# ---- one pass ---------------------------------------------------------------------------------

def run(s):
    return globals()[("_own_" if own else "_plain_") + s["op"]](s)


def _own_scan_step(s):
    a = s["a"]
    s["mk"].selective_scan_step(a["y"], a["next"], a["state"], a["u"], a["delta"], a["A"], a["B"], a["C"],
                                D=a["skip"], z=a["z"], bias=a["bias"], slots=a["slots"])
    return {"y": s["y"], "state": s["next"]}


def _own_scan_prompt(s):
    a = s["a"]
    s["mk"].selective_scan(a["y"], a["u"], a["delta"], a["A"], a["B"], a["C"], D=a["skip"], z=a["z"],
                           bias=a["bias"], seqs=a["seqs"], init=a.get("init"), last=a["last"], slots=a["slots"])
    return {"y": s["y"], "state": s["last"]}


def _own_scan_train(s):
    a, mk = s["a"], s["mk"]
    mk.selective_scan(a["y"], a["u"], a["delta"], a["A"], a["B"], a["C"], D=a["skip"], z=a["z"], bias=a["bias"],
                      seqs=a["seqs"], saved=a["saved"])
    mk.selective_scan_grad(a["du"], a["ddelta"], a["dA"], a["dB"], a["dC"], a["dy"], a["u"], a["delta"], a["A"],
                           a["B"], a["C"], a["saved"], D=a["skip"], dD=a["dskip"], z=a["z"], dz=a["dz"],
                           bias=a["bias"], dbias=a["dbias"], seqs=a["seqs"])
    return {k: s[k] for k in ("y", "du", "ddelta", "dz", "dA", "dB", "dC", "dskip", "dbias")}


def _own_conv_step(s):
    a = s["a"]
    s["mk"].causal_conv_step(a["y"], a["next"], a["state"], a["x"], a["w"], bias=a["bias"], slots=a["slots"])
    return {"y": s["y"], "state": s["next"]}


def _own_conv_prompt(s):
    a = s["a"]
    s["mk"].causal_conv(a["y"], a["x"], a["w"], bias=a["bias"], seqs=a["seqs"], init=a["init"], last=a["last"],
                        slots=a["slots"])
    return {"y": s["y"], "state": s["last"]}


def _own_conv_train(s):
    a, mk = s["a"], s["mk"]
    mk.causal_conv(a["y"], a["x"], a["w"], bias=a["bias"], seqs=a["seqs"])
    mk.causal_conv_grad(a["dx"], a["dw"], a["dy"], a["x"], a["w"], bias=a["bias"], dbias=a["dbias"], seqs=a["seqs"])
    return {k: s[k] for k in ("y", "dx", "dw", "dbias")}


def _own_norm(s):
    a = s["a"]
    s["mk"].block_norm(a["y"], a["rout"], a["r"], a["w"], h=a["h"], hw=a["hw"], gate=a["gate"], scale=a["scale"],
                       eps=s["eps"])
    return {"y": s["y"], "rout": s["rout"]}


def _own_norm_train(s):
    a, mk = s["a"], s["mk"]
    mk.block_norm(a["y"], a["rout"], a["r"], a["w"], h=a["h"], hw=a["hw"], gate=a["gate"], scale=a["scale"],
                  eps=s["eps"])
    mk.block_norm_grad(a["dr"], a["dw"], a["dy"], a["r"], a["w"], drout=a["drout"], h=a["h"], dh=a["dh"],
                       hw=a["hw"], dhw=a["dhw"], gate=a["gate"], dgate=a["dgate"], scale=a["scale"],
                       dscale=a["dscale"], eps=s["eps"])
    return {k: s[k] for k in ("y", "rout", "dr", "dh", "dgate", "dw", "dhw", "dscale")}


# ---- plain forms: 32 bits, rounded once at the end -----------------------------------------------

def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _softplus(x):
    return torch.where(x > 20.0, x, torch.log1p(torch.exp(torch.clamp(x, max=20.0))))


def _recur(a, b):
    """h[t] = a[t] h[t-1] + b[t] from h = 0 along the first dimension: doubling inside chunks, then a chain
    over the chunks."""
    T = a.shape[0]
    if T == 0:
        return b
    nc = -(-T // CHUNK)
    if nc * CHUNK != T:
        tail = (nc * CHUNK - T,) + tuple(a.shape[1:])
        a, b = torch.cat([a, a.new_ones(tail)]), torch.cat([b, b.new_zeros(tail)])
    a, b = a.view(nc, CHUNK, *a.shape[1:]), b.view(nc, CHUNK, *b.shape[1:])
    k = 1
    while k < CHUNK:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    h, starts = torch.zeros_like(b[0, 0]), []
    for c in range(nc):
        starts.append(h)
        h = a[c, -1] * h + b[c, -1]
    b = b + a * torch.stack(starts)[:, None]
    return b.view(nc * CHUNK, *b.shape[2:])[:T]


def _per_channel(m, D):
    """(rows, G, N) of the groups as (rows, D, N) of their channels."""
    return m.float().repeat_interleave(D // m.shape[1], dim=1)


def _plain_scan(s, h0=None):
    """What the forward pass computes, and the values that its gradient takes up again."""
    D = s["D"]
    u, z = s["u"].float(), s["z"].float()
    raw = s["delta"].float() + s["bias"]
    dl = _softplus(raw)
    Bd, Cd = _per_channel(s["B"], D), _per_channel(s["C"], D)
    a = torch.exp(dl[..., None] * s["A"])
    b = (dl * u)[..., None] * Bd
    first = [p for p, n in zip(s["starts"], s["lens"]) if n]
    cut = a.clone()
    cut[first] = 0.0  # no sequence sees the one before it
    if h0 is not None:
        some = [i for i, n in enumerate(s["lens"]) if n]
        b[first] = b[first] + a[first] * h0[some]
    h = _recur(cut, b)
    yp = (h * Cd).sum(-1) + s["skip"] * u
    return u, z, raw, dl, Bd, Cd, a, cut, h, yp, first


def _plain_scan_step(s):
    live = s["slots"] > 0
    at = torch.clamp(s["slots"].long() - 1, min=0)
    u, z = s["u"].float(), s["z"].float()
    dl = _softplus(s["delta"].float() + s["bias"])
    h = torch.exp(dl[..., None] * s["A"]) * s["state"][at] + (dl * u)[..., None] * _per_channel(s["B"], s["D"])
    y = ((h * _per_channel(s["C"], s["D"])).sum(-1) + s["skip"] * u) * (z * _sigmoid(z))
    state = s["state"].clone()
    state[at[live]] = h[live]
    return {"y": torch.where(live[:, None], y, 0.0).to(s["dt"]), "state": state}


def _plain_scan_prompt(s):
    at = s["slots"].long() - 1
    h0 = s["init"][at] if s["init"] is not None else s["last"].new_zeros(s["S"], s["D"], s["N"])
    u, z, raw, dl, Bd, Cd, a, cut, h, yp, first = _plain_scan(s, h0)
    state = torch.zeros_like(s["last"])
    ends = torch.stack([h[p + n - 1] if n else h0[i] for i, (p, n) in enumerate(zip(s["starts"], s["lens"]))])
    state[at] = ends
    return {"y": (yp * (z * _sigmoid(z))).to(s["dt"]), "state": state}


def _plain_scan_train(s):
    dt, D, G, N = s["dt"], s["D"], s["G"], s["N"]
    u, z, raw, dl, Bd, Cd, a, cut, h, yp, first = _plain_scan(s)
    sz = _sigmoid(z)
    y = yp * (z * sz)
    dy = s["dy"].float()
    dyp = dy * (z * sz)
    dz = dy * yp * (sz * (1.0 + z * (1.0 - sz)))
    # g[t] = C[t] dyp[t] + a[t+1] g[t+1]: the same recurrence from the end, cut where a sequence begins
    ahead = torch.cat([cut[1:], torch.zeros_like(cut[:1])])
    g = _recur(ahead.flip(0), (Cd * dyp[..., None]).flip(0)).flip(0)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before[first] = 0.0
    q = g * a * before
    gB = (g * Bd).sum(-1)
    dA = (q * dl[..., None]).sum(0)
    ddl = (q * s["A"]).sum(-1) + u * gB
    du = dl * gB + s["skip"] * dyp
    draw_ = ddl * _sigmoid(raw)
    rows = s["rows"]
    dB = (g * (dl * u)[..., None]).view(rows, G, D // G, N).sum(2)
    dC = (h * dyp[..., None]).view(rows, G, D // G, N).sum(2)
    return {"y": y.to(dt), "du": du.to(dt), "ddelta": draw_.to(dt), "dz": dz.to(dt), "dA": dA, "dB": dB.to(dt),
            "dC": dC.to(dt), "dskip": (dyp * u).sum(0), "dbias": draw_.sum(0)}


def _plain_conv_step(s):
    live = s["slots"] > 0
    at = torch.clamp(s["slots"].long() - 1, min=0)
    seen = torch.cat([s["state"][at], s["x"][:, None]], 1)
    pre = s["bias"] + (s["w"] * seen.float()).sum(1)
    state = s["state"].clone()
    state[at[live]] = seen[live][:, 1:]
    return {"y": torch.where(live[:, None], pre * _sigmoid(pre), 0.0).to(s["dt"]), "state": state}


def _back(s, x, k, h0=None):
    """`x` k tokens earlier, zero (or the state) where that lies before the sequence."""
    out = torch.cat([torch.zeros_like(x[:k]), x[:max(0, x.shape[0] - k)]])[:x.shape[0]]
    for i, (p, n) in enumerate(zip(s["starts"], s["lens"])):
        if n:
            m = min(k, n)
            out[p:p + m] = 0.0 if h0 is None else h0[i, s["W"] - 1 - k:s["W"] - 1 - k + m]
    return out


def _ahead(s, x, k):
    out = torch.cat([x[k:], torch.zeros_like(x[:k])])[:x.shape[0]]
    for p, n in zip(s["starts"], s["lens"]):
        if n:
            out[p + n - min(k, n):p + n] = 0.0
    return out


def _plain_conv_prompt(s):
    W, at = s["W"], s["slots"].long() - 1
    x, h0 = s["x"].float(), s["init"][at].float()
    pre = s["bias"] + sum(s["w"][W - 1 - k] * (_back(s, x, k, h0) if k else x) for k in range(W))
    state = torch.zeros_like(s["last"])
    for i, (p, n) in enumerate(zip(s["starts"], s["lens"])):
        state[at[i]] = torch.cat([h0[i].to(s["dt"]), s["x"][p:p + n]])[-(W - 1):]
    return {"y": (pre * _sigmoid(pre)).to(s["dt"]), "state": state}


def _plain_conv_train(s):
    W = s["W"]
    x, dy = s["x"].float(), s["dy"].float()
    seen = [_back(s, x, k) if k else x for k in range(W)]
    pre = s["bias"] + sum(s["w"][W - 1 - k] * seen[k] for k in range(W))
    sg = _sigmoid(pre)
    dp = dy * (sg * (1.0 + pre * (1.0 - sg)))
    dx = sum(s["w"][W - 1 - k] * (_ahead(s, dp, k) if k else dp) for k in range(W))
    dw = torch.stack([(dp * seen[W - 1 - k]).sum(0) for k in range(W)])
    return {"y": (pre * sg).to(s["dt"]), "dx": dx.to(s["dt"]), "dw": dw, "dbias": dp.sum(0)}


def _plain_block(s):
    r, h, gate = s["r"].float(), s["h"].float(), s["gate"].float()
    i1 = torch.rsqrt((h * h).mean(-1, keepdim=True) + s["eps"])
    n = h * i1 * s["hw"]
    sg = _sigmoid(gate)
    m = n * (gate * sg)
    rout = r + s["scale"] * m
    i2 = torch.rsqrt((rout * rout).mean(-1, keepdim=True) + s["eps"])
    return h, gate, i1, n, sg, m, rout, i2


def _plain_norm(s):
    h, gate, i1, n, sg, m, rout, i2 = _plain_block(s)
    return {"y": (rout * i2 * s["w"]).to(s["dt"]), "rout": rout.to(s["rt"])}


def _plain_norm_train(s):
    h, gate, i1, n, sg, m, rout, i2 = _plain_block(s)
    dt, dy = s["dt"], s["dy"].float()
    xh = rout * i2
    dxh = dy * s["w"]
    dro = s["drout"].float() + i2 * (dxh - xh * (dxh * xh).mean(-1, keepdim=True))
    dm = dro * s["scale"]
    dn = dm * (gate * sg)
    dgate = dm * n * (sg * (1.0 + gate * (1.0 - sg)))
    hh = h * i1
    dhh = dn * s["hw"]
    dh = i1 * (dhh - hh * (dhh * hh).mean(-1, keepdim=True))
    return {"y": (xh * s["w"]).to(dt), "rout": rout.to(s["rt"]), "dr": dro.to(s["rt"]), "dh": dh.to(dt),
            "dgate": dgate.to(dt), "dw": (dy * xh).sum(0), "dhw": (dn * hh).sum(0), "dscale": (dro * m).sum(0)}


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    op, D, e = case["op"], case["D"], TYPES[case["type"]].itemsize
    if "lens" in case:
        rows, S = sum(int(x) for x in case["lens"].split(",")), len(case["lens"].split(","))
    else:
        rows, S = case.get("B", case.get("T")), 0
    if op.startswith("scan"):
        N, G = case["N"], case["G"]
        cell, bc, par = rows * D, 2 * rows * G * N, 4 * D * (N + 2)
        if op == "scan_step":
            live = rows - case["pad"]
            return {"bytes": e * (4 * live * D + 2 * live * G * N) + 8 * live * D * N + par,
                    "flops": live * D * (7 * N + 12)}
        if op == "scan_prompt":
            return {"bytes": e * (4 * cell + bc) + par + 4 * S * D * N * (2 if case["state"] else 1),
                    "flops": cell * (7 * N + 12)}
        return {"bytes": e * (8 * cell + 2 * bc) + 2 * par, "flops": cell * (26 * N + 40)}
    if op.startswith("conv"):
        W = case["W"]
        cell, par = rows * D, 4 * D * (W + 1)
        if op == "conv_step":
            live = rows - case["pad"]
            return {"bytes": e * live * D * (2 + 2 * (W - 1)) + par, "flops": live * D * (2 * W + 5)}
        if op == "conv_prompt":
            return {"bytes": e * (2 * cell + 2 * S * (W - 1) * D) + par, "flops": cell * (2 * W + 5)}
        return {"bytes": e * 4 * cell + 2 * par, "flops": cell * (6 * W + 12)}
    q, cell = TYPES[case["res"]].itemsize, rows * D
    if op == "norm":
        return {"bytes": cell * (2 * q + 3 * e) + 12 * D, "flops": cell * 15}
    return {"bytes": cell * (4 * q + 6 * e) + 24 * D, "flops": cell * 50}


# ---- the definition in 64 bits: token by token, gradients by differentiation -----------------------

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    v = {k: (x.double() if isinstance(x, torch.Tensor) and x.is_floating_point() else x) for k, x in s.items()}
    op = case["op"]
    if op.startswith("norm"):
        return _exact_norm(v, op == "norm_train")
    if op.endswith("step"):
        return _exact_step(v, op)
    train = op.endswith("train")
    names = (["u", "delta", "z", "A", "B", "C", "skip", "bias"] if op.startswith("scan") else ["x", "w", "bias"])
    if train:
        for k in names:
            v[k].requires_grad_()
    with torch.set_grad_enabled(train):
        y, ends = (_exact_scan if op.startswith("scan") else _exact_conv)(v)
        if train:
            grads = torch.autograd.grad(y, [v[k] for k in names], v["dy"])
            return {"y": y.detach(), **{"d" + k: x for k, x in zip(names, grads)}}
    state = torch.zeros_like(v["last"])
    for i, slot in enumerate(s["slots"].tolist()):
        state[slot - 1] = ends[i]
    return {"y": y, "state": state}


def _padded(v):
    """Where token t of sequence i stands, (longest, S), and which places of it are none."""
    most = max(v["lens"])
    t = torch.arange(most)[:, None]
    lens, starts = torch.tensor(v["lens"]), torch.tensor(v["starts"][:-1])
    live = t < lens
    return torch.where(live, starts + t, 0).cuda(), live.cuda(), live


def _start(v, shape):
    if v.get("init") is None:
        return torch.zeros(shape, dtype=torch.float64, device="cuda")
    return v["init"][v["slots"].long() - 1]


def _exact_scan(v):
    where, live, _ = _padded(v)
    D, N, G, S = v["D"], v["N"], v["G"], v["S"]
    group = torch.arange(D, device="cuda") // (D // G)
    h = _start(v, (S, D, N))
    dl_all = torch.nn.functional.softplus(v["delta"] + v["bias"], threshold=700.0)
    out = []
    for t in range(where.shape[0]):
        w = where[t]
        dl = dl_all[w][..., None]
        new = torch.exp(dl * v["A"]) * h + dl * v["u"][w][..., None] * v["B"][w][:, group]
        h = torch.where(live[t][:, None, None], new, h)
        out.append((new * v["C"][w][:, group]).sum(-1))
    y = torch.stack(out)[live]  # token by token over the sequences: put back in their order
    y = torch.empty_like(y).index_copy(0, where[live], y)
    return (y + v["skip"] * v["u"]) * torch.nn.functional.silu(v["z"]), h


def _exact_conv(v):
    W, ys, ends = v["W"], [], []
    h0 = _start(v, (v["S"], W - 1, v["D"]))
    for i, (p, n) in enumerate(zip(v["starts"], v["lens"])):
        seen = torch.cat([h0[i], v["x"][p:p + n]])
        ys.append(sum(v["w"][k] * seen[k:k + n] for k in range(W)) + v["bias"])
        ends.append(seen[n:])
    return torch.nn.functional.silu(torch.cat(ys)), ends


def _exact_step(v, op):
    state, y = v["state"].clone(), torch.zeros_like(v["y"])
    for i, slot in enumerate(v["slots"].tolist()):
        if slot == 0:
            continue
        if op == "conv_step":
            seen = torch.cat([v["state"][slot - 1], v["x"][i:i + 1]])
            state[slot - 1] = seen[1:]
            y[i] = torch.nn.functional.silu((seen * v["w"]).sum(0) + v["bias"])
        else:
            dl = torch.nn.functional.softplus(v["delta"][i] + v["bias"], threshold=700.0)[:, None]
            rep = v["D"] // v["G"]
            h = torch.exp(dl * v["A"]) * v["state"][slot - 1]
            h = h + dl * v["u"][i][:, None] * v["B"][i].repeat_interleave(rep, 0)
            state[slot - 1] = h
            y[i] = (h * v["C"][i].repeat_interleave(rep, 0)).sum(-1) + v["skip"] * v["u"][i]
            y[i] *= torch.nn.functional.silu(v["z"][i])
    return {"y": y, "state": state}


def _exact_norm(v, train):
    names = ["r", "h", "gate", "w", "hw", "scale"]
    if train:
        for k in names:
            v[k].requires_grad_()

    def rms(x, w):
        return x / torch.sqrt(torch.mean(x ** 2, -1, keepdim=True) + v["eps"]) * w

    with torch.set_grad_enabled(train):
        rout = v["r"] + v["scale"] * rms(v["h"], v["hw"]) * torch.nn.functional.silu(v["gate"])
        y = rms(rout, v["w"])
        if not train:
            return {"y": y, "rout": rout}
        grads = torch.autograd.grad([y, rout], [v[k] for k in names], [v["dy"], v["drout"]])
    return {"y": y.detach(), "rout": rout.detach(), **{"d" + k: x for k, x in zip(names, grads)}}
