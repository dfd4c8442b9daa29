"""Cases that measure the operators of the gated recurrent block.

Three operators, used together by a recurrent block over node histories:

* ``scan``: the gated linear recurrence. Per step the input row is ``(x | r | i)``, each
  H wide; ``z = -rate softplus(decay) sigmoid(r)``, ``a = exp(z)``,
  ``h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) x_t``. A masked step carries the state.
  ``step`` is its form for one new token per row, which updates a table of states in place.
* ``norm``: ``v = rms(u) w_post``, ``y = x + scale sigmoid(gate) v``, ``n = rms(y) w_pre``.
* ``pack``: activations in 8 bits, groups of 32 along a row with one fp32 scale each.

``checkpoint`` cases of ``scan`` and ``norm`` keep their inputs in 8 bits between the
forward and the backward pass; gradients are those at the values that the codes stand for.
For the recurrence the states h are kept in 32 bits every 16 steps, and the backward pass
recomputes the steps in between from the codes.
"""
from __future__ import annotations

import math

import torch

own = False

RATE = 8.0
EPS = 1e-6
GROUP = 32
KEEP = 16  # steps between the states that the recurrence keeps

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "bf16": 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one training window of the MPNN-LSTM configuration: 8 snapshots of 200,000 nodes, hidden 64,
        # time-major as the snapshots are stacked
        dict(name="scan window fp32", op="scan", layout="time", batch=200_000, steps=8, width=64, dtype="fp32",
             mask=False, checkpoint=False),
        # a T-GCN window (4 snapshots, hidden 128, a rank's share of the nodes), inputs kept in 8 bits
        dict(name="scan window 8-bit", op="scan", layout="time", batch=400_000, steps=4, width=128, dtype="fp32",
             mask=False, checkpoint=True),
        # a few very long streams, as one sequence per community or per site
        dict(name="scan long bf16", op="scan", layout="batch", batch=2, steps=65_537, width=256, dtype="bf16",
             mask=False, checkpoint=False),
        # nodes absent from some or all snapshots, odd sizes; absent rows hold NaN
        dict(name="scan masked odd", op="scan", layout="batch", batch=37, steps=1001, width=65, dtype="fp32",
             mask=True, checkpoint=False),
        # event histories of unequal lengths (a few hubs, many short ones, empty ones), hidden 100 as in TGN
        dict(name="scan histories", op="scan", layout="packed", batch=20_000, steps=1_000_000, width=100,
             dtype="fp32", mask=False, checkpoint=False),
        # one new event batch: 600 roots read and update their rows of a table of node states
        dict(name="step 600 rows", op="step", batch=600, table=9_000, width=100, dtype="fp32"),
        # the block's norms over that window: 8 x 200,000 rows of 64
        dict(name="norm window fp32", op="norm", rows=1_600_000, width=64, dtype="fp32", train=True,
             checkpoint=False),
        # wide rows in bf16
        dict(name="norm wide bf16", op="norm", rows=16_384, width=2048, dtype="bf16", train=True, checkpoint=False),
        # JODIE's width, inputs kept in 8 bits
        dict(name="norm 8-bit", op="norm", rows=400_000, width=172, dtype="fp32", train=True, checkpoint=True),
        # the 600 roots of one new event batch, no gradient
        dict(name="norm 600 rows", op="norm", rows=600, width=100, dtype="fp32", train=False, checkpoint=False),
        # the saved activations of one layer of that window, packed and restored
        dict(name="pack window fp32", op="pack", rows=1_600_000, width=64, dtype="fp32"),
        # a batch of neighbour rows at JODIE's width
        dict(name="pack rows bf16", op="pack", rows=48_001, width=172, dtype="bf16"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """One case of the ranges above; its elements are at most those of the largest listed case of its kind."""
    op = rng.choice(["scan", "scan", "scan", "step", "norm", "norm", "pack"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "step":
        rows = _log(rng, 1, 200_000)
        return dict(op=op, batch=rows, table=rows + _log(rng, 1, 20_000), width=_log(rng, 1, 512), dtype=dtype)
    if op == "pack":
        width = _log(rng, 1, 2048)
        return dict(op=op, rows=_log(rng, 1, 100_000_000 // width), width=width, dtype=dtype)
    if op == "norm":
        width = _log(rng, 8, 2048)
        return dict(op=op, rows=_log(rng, 1, min(1_600_000, 60_000_000 // width)), width=width, dtype=dtype,
                    train=rng.random() < 0.75, checkpoint=rng.random() < 0.4)
    layout = rng.choice(["time", "batch", "packed"])
    width = _log(rng, 4, 512)
    most = 60_000_000 // width  # steps over all sequences
    if layout == "packed":
        steps = _log(rng, 100, min(most, 1_000_000))
        return dict(op=op, layout=layout, batch=_log(rng, 1, max(2, steps // 4)), steps=steps, width=width,
                    dtype=dtype, mask=rng.random() < 0.3, checkpoint=rng.random() < 0.4)
    steps = _log(rng, 1, min(most, 65_536))
    return dict(op=op, layout=layout, batch=_log(rng, 1, max(2, min(200_000, most // steps))), steps=steps,
                width=width, dtype=dtype, mask=rng.random() < 0.3, checkpoint=rng.random() < 0.4)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(total: int, count: int, g: torch.Generator) -> torch.Tensor:
    """Lengths of `count` histories that sum to `total`: heavy-tailed, every 17th one empty."""
    w = torch.rand(count, generator=g, device="cuda").clamp_min(1e-4).pow(-0.7)
    w[::17] = 0.0
    if count < 2:
        w[:] = 1.0
    cut = torch.floor(torch.cumsum(w.double(), 0) / w.double().sum() * total + 0.5).long()
    cut[-1] = total
    return torch.diff(cut, prepend=cut.new_zeros(1))


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    H = case["width"]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    s = {"case": case}
    if case["op"] in ("scan", "step"):
        # decays of 0.9 to 0.999 a step at an open half gate: softplus(decay) rate / 2 = -log(a)
        a = 1 - 10 ** -(1 + 2 * torch.rand(H, generator=g, device="cuda"))
        s["decay"] = torch.log(torch.expm1(-torch.log(a) * 2 / RATE))
    if case["op"] == "step":
        s["p"] = normal(case["batch"], 3 * H)
        s["state"] = normal(case["table"], H, std=0.5, dtype=torch.float32)
        s["rows"] = torch.randperm(case["table"], generator=g, device="cuda")[: case["batch"]].contiguous()
        return s
    if case["op"] == "scan":
        B, T = case["batch"], case["steps"]
        lead = {"time": (T, B), "batch": (B, T), "packed": (T,)}[case["layout"]]
        p = normal(*lead, 3 * H)
        s["dh"] = normal(*lead, H)
        s["mask"] = None
        if case["mask"]:
            m = torch.rand(*lead, generator=g, device="cuda") < 0.8
            gone = torch.rand(B, generator=g, device="cuda") < 0.1  # sequences without any valid step
            if case["layout"] == "time":
                m &= ~gone
            elif case["layout"] == "batch":
                m &= ~gone.unsqueeze(1)
            p[~m] = float("nan")
            s["mask"] = m
        if case["layout"] == "time":  # [batch, steps, ...] views of stacked snapshots
            p, s["dh"] = p.transpose(0, 1), s["dh"].transpose(0, 1)
            s["mask"] = None if s["mask"] is None else s["mask"].transpose(0, 1)
        s["offsets"] = None
        if case["layout"] == "packed":
            s["offsets"] = torch.cumsum(torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"),
                                                   _lengths(T, B, g)]), 0)
        s["p"] = p.requires_grad_()
        s["h0"] = normal(B, H, std=0.5, dtype=torch.float32).requires_grad_()
        s["dlast"] = normal(B, H, dtype=torch.float32)
        s["decay"] = s["decay"].requires_grad_()
        return s
    R = case["rows"]
    s["x"] = normal(R, H)
    if case["op"] == "pack":  # rows of unequal size, some of them zero (padding)
        s["x"] *= torch.exp(torch.randn(R, 1, generator=g, device="cuda")).to(dt)
        s["x"][::101] = 0
        return s
    s["u"], s["gate"] = normal(R, H, std=0.7), normal(R, H)
    s["w_post"] = 1 + normal(H, std=0.1, dtype=torch.float32)
    s["w_pre"] = 1 + normal(H, std=0.1, dtype=torch.float32)
    s["scale"] = 0.5 + normal(H, std=0.1, dtype=torch.float32)
    if case["train"]:
        s["dy"], s["dn"] = normal(R, H), normal(R, H)
        for k in ("x", "u", "gate", "w_post", "w_pre", "scale"):
            s[k].requires_grad_()
    return s


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _run_own(s: dict):
    from starry_unigraph.ops.checkpoint8 import quantize8
    from starry_unigraph.ops.norm import norm_residual
    from starry_unigraph.ops.recurrence import gated_scan, gated_scan_step

    c = s["case"]
    if c["op"] == "step":
        h = gated_scan_step(s["p"], s["decay"], s["state"], s["rows"], rate=RATE)
        return {"h": h, "state": s["state"]}
    if c["op"] == "pack":
        q = quantize8(s["x"])
        return {"x": q.dequantize(), "scales": q.scales}
    keep = "int8" if c["checkpoint"] else None
    if c["op"] == "scan":
        h, last = gated_scan(s["p"], s["decay"], s["h0"], mask=s["mask"], offsets=s["offsets"], rate=RATE,
                             checkpoint=keep)
        dp, dd, d0 = torch.autograd.grad((h, last), (s["p"], s["decay"], s["h0"]), (s["dh"], s["dlast"]))
        return {"h": h.detach(), "last": last.detach(), "dp": dp, "ddecay": dd, "dh0": d0}
    y, n = norm_residual(s["x"], s["u"], s["w_post"], s["w_pre"], gate=s["gate"], scale=s["scale"], eps=EPS,
                         checkpoint=keep)
    if not c["train"]:
        return {"y": y, "n": n}
    names = ("x", "u", "gate", "w_post", "w_pre", "scale")
    grads = torch.autograd.grad((y, n), [s[k] for k in names], (s["dy"], s["dn"]))
    return {"y": y.detach(), "n": n.detach(), **{"d" + k: v for k, v in zip(names, grads)}}


# ---------------------------------------------------------------------------
# plain form: elementary torch operations in fp32
# ---------------------------------------------------------------------------
def _codes(x: torch.Tensor):
    """(values that the 8-bit codes of x stand for, scales), in the type of x."""
    H = x.size(-1)
    v = torch.nn.functional.pad(x, (0, -H % GROUP)).unflatten(-1, (-1, GROUP))
    top = v.abs().amax(-1, keepdim=True)
    tiny = top < 2.0 ** -100
    inv = torch.where(tiny, torch.zeros_like(top), torch.full_like(top, 127.0) / top)
    scale = torch.where(tiny, torch.zeros_like(top), top * (1.0 / 127.0))
    q = torch.clamp(torch.round(v * inv), -127, 127)
    return (q * scale).flatten(-2)[..., :H], scale.squeeze(-1)


def _doubling(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """Inclusive scan of h = a h + b over dimension 0 by doubling (log2 of the length passes over the data)."""
    k = 1
    while k < a.size(0):
        b = torch.cat([b[:k], torch.addcmul(b[k:], a[k:], b[:-k])])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _gates(p: torch.Tensor, decay: torch.Tensor, mask):
    """Per step (time first): a, sqrt(1 - a^2), z, sigmoid(r), sigmoid(i), x; a masked step has a = 1 and x = 0."""
    if mask is not None:
        p = torch.where(mask.unsqueeze(-1), p, torch.zeros_like(p))
    x, r, i = p.chunk(3, -1)
    sr, si = torch.sigmoid(r), torch.sigmoid(i)
    z = -RATE * torch.nn.functional.softplus(decay) * sr
    if mask is not None:
        z = z * mask.unsqueeze(-1)
    return torch.exp(z), torch.sqrt(-torch.expm1(2 * z)), z, sr, si, x


def _run_scan(s: dict):
    c = s["case"]
    packed = c["layout"] == "packed"
    p, dh, mask = s["p"].float(), s["dh"].float(), s["mask"]
    if not packed:  # time first
        p, dh = p.transpose(0, 1), dh.transpose(0, 1)
        mask = None if mask is None else mask.transpose(0, 1)
    h0, dlast, decay = s["h0"].float(), s["dlast"].float(), s["decay"].float()
    T = p.size(0)
    if packed:
        lo, hi = s["offsets"][:-1], s["offsets"][1:]
        live = hi > lo
        first, final = lo[live], hi[live] - 1
    a, sq, z, sr, si, x = _gates(p, decay, mask)
    b = sq * si * x
    start = a.clone()  # the factor of h0 at a first step, and 0 between sequences
    if packed:
        b[first] += a[first] * h0[live]
        start[first] = 0
    else:
        b[0] += a[0] * h0
    h = _doubling(start, b)
    if packed:
        last = h0.clone()
        last[live] = h[final]
        before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
        before[first] = h0[live]
    else:
        last = h[-1]
        before = torch.cat([h0.unsqueeze(0), h[:-1]])
    if c["checkpoint"]:
        # gradients at the values of the codes; the states before every KEEP steps are the forward's
        x3 = p.unflatten(-1, (3, -1))
        if mask is not None:
            x3 = torch.where(mask[..., None, None], x3, torch.zeros_like(x3))
        a, sq, z, sr, si, x = _gates(_codes(x3)[0].flatten(-2), decay, mask)
        b = sq * si * x
        start = a.clone()
        if packed:
            b[first] += a[first] * h0[live]
            start[first] = 0
        keep = torch.arange(0, T, KEEP, device=p.device)
        b[keep] = torch.addcmul(b[keep], start[keep], before[keep])
        pad = -T % KEEP
        fold = lambda v: torch.nn.functional.pad(v, (0, 0) * (v.dim() - 1) + (0, pad)).unflatten(0, (-1, KEEP)).transpose(0, 1)  # noqa: E731
        again = _doubling(fold(start), fold(b)).transpose(0, 1).flatten(0, 1)[:T]
        again = torch.cat([before[:1], again[:-1]])
        again[keep] = before[keep]
        if packed:
            again[first] = h0[live]
        before = again
    # g_t = dh_t + a_{t+1} g_{t+1}, no factor over the end of a sequence
    ahead = torch.cat([a[1:], torch.zeros_like(a[:1])])
    gin = dh.clone()
    if packed:
        ahead[final] = 0
        gin[final] += dlast[live]
    else:
        gin[-1] += dlast
    g = _doubling(ahead.flip(0), gin.flip(0)).flip(0)
    dx = g * sq * si
    di = dx * x * (1 - si)
    # a^2 / s and z are both 0 in the limit of a closed gate, where s = 0
    slope = torch.where(sq > 0, a * a / sq, torch.zeros_like(sq))
    dz = g * (a * before - slope * si * x)
    dr = dz * z * (1 - sr)
    dp = torch.cat([dx, dr, di], -1)
    each = dz * (-RATE * sr)
    if mask is not None:
        dp = torch.where(mask.unsqueeze(-1), dp, torch.zeros_like(dp))
        each = each * mask.unsqueeze(-1)
    dd = each.flatten(0, -2).sum(0) * torch.sigmoid(decay)
    if packed:
        d0 = dlast.clone()
        d0[live] = a[first] * g[first]
    else:
        d0 = a[0] * g[0]
        h, dp = h.transpose(0, 1), dp.transpose(0, 1)
    dt = s["p"].dtype
    return {"h": h.to(dt), "last": last, "dp": dp.to(dt), "ddecay": dd, "dh0": d0}


def _run_step(s: dict):
    a, sq, _, _, si, x = _gates(s["p"].float(), s["decay"], None)
    state = s["state"]
    h = a * state[s["rows"]] + sq * si * x
    state[s["rows"]] = h
    return {"h": h.to(s["p"].dtype), "state": state}


def _run_norm(s: dict):
    c = s["case"]
    dt = s["x"].dtype
    x, u, g = (s[k].float() for k in ("x", "u", "gate"))
    wp, wn, sc = (s[k].float() for k in ("w_post", "w_pre", "scale"))

    def forward(x, u, g):
        ru = torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS)
        v = u * ru * wp
        sg = torch.sigmoid(g)
        y = x + sc * sg * v
        ry = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
        return ru, v, sg, y, ry

    ru, v, sg, y, ry = forward(x, u, g)
    out = {"y": y.to(dt), "n": (y * ry * wn).to(dt)}
    if not c["train"]:
        return out
    if c["checkpoint"]:
        x, u, g = _codes(x)[0], _codes(u)[0], _codes(g)[0]
        ru, v, sg, y, ry = forward(x, u, g)
    dy, dn = s["dy"].float(), s["dn"].float()
    yh = y * ry
    q = dn * wn
    dy = dy + ry * (q - yh * (q * yh).mean(-1, keepdim=True))
    dv = dy * sc * sg
    uh = u * ru
    t = dv * wp
    du = ru * (t - uh * (t * uh).mean(-1, keepdim=True))
    return {**out, "dx": dy.to(dt), "du": du.to(dt), "dgate": (dy * sc * v * sg * (1 - sg)).to(dt),
            "dw_post": (dv * uh).sum(0), "dw_pre": (dn * yh).sum(0), "dscale": (dy * sg * v).sum(0)}


def _run_pack(s: dict):
    x, scales = _codes(s["x"].float())
    return {"x": x.to(s["x"].dtype), "scales": scales}


@torch.no_grad()
def _run_plain(s: dict):
    return {"scan": _run_scan, "step": _run_step, "norm": _run_norm, "pack": _run_pack}[s["case"]["op"]](s)


def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    """Every input read once and every output written once; operations by the formulas, one for each
    addition, product, exponential, division or root."""
    e, H = _BYTES[case["dtype"]], case["width"]
    if case["op"] == "step":
        n = case["batch"] * H
        return {"bytes": n * (4 * e + 8) + 8 * case["batch"] + 4 * H, "flops": 17 * n}
    if case["op"] == "pack":  # the values in, the codes and scales out and in, the values out
        n, groups = case["rows"] * H, case["rows"] * -(-H // GROUP)
        return {"bytes": 2 * n * e + 2 * n + 8 * groups, "flops": 5 * n}
    if case["op"] == "norm":
        n = case["rows"] * H
        if not case["train"]:
            return {"bytes": 5 * n * e + 12 * H, "flops": 15 * n}
        return {"bytes": 10 * n * e + 24 * H, "flops": 50 * n}
    steps = case["steps"] * (1 if case["layout"] == "packed" else case["batch"])
    n = steps * H  # p and dh in, h and dp out
    return {"bytes": 8 * n * e + 16 * case["batch"] * H + (steps if case["mask"] else 0), "flops": 60 * n}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _walk(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """h_t = a_t h_{t-1} + b_t over dimension 0 from 0: blocks of steps walked side by side from 0, then
    each block's incoming state, in order, carried through the block."""
    T = a.size(0)
    L = max(1, math.isqrt(T))
    n = -(-T // L)
    pad = (0, 0) * (a.dim() - 1) + (0, n * L - T)
    a = torch.nn.functional.pad(a, pad, value=1.0).unflatten(0, (n, L))
    b = torch.nn.functional.pad(b, pad).unflatten(0, (n, L))
    h, f = torch.empty_like(b), torch.empty_like(b)
    ch, cf = torch.zeros_like(b[:, 0]), torch.ones_like(b[:, 0])
    for t in range(L):
        ch = a[:, t] * ch + b[:, t]
        cf = cf * a[:, t]
        h[:, t], f[:, t] = ch, cf
    carry = torch.zeros_like(b[0, 0])
    for k in range(n):
        h[k] += f[k] * carry
        carry = h[k, -1]
    return h.flatten(0, 1)[:T]


def _values64(x: torch.Tensor) -> torch.Tensor:
    """What the 8-bit codes of x stand for, group by group along the last dimension."""
    H = x.size(-1)
    out = torch.zeros_like(x)
    for lo in range(0, H, GROUP):
        part = x[..., lo:lo + GROUP]
        unit = part.abs().max(-1, keepdim=True).values / 127
        whole = unit > 0
        out[..., lo:lo + GROUP] = torch.where(whole, torch.round(part / torch.where(whole, unit, 1.0)) * unit, 0.0)
    return out


def _exact_scan(s: dict):
    c = s["case"]
    packed = c["layout"] == "packed"
    f64 = lambda t: t.detach().double()  # noqa: E731
    p, dh, h0, dlast = f64(s["p"]), f64(s["dh"]), f64(s["h0"]), f64(s["dlast"])
    mask = s["mask"]
    if not packed:
        p, dh = p.transpose(0, 1), dh.transpose(0, 1)
        mask = None if mask is None else mask.transpose(0, 1)
    if mask is not None:
        p = p.masked_fill(~mask.unsqueeze(-1), 0.0)
    T = p.size(0)
    first = torch.zeros(T, dtype=torch.bool, device=p.device)
    if packed:
        off = s["offsets"]
        live = (off[1:] > off[:-1]).nonzero().flatten()
        begin, end = off[live], off[live + 1] - 1
        first[begin] = True
    else:
        first[0] = True

    def one(p, decay, before):
        x, r, i = p.chunk(3, -1)
        log_a = -RATE * torch.log1p(torch.exp(decay)) / (1 + torch.exp(-r))
        if mask is not None:
            log_a = torch.where(mask.unsqueeze(-1), log_a, torch.zeros_like(log_a))
        a = torch.exp(log_a)
        add = torch.sqrt(torch.clamp_min(-torch.expm1(2 * log_a), 0)) / (1 + torch.exp(-i)) * x
        if mask is not None:
            add = torch.where(mask.unsqueeze(-1), add, torch.zeros_like(add))
        return a, a * before + add

    def states(a, add, heads):
        """State before each step, and after it; `heads`: steps whose incoming state is given there."""
        b, f = add.clone(), a.clone()
        at, given = heads
        b[at] += a[at] * given
        f[at] = 0
        after = _walk(f, b)
        before = torch.cat([torch.zeros_like(after[:1]), after[:-1]])
        before[at] = given
        return before, after

    decay = f64(s["decay"])
    zero = torch.zeros_like(p[..., : c["width"]])
    heads = (begin, h0[live]) if packed else (torch.zeros(1, dtype=torch.long, device=p.device), h0.unsqueeze(0))
    a, add = one(p, decay, zero)
    before, h = states(a, add, heads)
    last = h0.clone()
    if packed:
        last[live] = h[end]
    else:
        last = h[-1].clone()
    at = p
    if c["checkpoint"]:
        at = _values64(p.unflatten(-1, (3, -1))).flatten(-2)
        a, add = one(at, decay, zero)
        mark = first.clone()
        mark[::KEEP] = True
        where = mark.nonzero().flatten()
        before, _ = states(a, add, (where, before[where]))
    gin, f = dh.clone(), torch.zeros_like(a)
    f[:-1] = a[1:]
    if packed:
        gin[end] += dlast[live]
        f[end] = 0
    else:
        gin[-1] += dlast
    g = _walk(f.flip(0), gin.flip(0)).flip(0)
    del gin, f, add
    # one step's derivatives by autograd, at the state before it and with the gradient after it, in slices
    dp, each = torch.empty_like(p), torch.zeros_like(decay)
    d0 = torch.zeros_like(before)
    size = max(1, 40_000_000 // max(1, p[0].numel()))
    whole = mask
    for lo in range(0, T, size):
        part = slice(lo, min(T, lo + size))
        mask = None if whole is None else whole[part]
        leaves = [v.clone().requires_grad_() for v in (at[part], decay, before[part])]
        with torch.enable_grad():
            _, out = one(*leaves)
        a1, a2, a3 = torch.autograd.grad(out, leaves, g[part])
        dp[part], d0[part] = a1, a3
        each += a2
    if packed:
        dh0 = dlast.clone()
        dh0[live] = d0[begin]
    else:
        dh0 = d0[0].clone()
        h, dp = h.transpose(0, 1), dp.transpose(0, 1)
    return {"h": h, "last": last, "dp": dp, "ddecay": each, "dh0": dh0}


def _exact_norm(s: dict):
    c = s["case"]
    names = ("x", "u", "gate", "w_post", "w_pre", "scale")
    v = {k: s[k].detach().double() for k in names}

    def block(x, u, gate, w_post, w_pre, scale):
        y = x + scale / (1 + torch.exp(-gate)) * (u / torch.sqrt(u.pow(2).mean(-1, keepdim=True) + EPS) * w_post)
        return y, y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * w_pre

    y, n = block(*v.values())
    out = {"y": y, "n": n}
    if not c["train"]:
        return out
    if c["checkpoint"]:
        v |= {k: _values64(v[k]) for k in ("x", "u", "gate")}
    leaves = [t.requires_grad_() for t in v.values()]
    with torch.enable_grad():
        got = torch.autograd.grad(block(*leaves), leaves, (s["dy"].double(), s["dn"].double()))
    return {**out, **{"d" + k: t for k, t in zip(names, got)}}


@torch.no_grad()
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "scan":
        return _exact_scan(s)
    if case["op"] == "norm":
        return _exact_norm(s)
    if case["op"] == "step":
        x, r, i = s["p"].double().chunk(3, -1)
        log_a = -RATE * torch.log1p(torch.exp(s["decay"].double())) / (1 + torch.exp(-r))
        h = torch.exp(log_a) * s["state"].double()[s["rows"]]
        h = h + torch.sqrt(-torch.expm1(2 * log_a)) / (1 + torch.exp(-i)) * x
        return {"h": h, "state": s["state"].double().index_copy(0, s["rows"], h)}
    x = s["x"].double()
    unit = torch.nn.functional.pad(x, (0, -case["width"] % GROUP)).unflatten(-1, (-1, GROUP)).abs().amax(-1) / 127
    return {"x": _values64(x), "scales": unit}
