"""The gated recurrence, the norms around a block and 8-bit activations on CUDA against the
same formulas in 64 bits (the CPU forms, themselves checked against plain loops).

Tolerances. fp32: every step rounds a handful of times (2^-24 each, the exponential and the
reciprocal approximations 2^-22), and a state gathers the errors of its memory, at most a
few hundred steps at the decays used: their root sum square stays below 5e-6 of a result's
norm. bf16 results are rounded once, from 8 significant bits: by at most 2^-8 of each value
(and so of the norm), beside the fp32 bound. fp32 results of bf16 inputs keep the fp32 bound."""
import pytest
import torch

from starry_unigraph.ops.checkpoint8 import _dequantize_torch, _quantize_torch

pytestmark = pytest.mark.gpu
F32, BF16 = 5e-6, 2.0 ** -8 + 5e-6


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape
    assert torch.isfinite(a).all()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def bound(t):
    return BF16 if t.dtype == torch.bfloat16 else F32


def status_clear():
    from starry_unigraph.ops import check_status

    check_status()


def scan_inputs(B, T, H, dtype, layout, seed, masked=False, lens=None):
    g = torch.Generator().manual_seed(seed)
    lead = (sum(lens),) if lens is not None else ((T, B) if layout == "time" else (B, T))
    p = torch.randn(*lead, 3 * H, generator=g).to(dtype)
    dh = torch.randn(*lead, H, generator=g).to(dtype)
    decay = torch.randn(H, generator=g) - 3
    h0, dl = torch.randn(B, H, generator=g), torch.randn(B, H, generator=g)
    mask = None
    if masked:
        mask = torch.rand(*lead, generator=g) < 0.7
        if lens is None:
            mask[(slice(None), 0) if layout == "time" else 0] = False  # a sequence without a valid step
        p[~mask] = float("nan")
        p[..., 0][~mask] = float("inf")
    off = None if lens is None else torch.tensor([0] + list(lens)).cumsum(0)
    return p, dh, decay, h0, dl, mask, off


def run_scan(p, dh, decay, h0, dl, mask, off, layout, device, dtype=None, checkpoint=None):
    from starry_unigraph.ops.recurrence import gated_scan

    def put(t, d=dtype):
        return None if t is None else t.to(device=device, dtype=d if d is not None and t.is_floating_point() else None)

    p, dh, decay, h0, dl, mask, off = (put(t) for t in (p, dh, decay, h0, dl, mask, off))
    leaves = [p.requires_grad_(), decay.requires_grad_(), h0.requires_grad_()]
    flip = (lambda t: t.transpose(0, 1)) if layout == "time" and off is None else (lambda t: t)
    h, last = gated_scan(flip(p), decay, h0, mask=None if mask is None else flip(mask), offsets=off,
                         checkpoint=checkpoint)
    grads = torch.autograd.grad((h, last), leaves, (flip(dh), dl))
    return [flip(h), last, *grads]


SIZES = [(1, 1, 1), (3, 2, 4), (2, 4, 8), (5, 7, 12), (300, 8, 64), (2, 15, 33), (2, 16, 32), (2, 17, 31), (4, 33, 100),
         (1, 130, 65), (3, 129, 64), (2, 1000, 20), (1, 3000, 5), (70, 40, 300), (1, 700, 1100)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["time", "batch"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,T,H", SIZES)
def test_scan(B, T, H, masked, layout, dtype):
    x = scan_inputs(B, T, H, dtype, layout, B + T + H, masked)
    got = run_scan(*x, layout, "cuda")
    want = run_scan(*x, layout, "cpu", torch.float64)
    for a, b in zip(got, want):
        assert rel(a, b) < bound(a)
    status_clear()


LENS = [[1], [0, 0, 3, 0], [5, 0, 1, 1, 1, 40, 0, 16, 16, 0], [300, 1, 0, 2, 129], [0, 2000, 0], [1] * 70 + [64, 0, 128],
        [3, 700, 31, 1, 0, 0, 0, 0, 257]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("H", [3, 32, 100])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_scan_packed(lens, H, masked, dtype):
    x = scan_inputs(len(lens), None, H, dtype, "batch", sum(lens) + H, masked, lens)
    got = run_scan(*x, "batch", "cuda")
    want = run_scan(*x, "batch", "cpu", torch.float64)
    for a, b in zip(got, want):
        assert rel(a, b) < bound(a)
    status_clear()


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("H", [6, 33, 64])
@pytest.mark.parametrize("lens", [[32] * 9, [31, 1, 64, 33, 0, 31, 96, 1, 31], [1, 200, 32, 1, 1, 30, 160, 31]], ids=str)
def test_scan_packed_at_segment_edges(lens, H, masked):
    """Sequences that start, end, start one row early and end one row late where segments of 32 steps do."""
    x = scan_inputs(len(lens), None, H, torch.float32, "batch", sum(lens) + H, masked, lens)
    got = run_scan(*x, "batch", "cuda")
    want = run_scan(*x, "batch", "cpu", torch.float64)
    for a, b in zip(got, want):
        assert rel(a, b) < bound(a)
    status_clear()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,T,H", [(3, 1, 5), (40, 4, 64), (9, 8, 128), (2, 16, 33), (3, 50, 100), (2, 300, 64), (1, 400, 30)])
def test_scan_int8(B, T, H, masked, dtype):
    """The CPU form in fp32 takes the same codes bit for bit."""
    for layout, lens in (("time", None), ("batch", None), ("batch", [T] * (B - 1) + [0] + [T])):
        x = scan_inputs(B if lens is None else len(lens), T, H, dtype, layout, T + H, masked, lens)
        got = run_scan(*x, layout, "cuda", checkpoint="int8")
        want = run_scan(*x, layout, "cpu", checkpoint="int8")
        for a, b in zip(got, want):
            # two fp32 (or bf16) results: the bound of each
            assert rel(a, b) < 2 * bound(a)


def test_scan_strides_and_slices():
    """p as a slice of a wider projection, rows on odd addresses, a reversed-order batch, broadcast gradients."""
    from starry_unigraph.ops.recurrence import gated_scan

    torch.manual_seed(0)
    B, T, H = 4, 37, 20
    wide = torch.randn(B, T, 3 * H + 7, device="cuda")
    decay = torch.randn(H, device="cuda")
    for off in (0, 1, 4, 7):
        p = wide[..., off:off + 3 * H].requires_grad_()
        h, last = gated_scan(p, decay)
        ref, rlast = gated_scan(p.detach().double().cpu(), decay.double().cpu())
        assert rel(h, ref) < F32 and rel(last, rlast) < F32
        g, = torch.autograd.grad(h.sum(), p)  # the gradient of h is expanded from one value
        q = p.detach().double().cpu().requires_grad_()
        want, = torch.autograd.grad(gated_scan(q, decay.double().cpu())[0].sum(), q)
        assert rel(g, want) < F32
    every = wide[:, :, : 3 * H].permute(2, 0, 1).contiguous().permute(1, 2, 0)  # channels outermost in memory
    assert rel(gated_scan(every, decay)[0], gated_scan(wide[..., : 3 * H].double().cpu(), decay.double().cpu())[0]) < F32


def test_scan_one_output_used_and_repeatable():
    from starry_unigraph.ops.recurrence import gated_scan

    torch.manual_seed(1)
    p = torch.randn(3, 500, 96, device="cuda", requires_grad=True)
    d = torch.randn(32, device="cuda", requires_grad=True)
    g0 = torch.autograd.grad(gated_scan(p, d)[1].square().sum(), (p, d))
    q, e = p.detach().double().cpu().requires_grad_(), d.detach().double().cpu().requires_grad_()
    want = torch.autograd.grad(gated_scan(q, e)[1].square().sum(), (q, e))
    for a, b in zip(g0, want):
        assert rel(a, b) < F32
    for _ in range(3):  # the same bits every time
        again = torch.autograd.grad(gated_scan(p, d)[1].square().sum(), (p, d))
        assert all(torch.equal(a, b) for a, b in zip(g0, again))


def test_scan_extremes():
    """Decays near 1 over a long memory, gates far open and closed; values in 64 bits."""
    from starry_unigraph.ops.recurrence import gated_scan

    torch.manual_seed(2)
    p = torch.randn(2, 4000, 24)
    p[..., 8:16] *= 30
    p[0, :, 8:16] = -200.0  # never decays, takes nothing in
    decay = torch.linspace(-9, 4, 8)
    h0 = torch.randn(2, 8)
    x, d, s = p.cuda().requires_grad_(), decay.cuda().requires_grad_(), h0.cuda().requires_grad_()
    h, last = gated_scan(x, d, s)
    assert torch.equal(h[0].detach(), h0[0].cuda().expand(4000, 8))
    g = torch.autograd.grad(h.sum(), (x, d, s))
    assert all(torch.isfinite(t).all() for t in g)
    X, D, S = (t.double().requires_grad_() for t in (p, decay, h0))
    H, L = gated_scan(X, D, S)
    # memories of up to 1 / (8 softplus(-9)) = 1000 steps and beyond: 1000 roundings of 2^-24 side by side
    assert rel(h, H) < 2e-5 and rel(last, L) < 2e-5
    for a, b in zip(g, torch.autograd.grad(H.sum(), (X, D, S))):
        assert rel(a, b) < 5e-5


def test_scan_bad_offsets_are_reported():
    from starry_unigraph.ops import check_status
    from starry_unigraph.ops.recurrence import gated_scan

    status_clear()
    p, d = torch.randn(10, 12, device="cuda"), torch.randn(4, device="cuda")
    for off in ([0, 4, 11], [0, 6, 3, 10], [0, -2, 10]):
        gated_scan(p, d, offsets=torch.tensor(off, device="cuda"))
        with pytest.raises(RuntimeError, match="index out of range"):
            check_status()
    status_clear()


def test_scan_refuses_on_cuda():
    from starry_unigraph.ops.recurrence import gated_scan, gated_scan_step

    p, d = torch.randn(2, 3, 12, device="cuda"), torch.randn(4, device="cuda")
    t = torch.zeros(5, 4, device="cuda")
    for bad in (lambda: gated_scan(p.half(), d), lambda: gated_scan(p, d.cpu()), lambda: gated_scan(p, d.double()),
                lambda: gated_scan(p[0], d, offsets=torch.tensor([0, 3])), lambda: gated_scan(p, d, torch.zeros(2, 4)),
                lambda: gated_scan(p[0], d, offsets=torch.tensor([0, 3], device="cuda", dtype=torch.int32)),
                lambda: gated_scan_step(p[0], d, t), lambda: gated_scan_step(p[0], d, t.double()[:3]),
                lambda: gated_scan_step(p[0], d, t[:1].expand(3, 4)),
                lambda: gated_scan_step(p[0], d, t, torch.tensor([0, 1, 2]))):
        with pytest.raises((RuntimeError, ValueError)):
            bad()


def test_scan_of_nothing_on_cuda():
    from starry_unigraph.ops.recurrence import gated_scan

    d = torch.randn(2, device="cuda", requires_grad=True)
    h0 = torch.ones(3, 2, device="cuda", requires_grad=True)
    for keep in (None, "int8"):
        h, last = gated_scan(torch.randn(3, 0, 6, device="cuda"), d, h0, checkpoint=keep)
        assert h.shape == (3, 0, 2) and torch.equal(last, h0)
        gd, gh = torch.autograd.grad(last.sum(), (d, h0))
        assert torch.equal(gd, torch.zeros_like(gd)) and torch.equal(gh, torch.ones_like(gh))
        h, last = gated_scan(torch.randn(0, 5, 6, device="cuda"), d, checkpoint=keep)
        assert h.shape == (0, 5, 2) and last.shape == (0, 2)
        gd, = torch.autograd.grad(h.sum(), d)
        assert torch.equal(gd, torch.zeros_like(gd))
        off = torch.zeros(4, dtype=torch.long, device="cuda")
        h, last = gated_scan(torch.randn(0, 6, device="cuda"), d, h0, offsets=off, checkpoint=keep)
        assert h.shape == (0, 2) and torch.equal(last, h0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,H", [(1, 1), (600, 100), (37, 65), (1000, 128), (3, 700)])
def test_step(n, H, dtype):
    from starry_unigraph.ops.recurrence import gated_scan_step

    torch.manual_seed(n + H)
    p, decay, table = torch.randn(n, 3 * H).to(dtype), torch.randn(H), torch.randn(2 * n + 1, H)
    rows = torch.randperm(2 * n + 1)[:n]
    ref = table.double()
    want = gated_scan_step(p.double(), decay.double(), ref, rows)
    got = table.cuda()
    h = gated_scan_step(p.cuda(), decay.cuda(), got, rows.cuda())
    assert h.dtype == dtype and rel(h, want) < bound(h) and rel(got, ref) < F32
    wide = torch.randn(n, 3 * H + 5).to(dtype).cuda()  # strided rows of p and of the table, no index
    tab = torch.randn(n, H + 3).cuda()
    keep = tab.clone()
    h = gated_scan_step(wide[:, 2:2 + 3 * H], decay.cuda(), tab[:, 1:1 + H])
    ref = keep[:, 1:1 + H].double().cpu()
    want = gated_scan_step(wide[:, 2:2 + 3 * H].double().cpu(), decay.double(), ref)
    assert rel(h, want) < bound(h) and rel(tab[:, 1:1 + H], ref) < F32
    assert torch.equal(tab[:, 0], keep[:, 0]) and torch.equal(tab[:, 1 + H:], keep[:, 1 + H:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [128, 130, 132])
def test_step_of_many_rows(H, dtype):
    """More rows than fill the device: groups of channels a thread where the table's and p's rows allow."""
    from starry_unigraph.ops.recurrence import gated_scan_step

    torch.manual_seed(H)
    n = 5003
    p, decay, table = torch.randn(n, 3 * H + 4).to(dtype), torch.randn(H), torch.randn(2 * n, H + 4)
    rows = torch.randperm(2 * n)[:n]
    rows[7] = 2 * n  # outside the table
    for shift in (0, 1, 4):
        q, ref = p[:, shift:shift + 3 * H], table[:, shift:shift + H].double()
        keep = torch.arange(n) != 7
        want = gated_scan_step(q.double()[keep], decay.double(), ref, rows[keep])
        got = table.cuda()
        h = gated_scan_step(p.cuda()[:, shift:shift + 3 * H], decay.cuda(), got[:, shift:shift + H], rows.cuda())
        assert rel(h[keep.cuda()], want) < bound(h) and rel(got[:, shift:shift + H], ref) < F32
        assert h[7].abs().max() == 0 and torch.equal(got[:, shift + H:].cpu(), table[:, shift + H:])
        assert torch.equal(got[:, :shift].cpu(), table[:, :shift])
        with pytest.raises(RuntimeError, match="index out of range"):
            status_clear()


def test_step_reports_places_outside_the_table():
    from starry_unigraph.ops import check_status
    from starry_unigraph.ops.recurrence import gated_scan_step

    status_clear()
    p, d, table = torch.randn(3, 12, device="cuda"), torch.randn(4, device="cuda"), torch.ones(5, 4, device="cuda")
    h = gated_scan_step(p, d, table, torch.tensor([1, 5, -1], device="cuda"))
    with pytest.raises(RuntimeError, match="index out of range"):
        check_status()
    assert torch.equal(h[1:], torch.zeros_like(h[1:]))
    assert torch.equal(table[[0, 2, 3, 4]], torch.ones(4, 4, device="cuda"))


def norm_inputs(rows, H, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, u, gate, dy, dn = (r(rows, H).to(dtype) for _ in range(5))
    if rows > 2:
        u[1] = 0  # a block that puts out nothing
    return x, u, gate, dy, dn, r(H), r(H), r(H)


def run_norm(inp, device, dtype=None, checkpoint=None, parts="ugpns", vec=None):
    """parts: which of u, gate, w_post, n (w_pre) and scale take part."""
    from starry_unigraph.ops.norm import norm_residual, rms_norm

    x, u, gate, dy, dn, wp, wn, sc = (t.to(device=device, dtype=dtype) for t in inp)
    if vec is not None:
        wp, wn, sc = (t.to(vec) for t in (wp, wn, sc))
    leaves = {"x": x, "u": u, "g": gate, "p": wp, "n": wn, "s": sc}
    leaves = {k: v.requires_grad_() for k, v in leaves.items() if k == "x" or k in parts}
    # the norm of a single value is its sign but for eps: with a small eps the gradient is a
    # difference of equal numbers in any arithmetic
    eps = 0.5 if x.size(1) == 1 else 1e-6
    if "u" in parts:
        out = norm_residual(x, u, leaves.get("p"), leaves.get("n"), gate=leaves.get("g"), scale=leaves.get("s"),
                            eps=eps, checkpoint=checkpoint)
    else:
        out = (rms_norm(x, wn, eps=eps, checkpoint=checkpoint),)
        dy = dn
    pairs = [(o, g) for o, g in zip(out, (dy, dn)) if o is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs])
    return [o for o, _ in pairs] + list(grads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,H", [(1, 1), (5, 3), (700, 64), (33, 100), (9, 172), (4, 257), (100, 512), (3, 1000),
                                    (3, 1001), (700, 2048), (2, 2049), (2, 5000), (2, 8192), (2, 9001), (2, 16383),
                                    (2, 16384)])
def test_norm(rows, H, dtype):
    inp = norm_inputs(rows, H, dtype, rows + H)
    for a, b in zip(run_norm(inp, "cuda"), run_norm(inp, "cpu", torch.float64)):
        assert rel(a, b) < bound(a)
    if dtype == torch.bfloat16:  # fp32 vectors beside bf16 rows, their gradients in fp32
        got = run_norm(inp, "cuda", vec=torch.float32)
        want = run_norm(inp, "cpu", torch.float64)
        for a, b in zip(got, want):
            assert rel(a, b) < bound(a)


@pytest.mark.parametrize("parts", ["ugpn", "upns", "ugns", "ugps", "un", "u", "n", "ug"])
@pytest.mark.parametrize("rows,H", [(50, 64), (3, 65), (3, 3000)])
def test_norm_parts(rows, H, parts):
    inp = norm_inputs(rows, H, torch.float32, H)
    for keep in (None, "int8"):
        got = run_norm(inp, "cuda", parts=parts, checkpoint=keep)
        # int8: the CPU form in fp32 takes the same codes bit for bit
        want = run_norm(inp, "cpu", torch.float64 if keep is None else None, parts=parts, checkpoint=keep)
        for a, b in zip(got, want):
            assert rel(a, b) < F32 * (1 if keep is None else 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,H", [(1, 1), (700, 64), (33, 100), (9, 172), (4, 257), (3, 1001), (60, 2048), (2, 9001)])
def test_norm_int8(rows, H, dtype):
    inp = norm_inputs(rows, H, dtype, rows + H)
    for a, b in zip(run_norm(inp, "cuda", checkpoint="int8"), run_norm(inp, "cpu", checkpoint="int8")):
        assert rel(a, b) < 2 * bound(a)


def test_norm_strides_and_one_output():
    from starry_unigraph.ops.norm import norm_residual

    torch.manual_seed(3)
    wide = torch.randn(40, 3, 70, device="cuda")
    w = torch.randn(64, device="cuda")
    for off in (0, 1, 4):
        x, u, g = (wide[:, k, off:off + 64] for k in range(3))
        ref = norm_residual(*(t.double().cpu() for t in (x, u)), w.double().cpu(), w.double().cpu(),
                            gate=g.double().cpu())
        out = norm_residual(x, u, w, w, gate=g)
        assert all(rel(a, b) < F32 for a, b in zip(out, ref))
    x = wide[..., :64].clone().requires_grad_()  # three dimensions, a gradient expanded from one value
    X = x.detach().double().cpu().requires_grad_()
    for pick in (0, 1):
        got, = torch.autograd.grad(norm_residual(x, x, w, w)[pick].sum(), x)
        want, = torch.autograd.grad(norm_residual(X, X, w.double().cpu(), w.double().cpu())[pick].sum(), X)
        assert rel(got, want) < F32


def test_norm_refuses_on_cuda():
    from starry_unigraph.ops.norm import norm_residual, rms_norm

    x, w = torch.randn(3, 8, device="cuda"), torch.randn(8, device="cuda")
    for bad in (lambda: norm_residual(x, x.cpu(), w), lambda: norm_residual(x.half(), x.half(), w),
                lambda: norm_residual(x, x, w.cpu()), lambda: norm_residual(x, x, w.double()),
                lambda: rms_norm(torch.randn(1, 16385, device="cuda"), torch.randn(16385, device="cuda"))):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    y, n = norm_residual(x[:0], x[:0], w, w)
    assert y.shape == n.shape == (0, 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (5, 31), (1000, 64), (7, 100), (3, 4, 172), (2, 4097), (100, 32)])
def test_codes_equal_the_plain_ones(shape, dtype):
    from starry_unigraph.ops.checkpoint8 import quantize8

    torch.manual_seed(sum(shape))
    x = (torch.randn(*shape) * torch.exp(4 * torch.randn(*shape[:-1], 1))).to(dtype)
    x.view(-1, shape[-1])[-1, -1] = 0
    for bad in (None, float("nan"), float("inf"), 1e-38):
        if bad is not None:
            x.view(-1, shape[-1])[0, 0] = bad
        if bad == 1e-38:
            x.view(-1, shape[-1])[0] = bad
        q = quantize8(x.cuda())
        rows = x.reshape(-1, shape[-1])
        codes, scales = _quantize_torch(rows)
        assert torch.equal(q.codes.cpu(), codes)
        assert torch.equal(q.scales.cpu().nan_to_num(nan=-1.0), scales.nan_to_num(nan=-1.0))
        back = q.dequantize().cpu()
        want = _dequantize_torch(codes, scales, dtype).view(shape)
        assert back.dtype == dtype and torch.equal(back.nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))
        assert q.dequantize(torch.float32).dtype == torch.float32
    wide = torch.randn(6, shape[-1] + 3).to(dtype).cuda()
    part = wide[:, 1:1 + shape[-1]]
    assert torch.equal(quantize8(part).codes.cpu(), _quantize_torch(part.cpu())[0])


def test_rows_beyond_32_bits():
    """Element offsets past 2^31: the last rows of a large call equal the same rows alone."""
    from starry_unigraph.ops.checkpoint8 import quantize8
    from starry_unigraph.ops.norm import norm_residual
    from starry_unigraph.ops.recurrence import gated_scan

    H, T = 32, 4
    B = (1 << 31) // (3 * H * T) + 1001  # p holds more than 2^31 values
    g = torch.Generator(device="cuda").manual_seed(0)
    p = torch.randn(T, B, 3 * H, device="cuda", generator=g, dtype=torch.bfloat16)
    d = torch.randn(H, device="cuda")
    view = p.transpose(0, 1).requires_grad_()
    for keep in (None, "int8"):
        h, last = gated_scan(view, d, checkpoint=keep)
        dp, = torch.autograd.grad(last.sum() + h.sum(), view)
        tail = view.detach()[-500:].clone().requires_grad_()
        ht, lt = gated_scan(tail, d, checkpoint=keep)
        dt, = torch.autograd.grad(lt.sum() + ht.sum(), tail)
        assert torch.equal(h[-500:], ht) and torch.equal(last[-500:], lt) and torch.equal(dp[-500:], dt)
        del h, last, dp
    off = torch.tensor([0, T * B - 3000, T * B], device="cuda")
    flat = p.detach().view(-1, 3 * H)
    h, last = gated_scan(flat, d, offsets=off)
    ht, lt = gated_scan(flat[-3000:], d, offsets=torch.tensor([0, 3000], device="cuda"))
    # chunks of the packed axis fall elsewhere: equal up to rounding
    assert rel(h[-3000:], ht) < BF16 and rel(last[1:], lt) < F32
    del h, last
    rows = p.detach().view(-1, H)
    w = torch.randn(H, device="cuda")
    for keep in (None, "int8"):
        x = rows.requires_grad_()
        y, n = norm_residual(x, x, w, w, gate=x, checkpoint=keep)
        dx, = torch.autograd.grad(n, x, y.detach())
        t = rows.detach()[-700:].clone().requires_grad_()
        yt, nt = norm_residual(t, t, w, w, gate=t, checkpoint=keep)
        dt, = torch.autograd.grad(nt, t, yt.detach())
        assert torch.equal(y[-700:], yt) and torch.equal(n[-700:], nt) and torch.equal(dx[-700:], dt)
        del x, y, n, dx
    q = quantize8(rows.detach())
    assert torch.equal(q.codes[-900:], quantize8(rows.detach()[-900:]).codes)
    assert torch.equal(q.dequantize()[-900:], quantize8(rows.detach()[-900:]).dequantize())


def test_other_streams_and_graphs():
    """Calls follow the current stream; a captured call replays on new inputs."""
    from starry_unigraph.ops.norm import norm_residual
    from starry_unigraph.ops.recurrence import gated_scan, gated_scan_step

    torch.manual_seed(5)
    p, d = torch.randn(2, 900, 96, device="cuda"), torch.randn(32, device="cuda")
    x, w = torch.randn(500, 32, device="cuda"), torch.randn(32, device="cuda")
    table = torch.randn(500, 32, device="cuda")
    start = table.clone()
    tok = torch.randn(500, 96, device="cuda")
    want = gated_scan(p, d)[0], norm_residual(x, x, w, w)[1], gated_scan_step(tok, d, table.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gated_scan(p, d)[0], norm_residual(x, x, w, w)[1], gated_scan_step(tok, d, table)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    def both(p, x):
        q, t = p.requires_grad_(), x.requires_grad_()
        h, last = gated_scan(q, d, checkpoint="int8")
        y, n = norm_residual(t, t, w, w)
        return (h, n, *torch.autograd.grad(h.sum() + last.sum() + n.square().sum() + y.sum(), (q, t)))

    ps, xs = p.clone(), x.clone()
    both(ps, xs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(ps, xs)
    for seed in (6, 7):
        torch.manual_seed(seed)
        new_p, new_x = torch.randn_like(p), torch.randn_like(x)
        with torch.no_grad():
            ps.copy_(new_p)
            xs.copy_(new_x)
        graph.replay()
        ref = both(new_p.clone(), new_x.clone())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref))
    assert torch.equal(start[:0], table[:0])


def test_saved8_on_cuda():
    """The framework's linear inside saved8: weight gradients of the packed input; a scan that
    keeps codes already is not packed twice."""
    from starry_unigraph.ops.checkpoint8 import quantize8, saved8
    from starry_unigraph.ops.dtdg import linear
    from starry_unigraph.ops.recurrence import gated_scan

    torch.manual_seed(8)
    x, w = torch.randn(2000, 64, device="cuda"), torch.randn(96, 64, device="cuda", requires_grad=True)
    with saved8(min_numel=1):
        y = linear(x * 1.0, w)
    g = torch.randn_like(y)
    gw, = torch.autograd.grad(y, w, g)
    want, = torch.autograd.grad(linear(quantize8(x).dequantize(), w), w, g)
    torch.testing.assert_close(gw, want, rtol=1e-4, atol=1e-3)  # split sums meet in any order
    p, d = torch.randn(4, 100, 96, device="cuda", requires_grad=True), torch.randn(32, device="cuda")
    a, = torch.autograd.grad(gated_scan(p * 1.0, d, checkpoint="int8")[0].sum(), p)
    with saved8(min_numel=1):
        h = gated_scan(p * 1.0, d, checkpoint="int8")[0]
    b, = torch.autograd.grad(h.sum(), p)
    assert torch.equal(a, b)


def test_stack_on_cuda():
    """The blocks against their CPU form; the linear layers' tensor cores read tf32 operands (2^-11
    each), which two layers and their gradients pass on."""
    import copy

    from starry_unigraph.lib_stable import GatedRecurrentStack
    from starry_unigraph.ops import gemm_precision

    torch.manual_seed(9)
    m = GatedRecurrentStack(64, num_layers=2)
    x = torch.randn(20, 30, 64)
    mask = torch.rand(20, 30) < 0.8
    mask[:, 3] = False
    x[~mask] = float("nan")
    c = copy.deepcopy(m).cuda()
    n, last = m(x, mask=mask)
    (n * n.detach().cos()).sum().backward()
    with gemm_precision(True):
        cn, clast = c(x.cuda(), mask=mask.cuda())
        (cn * n.detach().cos().cuda()).sum().backward()
    assert rel(cn, n) < 5e-3 and all(rel(a, b) < 5e-3 for a, b in zip(clast, last))
    for (k, a), b in zip(c.named_parameters(), m.parameters()):
        if b.grad.norm() > 1e-6:
            assert rel(a.grad, b.grad) < 2e-2, k
    state = c.init_state(40)
    rows = torch.randperm(40, device="cuda")[:30]
    y = torch.randn(20, 30, 64, device="cuda")
    with gemm_precision(True), torch.no_grad():
        whole, end = c(y)
        for t in range(20):
            out = c.step(y[t], state, rows)
            assert rel(out, whole[t]) < 5e-3
    assert all(rel(s[rows], e) < 5e-3 for s, e in zip(state, end))


def test_example_on_cuda(tmp_path, monkeypatch):
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "train_gated_recurrence.py"
    spec = importlib.util.spec_from_file_location("train_gated_recurrence", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    monkeypatch.chdir(tmp_path)
    res = {}
    for keep in ("none", "int8"):
        res[keep] = ex.main(["--nodes", "3000", "--edges", "30000", "--snapshots", "20", "--epochs", "3", "--device", "cuda",
                             "--checkpoint", keep, "--artifact-root", str(tmp_path / keep)])
        assert res[keep]["train"][-1] < res[keep]["train"][0]
    assert abs(res["int8"]["train"][-1] - res["none"]["train"][-1]) < 0.02 * res["none"]["train"][-1]


def test_more_refusals_on_cuda():
    """Shapes, devices and types that the calls refuse, each before anything is launched."""
    from starry_unigraph.ops.checkpoint8 import quantize8
    from starry_unigraph.ops.norm import norm_residual, rms_norm
    from starry_unigraph.ops.recurrence import gated_scan, gated_scan_step

    p, d = torch.randn(2, 3, 12, device="cuda"), torch.randn(4, device="cuda")
    m = torch.ones(2, 3, dtype=torch.bool, device="cuda")
    off = torch.tensor([0, 1, 3], device="cuda")
    x, w = torch.randn(3, 8, device="cuda"), torch.randn(8, device="cuda")
    t = torch.zeros(5, 4, device="cuda")
    for bad in (lambda: gated_scan(p[..., :11], d), lambda: gated_scan(p, d[:3]), lambda: gated_scan(p, torch.stack([d, d])),
                lambda: gated_scan(p, d, torch.zeros(3, 4, device="cuda")), lambda: gated_scan(p, d, mask=m.t()),
                lambda: gated_scan(p, d, mask=m.float()), lambda: gated_scan(p, d, mask=m.cpu()),
                lambda: gated_scan(p, d, offsets=off), lambda: gated_scan(p[0], d), lambda: gated_scan(p, d, rate=-1.0),
                lambda: gated_scan(p, d, rate=float("inf")), lambda: gated_scan(p, d, checkpoint="int4"),
                lambda: gated_scan(p[0], d, torch.zeros(3, 4, device="cuda"), offsets=off),
                lambda: gated_scan(torch.randn(1, 1, 3 << 19, device="cuda"), torch.randn(1 << 19, device="cuda")),
                lambda: gated_scan_step(p[0, :, :11], d, t), lambda: gated_scan_step(p[0].half(), d, t[:3]),
                lambda: gated_scan_step(p[0], d, t[:3], rate=0.0), lambda: gated_scan_step(p[0], d, t.t()[:3]),
                lambda: norm_residual(x, x[:2], w), lambda: norm_residual(x, x, w[:7]), lambda: norm_residual(x, x.bfloat16(), w),
                lambda: norm_residual(x, x, w, eps=0.0), lambda: norm_residual(x, x, w, gate=x[:, :4]),
                lambda: norm_residual(x, x, w, scale=torch.ones(8)), lambda: rms_norm(x[:, :0], w[:0]),
                lambda: norm_residual(x, x, w, checkpoint="fp8"), lambda: quantize8(x.half()), lambda: quantize8(x[:, :0]),
                lambda: quantize8(torch.tensor(1.0, device="cuda")), lambda: quantize8(x).dequantize(torch.float16)):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    status_clear()


def test_gradients_are_not_differentiated_again():
    from starry_unigraph.ops.norm import norm_residual
    from starry_unigraph.ops.recurrence import gated_scan

    p, d = torch.randn(2, 3, 12, device="cuda", requires_grad=True), torch.randn(4, device="cuda")
    x, w = torch.randn(3, 8, device="cuda", requires_grad=True), torch.randn(8, device="cuda")
    for out, leaf in ((gated_scan(p, d)[0], p), (norm_residual(x, x, w)[0], x)):
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(out.sum(), leaf, create_graph=True)
    out = gated_scan(p, d)[0]
    a, = torch.autograd.grad(out.sum(), p, retain_graph=True)
    b, = torch.autograd.grad(out.sum(), p)  # the same graph again
    assert torch.equal(a, b)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_scan_gradient_against_differences_on_cuda(checkpoint):
    """Directional derivatives of the forward kernel alone: central differences with a step of 2^-6,
    whose error is h^2 / 6 of the third derivative (below 2e-4 of the gradient here) plus the
    rounding of fp32 sums over the step (1e-4); with 8-bit inputs the gradient is that at values up
    to half a scale off (amax / 254, near 1 %)."""
    from starry_unigraph.ops.recurrence import gated_scan

    torch.manual_seed(11)
    B, T, H = 3, 40, 64
    p, d, h0 = (torch.randn(*s, device="cuda") for s in ((B, T, 3 * H), (H,), (B, H)))
    gh, gl = torch.randn(B, T, H, device="cuda"), torch.randn(B, H, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (p, d, h0)]
    h, last = gated_scan(*leaves, checkpoint=checkpoint)
    grads = torch.autograd.grad((h, last), leaves, (gh, gl))

    def f(*a):
        h, last = gated_scan(*a)
        return float((h.double() * gh).sum() + (last.double() * gl).sum())

    for k in range(3):
        u = [torch.zeros_like(t) for t in (p, d, h0)]
        # along the gradient: the derivative is its norm, nothing cancels
        u[k] = grads[k] / grads[k].norm()
        e = 2.0 ** -6
        got = (f(*[t + e * v for t, v in zip((p, d, h0), u)]) - f(*[t - e * v for t, v in zip((p, d, h0), u)])) / (2 * e)
        want = float(grads[k].double().norm())
        assert abs(got - want) < (2e-3 if checkpoint is None else 2e-2) * want


@pytest.mark.parametrize("steps", [9, 31, 65, 200])
@pytest.mark.parametrize("batch,H", [(1, 64), (1, 2048), (40, 300), (700, 129)])
def test_scan_split_and_whole_agree(batch, H, steps):
    """Few sequences are cut into segments, many are walked whole: the first of many equal the few
    up to rounding, as 1, `batch` and many times `batch` sequences."""
    from starry_unigraph.ops.recurrence import gated_scan

    g = torch.Generator(device="cuda").manual_seed(steps)
    many = batch * max(1, 200_000 // (batch * H))
    p = torch.randn(many, steps, 3 * H, device="cuda", generator=g)
    d, gh = torch.randn(H, device="cuda", generator=g) - 3, torch.randn(many, steps, H, device="cuda", generator=g)

    def run(n):
        q = p[:n].clone().requires_grad_()
        h, last = gated_scan(q, d)
        return h, last, torch.autograd.grad((h, last), q, (gh[:n], gh[:n, 0]))[0]

    whole = run(many)
    for n in (1, batch):
        for a, b in zip(run(n), whole):
            assert rel(a, b[:n]) < 2 * F32  # two fp32 results


def test_codes_of_very_long_rows():
    from starry_unigraph.ops.checkpoint8 import quantize8

    x = torch.randn((1 << 25) + 35, device="cuda")
    q = quantize8(x)
    whole = quantize8(x[: 1 << 25].view(-1, 4096))
    assert torch.equal(q.codes[0, : 1 << 25], whole.codes.view(-1))
    assert torch.equal(q.dequantize()[-35:], quantize8(x[-35:]).dequantize())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [1, 2, 3, 5, 6, 8, 10, 12, 17, 20, 26, 30, 34, 38])
def test_narrow_and_even_widths(H, dtype):
    """Rows narrower than a group of codes, and widths that are even but no multiple of four."""
    for B, T, lens in ((3, 3, None), (4, 7, None), (2, 90, None), (3, 0, [50, 0, 41])):
        for masked in (False, True):
            x = scan_inputs(B, T, H, dtype, "batch", B + T + H, masked, lens)
            got, want = run_scan(*x, "batch", "cuda"), run_scan(*x, "batch", "cpu", torch.float64)
            for k, (a, b) in enumerate(zip(got, want)):
                assert rel(a, b) < bound(a) * (4 if k == 3 else 1)  # ddecay: one sum a channel, whose terms may cancel
            got = run_scan(*x, "batch", "cuda", checkpoint="int8")
            for k, (a, b) in enumerate(zip(got, run_scan(*x, "batch", "cpu", checkpoint="int8"))):
                assert rel(a, b) < 2 * bound(a) * (4 if k == 3 else 1)
    for rows in (5, 5000):
        inp = norm_inputs(rows, H, dtype, rows + H)
        for a, b in zip(run_norm(inp, "cuda"), run_norm(inp, "cpu", torch.float64)):
            assert rel(a, b) < bound(a)
        for a, b in zip(run_norm(inp, "cuda", checkpoint="int8"), run_norm(inp, "cpu", checkpoint="int8")):
            assert rel(a, b) < 2 * bound(a)
