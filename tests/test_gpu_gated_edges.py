"""Edges of the gated recurrence, the norms around a block and 8-bit activations on CUDA: what a
call does with rows of the largest width, with values that are not finite, with outside
writes to its tensors and with arguments that it has to refuse."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = 5e-6  # relative, fp32 results against 64 bits: derived in test_gpu_gated.py


@pytest.mark.parametrize("H", [(1 << 31) - 1, (1 << 31) - 4, (1 << 31) - 40])
def test_codes_of_the_longest_rows(H):
    """Up to 2^31 - 1 values a row, the last group partly filled: both ends equal the same values alone."""
    from starry_unigraph.ops.checkpoint8 import Packed8, quantize8

    x = torch.randn(1 << 24, device="cuda", dtype=torch.bfloat16).repeat(1 << 7)[:H]
    q = quantize8(x)
    tail = H % 32
    want = quantize8(x[-tail:])
    assert q.codes.shape == (1, H) and q.scales.shape == (1, H // 32 + 1)
    assert torch.equal(q.codes[0, -tail:], want.codes[0]) and q.scales[0, -1] == want.scales[0, 0]
    n = 1 << 24  # the values repeat, and so do their codes
    for k in (0, 63, 126):
        assert torch.equal(q.codes[0, k * n:k * n + n].view(-1, 4096), quantize8(x[:n].view(-1, 4096)).codes)
    back = q.dequantize()
    assert torch.equal(back[-tail:], want.dequantize()) and torch.equal(back[:n], back[126 * n:127 * n])
    del x, back
    two = Packed8(q.codes.expand(2, H).contiguous(), q.scales.expand(2, -1).contiguous(), torch.Size((2, H)), torch.bfloat16)
    del q
    both = two.dequantize()
    assert torch.equal(both[0, -n:], both[1, -n:]) and torch.equal(both[0, :n], both[1, :n])


@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("H,dtype", [(5, torch.float32), (6, torch.float32), (100, torch.float32), (100, torch.bfloat16)])
def test_a_broken_history_stays_alone(H, dtype, masked, checkpoint):
    """A NaN or an infinity in one packed history, or in a gradient that enters it, leaves every bit of the
    others' results: histories over several segments, of one row, from edge to edge and inside a segment."""
    from starry_unigraph.ops.recurrence import gated_scan

    lens = [100, 60, 1, 0, 31, 96, 200, 10]
    off = torch.tensor([0] + lens, device="cuda").cumsum(0)
    n = int(off[-1])
    g = torch.Generator(device="cuda").manual_seed(H)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    p, dh, d = r(n, 3 * H).to(dtype), r(n, H).to(dtype), r(H) - 3
    h0, dl = r(len(lens), H), r(len(lens), H)
    mask = None
    if masked:
        mask = torch.rand(n, device="cuda", generator=g) < 0.7
        mask[off[:-1].clamp_max(n - 1)] = True
    first, last = off[:-1].tolist(), (off[1:] - 1).tolist()

    def run(p, dh, h0, dl):
        q, s = p.clone().requires_grad_(), h0.clone().requires_grad_()
        h, end = gated_scan(q, d, s, offsets=off, mask=mask, checkpoint=checkpoint)
        return [h.detach(), end.detach(), *torch.autograd.grad((h, end), (q, s), (dh, dl))]

    clean = run(p, dh, h0, dl)
    for who, size in enumerate(lens):
        for bad in (float("nan"), float("inf")):
            args = [t.clone() for t in (p, dh, h0, dl)]
            if size:
                args[0][first[who], :H] = bad
                args[1][last[who]] = bad
            args[2][who], args[3][who] = bad, bad
            got = run(*args)
            for a, b in zip(got, clean):
                keep = torch.ones(len(a), dtype=torch.bool, device="cuda")
                keep[slice(first[who], first[who] + size) if len(a) == n else who] = False
                assert torch.equal(a[keep], b[keep]), (who, bad)
            own = slice(first[who], first[who] + size)
            assert not torch.isfinite(got[0][own]).any() and not torch.isfinite(got[2][own, :H][mask[own] if masked else ...]).any()


def test_autograd_sees_the_step():
    """A table that a node saved and a step overwrote before the backward pass is refused as after any
    write in place, through a view too. Tables of inference mode advance outside it as well."""
    from starry_unigraph.ops.recurrence import gated_scan, gated_scan_step

    torch.manual_seed(0)
    p, tok = torch.randn(3, 5, 12, device="cuda", requires_grad=True), torch.randn(3, 12, device="cuda")
    d, w = torch.randn(4, device="cuda"), torch.randn(3, 4, device="cuda", requires_grad=True)
    wide = torch.randn(3, 6, device="cuda")
    for table, rows in ((torch.randn(3, 4, device="cuda"), None), (wide[:, 1:5], torch.arange(3, device="cuda"))):
        outs = [w * table] + ([gated_scan(p, d, table)[0]] if table.is_contiguous() else [])
        gated_scan_step(tok, d, table, rows)
        for out in outs:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.sum().backward()
    with torch.inference_mode():
        table = torch.randn(3, 4, device="cuda")
    want = table.cpu().clone()
    gated_scan_step(tok, d, table)
    gated_scan_step(tok.cpu(), d.cpu(), want)
    assert float((table.cpu() - want).abs().max()) < 1e-5


def test_rows_without_a_sequence_are_refused():
    from starry_unigraph.ops.recurrence import gated_scan

    p, d = torch.randn(5, 12, device="cuda", requires_grad=True), torch.randn(4, device="cuda")
    one = torch.zeros(1, dtype=torch.long, device="cuda")
    for keep in (None, "int8"):
        for q in (p, p.detach()):
            with pytest.raises(RuntimeError, match="no sequence"):
                gated_scan(q, d, offsets=one, checkpoint=keep)
        h, last = gated_scan(p[:0], d, offsets=one, checkpoint=keep)
        assert h.shape == (0, 4) and last.shape == (0, 4)
    for off in (one[:0], one[0]):
        with pytest.raises(RuntimeError, match="offsets must be"):
            gated_scan(p, d, offsets=off)


def test_forward_mode_is_refused():
    """A dual tensor among the inputs, whether or not a gradient is wanted; values outside of it as before."""
    import torch.autograd.forward_ad as fwd

    from starry_unigraph.ops.norm import norm_residual, rms_norm
    from starry_unigraph.ops.recurrence import gated_scan

    p, d, h0 = torch.randn(2, 3, 12, device="cuda"), torch.randn(4, device="cuda"), torch.randn(2, 4, device="cuda")
    x, w = torch.randn(3, 8, device="cuda"), torch.randn(8, device="cuda")
    calls = [(gated_scan, (p, d, h0)), (lambda *a: gated_scan(*a, checkpoint="int8"), (p, d, h0)), (rms_norm, (x, w)),
             (lambda x, u, g, a, b, s: norm_residual(x, u, a, b, gate=g, scale=s), (x, x, x, w, w, w))]
    for f, args in calls:
        for grad in (False, True):
            for k in range(len(args)):
                with fwd.dual_level():
                    a = [t.clone().requires_grad_(grad) for t in args]
                    a[k] = fwd.make_dual(a[k], torch.ones_like(a[k]))
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        f(*a)
        f(*args)


@pytest.mark.parametrize("decay", [-9.0, -3.0, 0.0, 2.0, 3.0, 4.0, 5.0])
@pytest.mark.parametrize("batch,steps", [(2, 2000), (4000, 8)])
def test_gradients_of_fast_and_slow_decays(batch, steps, decay):
    """dr, ddecay and dh0 are multiples of a = exp(-y): they keep their relative precision channel by channel
    where a is small too. y, in the middle 4 softplus(decay), comes from the exponential and the reciprocal
    of a sigmoid (2^-22 and 2^-23 at most), softplus and three products (2^-24 each), 2^-22 of it taken
    together, and a loses as much as y does: y 2^-22 beside the fp32 bound. A dr holds the difference of
    two terms: twice that at the median; ddecay goes by the sum of its terms' magnitudes. A slow channel's
    state gathers the errors of hundreds of steps: four times the fp32 bound."""
    from starry_unigraph.ops.recurrence import gated_scan

    g = torch.Generator().manual_seed(int(decay) + batch)
    H = 8
    p, dh = torch.randn(batch, steps, 3 * H, generator=g), torch.randn(batch, steps, H, generator=g)
    d, h0 = torch.full((H,), decay), torch.randn(batch, H, generator=g)

    def run(device, dtype):
        a = [t.to(device, dtype).requires_grad_() for t in (p, d, h0)]
        return [t.double().cpu() for t in torch.autograd.grad(gated_scan(*a)[0], a, dh.to(device, dtype))]

    (gp, gd, g0), (wp, wd, w0) = run("cuda", torch.float32), run("cpu", torch.float64)
    r, soft = p[..., H:2 * H].double(), torch.nn.functional.softplus(d.double())
    tol = F32 * (4 if decay < 0 else 1) + 4 * float(soft[0]) * 2.0 ** -22
    dr, wr = gp[..., H:2 * H], wp[..., H:2 * H]
    assert ((dr - wr).abs() / wr.abs()).flatten(0, 1).median(0).values.max() < 2 * tol
    terms = wr / (soft * (1 - torch.sigmoid(r))) * torch.sigmoid(d.double())  # -dz c sigmoid(r) sigmoid(decay)
    torch.testing.assert_close(terms.sum((0, 1)), wd, rtol=1e-9, atol=1e-9 * float(terms.abs().sum()))
    assert ((gd - wd).abs() / terms.abs().sum((0, 1))).max() < tol
    assert ((g0 - w0).norm(dim=0) / w0.norm(dim=0)).max() < tol


def test_small_decays_reach_the_first_state():
    """dh0 after one step is a dh: precise relative to itself down to a near 2^-80, 0 below fp32's normal
    numbers. Softplus (2^-23), its product with the rate and the exponent's (2^-24 each) and the
    constant are off by less than 2^-21 of y together, the exponential and its product by 2^-22 each."""
    from starry_unigraph.ops.recurrence import gated_scan

    y = torch.tensor([1e-30, 1e-6, 0.2, 0.25, 0.26, 1, 5, 10, 17, 20, 40, 55, 100])  # -log a at an open gate
    H = len(y)
    p = torch.zeros(1, 1, 3 * H)
    p[..., H:2 * H] = 200.0  # sigmoid(r) = 1
    decay = torch.where(y > 15, y, torch.log(torch.expm1(y.double())).float())  # softplus(decay) = y
    h0 = torch.ones(1, H, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(gated_scan(p.cuda(), decay.cuda(), h0, rate=1.0)[0].sum(), h0)
    want = torch.exp(-torch.nn.functional.softplus(decay.double()))
    want[want < 2.0 ** -126] = 0
    assert ((g.double().cpu()[0] - want).abs() <= (2.0 ** -21 + 2.0 ** -21 * y.double()) * want).all()


@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("layout", ["time", "batch", "packed"])
@pytest.mark.parametrize("steps,H", [(3, 8), (20, 4), (20, 6), (90, 5), (300, 100)])
def test_masked_steps_get_no_gradient_whatever_the_state(steps, H, layout, checkpoint):
    """A sequence without a valid step whose first state is NaN or infinite, and one whose state becomes so,
    with gradients at h that are not finite there: zeros at the masked steps, no share in the decay's sum."""
    from starry_unigraph.ops.recurrence import gated_scan

    g = torch.Generator(device="cuda").manual_seed(steps + H)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    B, T = 3, steps
    p, d, h0, gh = r(B, T, 3 * H), r(H) - 3, r(B, H), r(B, T, H)
    mask = torch.rand(B, T, device="cuda", generator=g) < 0.5
    mask[1], mask[2, T // 2], mask[2, T // 2 + 1:] = False, True, False
    off = torch.arange(B + 1, device="cuda") * T if layout == "packed" else None

    def run(p, h0, gh):
        a = [p.clone().requires_grad_(), d.clone().requires_grad_(), h0.clone().requires_grad_()]
        q, m, e = a[0], mask, gh
        if layout == "time":
            q, m, e = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, m, e))
        if layout == "packed":
            q, m, e = (t.flatten(0, 1) for t in (q, m, e))
        h, _ = gated_scan(q, a[1], a[2], mask=m, offsets=off, checkpoint=checkpoint)
        return [h.detach().reshape(B, T, H), *torch.autograd.grad(h, a, e)]

    clean = run(p, h0, gh.clone().index_fill_(0, torch.tensor([1], device="cuda"), 0.0))
    for bad in (float("nan"), float("inf")):
        h1, g1, p1 = h0.clone(), gh.clone(), p.clone()
        h1[1], g1[1] = bad, bad
        h, dp, dd, d0 = run(p, h1, g1)
        assert torch.equal(dp[~mask], torch.zeros_like(dp[~mask])) and torch.equal(dp, clean[1])
        assert torch.equal(dd, clean[2]) and torch.equal(d0[[0, 2]], clean[3][[0, 2]])
        assert not torch.isfinite(h[1]).any() and not torch.isfinite(d0[1]).any()
        p1[2, T // 2, :H] = bad  # the state of the steps behind it
        dp = run(p1, h0, gh)[1]
        assert torch.equal(dp[~mask], torch.zeros_like(dp[~mask]))


def _turned(t):
    """The same values with the last two dimensions' memory exchanged, as a hook may bring a tensor back."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t


@pytest.mark.parametrize("hooks", ["pinned", "contiguous", "turned"])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("layout", ["time", "batch", "packed"])
def test_saved_tensors_come_back_in_any_layout(layout, checkpoint, hooks):
    """Saved-tensor hooks that move the saved tensors to the host or give them other strides change no bit."""
    from contextlib import nullcontext

    from starry_unigraph.ops.norm import norm_residual
    from starry_unigraph.ops.recurrence import gated_scan

    torch.manual_seed(0)
    p, d, h0 = torch.randn(40, 30, 108, device="cuda"), torch.randn(36, device="cuda"), torch.randn(40, 36, device="cuda")
    x, w = torch.randn(30, 40, 36, device="cuda"), torch.randn(36, device="cuda")
    off = torch.arange(0, 1201, 30, device="cuda") if layout == "packed" else None
    graph = torch.autograd.graph
    made = {"pinned": lambda: graph.save_on_cpu(pin_memory=True),
            "contiguous": lambda: graph.saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t),
            "turned": lambda: graph.saved_tensors_hooks(_turned, lambda t: t)}[hooks]

    def grads(ctx):
        a = [t.clone().requires_grad_() for t in (p, d, h0, x, w)]
        with ctx:
            q = a[0] if layout == "batch" else a[0].flatten(0, 1) if layout == "packed" else \
                a[0].transpose(0, 1).contiguous().transpose(0, 1)
            h, last = gated_scan(q, a[1], a[2], offsets=off, checkpoint=checkpoint)
            y, n = norm_residual(a[3], a[3].sin(), a[4], a[4], gate=a[3].cos(), scale=a[4], checkpoint=checkpoint)
        return torch.autograd.grad(h.square().sum() + last.sum() + y.square().sum() + n.sin().sum(), a)

    for a, b in zip(grads(made()), grads(nullcontext())):
        assert torch.equal(a, b)


_ORDER = """
import sys
import torch
from starry_unigraph.ops.norm import norm_residual
out = {}
for H in map(int, sys.argv[2:]):
    g = torch.Generator(device="cuda").manual_seed(H)
    x, u, gate, dy = (torch.randn(20_000, H, device="cuda", generator=g) for _ in range(4))
    ws = [torch.randn(H, device="cuda", generator=g).requires_grad_() for _ in range(3)]
    y, n = norm_residual(x, u, ws[0], ws[1], gate=gate, scale=ws[2], checkpoint="int8")
    out[H] = [t.cpu() for t in torch.autograd.grad((y, n), ws, (dy, dy))]
torch.save(out, sys.argv[1])
"""


def test_results_do_not_depend_on_which_width_ran_first(tmp_path):
    """172 and 3,000 columns with 8-bit inputs share a kernel and a block size, but not a block's memory."""
    import os
    import subprocess
    import sys
    from pathlib import Path

    root = str(Path(__file__).resolve().parents[1])
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([root, os.environ.get("PYTHONPATH", "")]))
    res = []
    for order in (["172", "3000"], ["3000", "172"]):
        path = str(tmp_path / ("-".join(order) + ".pt"))
        subprocess.run([sys.executable, "-c", _ORDER, path, *order], check=True, cwd=root, env=env, timeout=300)
        res.append(torch.load(path))
    for H in (172, 3000):
        assert all(torch.equal(a, b) for a, b in zip(res[0][H], res[1][H]))


def test_rates_and_eps_that_fp32_cannot_hold_are_refused():
    """An eps that rounds to 0 made NaN of rows of zeros, a rate that rounds to infinity of closed gates."""
    from starry_unigraph.ops.norm import norm_residual, rms_norm
    from starry_unigraph.ops.recurrence import gated_scan, gated_scan_step

    p, d = torch.randn(2, 3, 12, device="cuda"), torch.randn(4, device="cuda")
    x, w, t = torch.zeros(3, 8, device="cuda"), torch.ones(8, device="cuda"), torch.zeros(3, 4, device="cuda")
    for bad in (2.0 ** -150, 1e-60, 3.5e38, 1e300, float("inf"), float("nan"), 0.0, -1.0):
        for f in (lambda: gated_scan(p, d, rate=bad), lambda: gated_scan_step(p[0], d, t, rate=bad),
                  lambda: rms_norm(x, w, eps=bad), lambda: norm_residual(x, x, w, eps=bad)):
            with pytest.raises(RuntimeError, match="positive and finite"):
                f()
    assert not t.any()
    for good in (2.0 ** -149, 1e-40, 3.4e38):
        assert torch.equal(rms_norm(x, w, eps=good), x) and torch.isfinite(gated_scan(p, d - 50, rate=good)[0]).all()


def test_stack_in_bf16():
    """Blocks whose parameters are bfloat16 run the bfloat16 kernels, whole and token by token: about ten
    roundings of 2^-9 a layer apart from the fp32 blocks, root sum square below 1e-2; three times that."""
    import copy

    from starry_unigraph.lib_stable import GatedRecurrentStack

    torch.manual_seed(6)
    m = GatedRecurrentStack(64, num_layers=2).cuda().bfloat16()
    x = torch.randn(20, 30, 64, device="cuda").bfloat16()
    n, last = m(x)
    exact, end = copy.deepcopy(m).float().cpu()(x.float().cpu())
    assert n.dtype == torch.bfloat16 and last[0].dtype == torch.float32
    err = lambda a, b: float((a.float().cpu() - b).detach().norm() / b.detach().norm())  # noqa: E731
    assert err(n, exact) < 3e-2 and all(err(a, b) < 3e-2 for a, b in zip(last, end))
    n.float().square().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters() if p.grad is not None)
    state = m.init_state(30)
    out = torch.stack([m.step(row, state) for row in x])
    assert err(out, exact) < 3e-2 and all(err(a, b) < 3e-2 for a, b in zip(state, end))


def test_step_on_another_stream_advances_the_whole_table():
    from starry_unigraph.ops.recurrence import gated_scan_step

    torch.manual_seed(7)
    p, d, table = torch.randn(400, 96, device="cuda"), torch.randn(32, device="cuda"), torch.randn(500, 32, device="cuda")
    rows = torch.randperm(500, device="cuda")[:400]
    want = table.clone()
    h = gated_scan_step(p, d, want, rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = table.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = gated_scan_step(p, d, got, rows)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, h) and torch.equal(got, want) and not torch.equal(got, table)
    rest = torch.ones(500, dtype=torch.bool, device="cuda").index_fill_(0, rows, False)
    assert torch.equal(got[rest], table[rest])


def test_bytes_kept_in_8_bits():
    """What lives between the forward and the backward pass: 1.125 bytes a value of p, x, u and gate instead of
    four, beside the outputs and the states kept every 16 (8) steps, as asked of the allocator."""
    from starry_unigraph.ops.checkpoint8 import saved8
    from starry_unigraph.ops.norm import norm_residual
    from starry_unigraph.ops.recurrence import gated_scan

    B, T, H = 2000, 33, 64
    n = B * T * H
    p, x = torch.randn(B, T, 3 * H, device="cuda", requires_grad=True), torch.randn(B * T, H, device="cuda", requires_grad=True)
    d, w = torch.randn(H, device="cuda"), torch.randn(H, device="cuda")

    def asked():  # (whole blocks would count up to 1 MB a tensor more)
        return torch.cuda.memory_stats()["requested_bytes.all.current"]

    def kept(f):
        before = asked()
        out = f()
        assert all(t.grad_fn is not None for t in out)
        return asked() - before

    def scan(keep):
        return kept(lambda: gated_scan(p * 1, d, checkpoint=keep))

    def norm(keep):
        return kept(lambda: norm_residual(x * 1, x * 2, w, w, gate=x * 3, checkpoint=keep))

    def packed():
        with saved8():
            return (torch.sin(x * 1),)

    out = 4 * n + 4 * B * H  # h and the last states
    assert scan("int8") == out + 3.375 * n + 4 * B * 2 * H
    assert scan(None) == out + 12 * n + 4 * B * 4 * H
    assert norm("int8") == 8 * n + 3.375 * n
    assert norm(None) == 8 * n + 12 * n
    assert kept(packed) == 4 * n + 1.125 * n
