"""The gated recurrence, the norms around a block and 8-bit activations on CPU: against
plain loops in 64 bits, gradients against differences, refusals."""
import math

import pytest
import torch

from starry_unigraph.ops.checkpoint8 import Packed8, quantize8, saved8
from starry_unigraph.ops.norm import norm_residual, rms_norm
from starry_unigraph.ops.recurrence import STATE_EVERY, gated_scan, gated_scan_step


def naive_scan(p, decay, h0, mask=None, rate=8.0):
    """Element by element with Python floats (64 bits): h [B, T, H], last [B, H]."""
    B, T, W = p.shape
    H = W // 3
    h = torch.zeros(B, T, H, dtype=torch.float64)
    last = torch.zeros(B, H, dtype=torch.float64)
    for b in range(B):
        for c in range(H):
            s = float(h0[b, c]) if h0 is not None else 0.0
            soft = math.log1p(math.exp(float(decay[c])))
            for t in range(T):
                if mask is None or bool(mask[b, t]):
                    x, r, i = (float(p[b, t, c + k * H]) for k in range(3))
                    a = math.exp(-rate * soft / (1 + math.exp(-r)))
                    s = a * s + math.sqrt(1 - a * a) / (1 + math.exp(-i)) * x
                h[b, t, c] = s
            last[b, c] = s
    return h, last


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (2, 5, 3), (3, 20, 4)])
def test_scan_matches_the_loop(B, T, H, masked):
    torch.manual_seed(B * 100 + T)
    p = torch.randn(B, T, 3 * H, dtype=torch.float64)
    decay, h0 = torch.randn(H, dtype=torch.float64), torch.randn(B, H, dtype=torch.float64)
    mask = torch.rand(B, T) < 0.6 if masked else None
    if masked:
        mask[0] = False
        p[~mask] = float("nan")
    h, last = gated_scan(p, decay, h0, mask=mask)
    ref, rlast = naive_scan(p, decay, h0, mask)
    torch.testing.assert_close(h, ref, rtol=1e-10, atol=1e-12)
    torch.testing.assert_close(last, rlast, rtol=1e-10, atol=1e-12)


@pytest.mark.parametrize("masked", [False, True])
def test_scan_gradient_against_differences(masked):
    torch.manual_seed(0)
    p = torch.randn(2, 6, 6, dtype=torch.float64, requires_grad=True)
    decay = torch.randn(2, dtype=torch.float64, requires_grad=True)
    h0 = torch.randn(2, 2, dtype=torch.float64, requires_grad=True)
    mask = torch.rand(2, 6) < 0.6 if masked else None
    assert torch.autograd.gradcheck(lambda *a: gated_scan(*a, mask=mask, rate=2.0), (p, decay, h0))


def test_scan_packed_is_every_sequence_alone():
    torch.manual_seed(1)
    H, lens = 3, [0, 4, 1, 0, 0, 37, 2, 0]
    off = torch.tensor([0] + lens).cumsum(0)
    p = torch.randn(int(off[-1]), 3 * H, dtype=torch.float64)
    decay, h0 = torch.randn(H, dtype=torch.float64), torch.randn(len(lens), H, dtype=torch.float64)
    h, last = gated_scan(p, decay, h0, offsets=off)
    for s, n in enumerate(lens):
        a, b = int(off[s]), int(off[s + 1])
        if n == 0:
            assert torch.equal(last[s], h0[s])
            continue
        ref, rlast = gated_scan(p[a:b].unsqueeze(0), decay, h0[s:s + 1])
        assert torch.equal(h[a:b], ref[0]) and torch.equal(last[s], rlast[0])


def test_scan_closed_gate_keeps_the_state_and_has_finite_gradients():
    p = torch.zeros(1, 4, 3, dtype=torch.float64)
    p[..., 1] = -1e6  # sigmoid(r) underflows: a = 1, nothing enters
    p.requires_grad_()
    h, _ = gated_scan(p, torch.zeros(1, dtype=torch.float64), torch.full((1, 1), 2.0, dtype=torch.float64))
    assert torch.equal(h.detach(), torch.full_like(h, 2.0))
    g, = torch.autograd.grad(h.sum(), p)
    assert torch.isfinite(g).all()


def test_scan_steps_one_by_one():
    torch.manual_seed(2)
    B, T, H = 4, 9, 5
    p, decay, h0 = torch.randn(B, T, 3 * H), torch.randn(H), torch.randn(B, H)
    h, last = gated_scan(p, decay, h0)
    table = torch.zeros(10, H)
    rows = torch.tensor([7, 0, 3, 9])
    table[rows] = h0
    for t in range(T):
        out = gated_scan_step(p[:, t], decay, table, rows)
        torch.testing.assert_close(out, h[:, t], rtol=1e-6, atol=1e-6)
    torch.testing.assert_close(table[rows], last, rtol=1e-6, atol=1e-6)
    assert torch.equal(table[[1, 2, 4, 5, 6, 8]], torch.zeros(6, H))


@pytest.mark.parametrize("packed", [False, True])
def test_scan_int8_gradients_are_those_at_the_codes(packed):
    """One chunk of steps: nothing but the codes enters the gradient."""
    torch.manual_seed(3)
    B, T, H = 3, STATE_EVERY, 40
    p, decay, h0 = torch.randn(B, T, 3 * H), torch.randn(H), torch.randn(B, H)
    if packed:
        p, off = p.reshape(-1, 3 * H), torch.arange(B + 1) * T
    else:
        off = None
    g, gl = torch.randn(*p.shape[:-1], H), torch.randn(B, H)
    a = [t.clone().requires_grad_() for t in (p, decay, h0)]
    h, last = gated_scan(*a, offsets=off, checkpoint="int8")
    got = torch.autograd.grad((h, last), a, (g, gl))
    back = quantize8(p.unflatten(-1, (3, H))).dequantize().flatten(-2)
    b = [t.clone().requires_grad_() for t in (back, decay, h0)]
    want = torch.autograd.grad(gated_scan(*b, offsets=off), b, (g, gl))
    torch.testing.assert_close(h, gated_scan(p, decay, h0, offsets=off)[0])
    for x, y in zip(got, want):
        torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-6)


def test_scan_refuses():
    p, d = torch.randn(2, 3, 6), torch.randn(2)
    for bad in (lambda: gated_scan(torch.randn(2, 3, 7), d), lambda: gated_scan(p, torch.randn(3)),
                lambda: gated_scan(p[0], d), lambda: gated_scan(p, d, torch.randn(3, 2)),
                lambda: gated_scan(p, d, mask=torch.ones(2, 3)), lambda: gated_scan(p, d, rate=0.0),
                lambda: gated_scan(p, d, mask=torch.ones(3, 2, dtype=torch.bool)),
                lambda: gated_scan(p, d, checkpoint="fp8"),
                lambda: gated_scan(p[0], d, offsets=torch.tensor([0, 2])),
                lambda: gated_scan(p[0], d, offsets=torch.tensor([0, 2, 1, 3])),
                lambda: gated_scan_step(p[0], d, torch.zeros(2, 2)),
                lambda: gated_scan_step(p[0], d, torch.zeros(3, 3))):
        with pytest.raises(ValueError):
            bad()


def test_scan_of_nothing():
    d = torch.randn(2)
    h, last = gated_scan(torch.randn(3, 0, 6), d, torch.ones(3, 2))
    assert h.shape == (3, 0, 2) and torch.equal(last, torch.ones(3, 2))
    h, last = gated_scan(torch.randn(0, 5, 6), d)
    assert h.shape == (0, 5, 2) and last.shape == (0, 2)


@pytest.mark.parametrize("gate,scale,post,pre", [(1, 1, 1, 1), (0, 1, 1, 1), (1, 0, 0, 1), (1, 1, 1, 0), (0, 0, 0, 1)])
def test_norm_gradient_against_differences(gate, scale, post, pre):
    torch.manual_seed(4)
    mk = lambda *s: torch.randn(*s, dtype=torch.float64, requires_grad=True)  # noqa: E731
    x, u = mk(3, 5), mk(3, 5)
    args = {"w_post": mk(5) if post else None, "w_pre": mk(5) if pre else None, "gate": mk(3, 5) if gate else None,
            "scale": mk(5) if scale else None}
    names = [k for k, v in args.items() if v is not None]

    def f(x, u, *rest):
        a = args | dict(zip(names, rest))
        return tuple(t for t in norm_residual(x, u, a["w_post"], a["w_pre"], gate=a["gate"], scale=a["scale"],
                                              eps=1e-3) if t is not None)

    assert torch.autograd.gradcheck(f, (x, u, *[args[k] for k in names]))


def test_norm_formula():
    torch.manual_seed(5)
    x, u, g = (torch.randn(4, 7, dtype=torch.float64) for _ in range(3))
    wp, wn, sc = (torch.randn(7, dtype=torch.float64) for _ in range(3))
    y, n = norm_residual(x, u, wp, wn, gate=g, scale=sc, eps=1e-5)
    for r in range(4):
        ru = 1 / math.sqrt(sum(float(v) ** 2 for v in u[r]) / 7 + 1e-5)
        want = [float(x[r, c] + sc[c] / (1 + math.exp(-float(g[r, c]))) * u[r, c] * ru * wp[c]) for c in range(7)]
        ry = 1 / math.sqrt(sum(v * v for v in want) / 7 + 1e-5)
        torch.testing.assert_close(y[r], torch.tensor(want, dtype=torch.float64))
        torch.testing.assert_close(n[r], torch.tensor([v * ry * float(wn[c]) for c, v in enumerate(want)],
                                                      dtype=torch.float64))
    torch.testing.assert_close(rms_norm(y, wn, eps=1e-5), n)


def test_norm_int8_gradients_are_those_at_the_codes():
    torch.manual_seed(6)
    x, u, g = (torch.randn(6, 40) for _ in range(3))
    vec = [torch.randn(40) for _ in range(3)]
    gy, gn = torch.randn(6, 40), torch.randn(6, 40)

    def grads(x, u, g, keep):
        a = [t.clone().requires_grad_() for t in (x, u, g, *vec)]
        out = norm_residual(a[0], a[1], a[3], a[4], gate=a[2], scale=a[5], checkpoint=keep)
        return out, torch.autograd.grad(out, a, (gy, gn))

    out, got = grads(x, u, g, "int8")
    _, want = grads(*(quantize8(t).dequantize() for t in (x, u, g)), None)
    plain = norm_residual(x, u, vec[0], vec[1], gate=g, scale=vec[2])
    torch.testing.assert_close(out, plain)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)


def test_norm_refuses():
    x, w = torch.randn(3, 4), torch.randn(4)
    for bad in (lambda: norm_residual(x, torch.randn(3, 5), w), lambda: norm_residual(x, x, torch.randn(5)),
                lambda: norm_residual(x, x.double(), w), lambda: norm_residual(x, x, w, gate=x[:1]),
                lambda: norm_residual(x, x, w, eps=0.0), lambda: norm_residual(x, x, w, checkpoint="int4"),
                lambda: rms_norm(torch.randn(3, 0), torch.randn(0))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("H", [1, 31, 32, 33, 100])
def test_codes_stay_within_half_a_scale(H):
    torch.manual_seed(H)
    x = torch.randn(50, H) * torch.exp(3 * torch.randn(50, 1))
    x[7] = 0
    q = quantize8(x)
    assert q.codes.dtype == torch.int8 and q.scales.shape == (50, -(-H // 32))
    back = q.dequantize()
    wide = q.scales.repeat_interleave(32, 1)[:, :H]
    # half a scale for the rounding, and the two roundings of v * (127 / amax) at up to 127
    assert ((back - x).abs() <= wide * (0.5 + 127 * 2.0 ** -22)).all()
    assert torch.equal(back[7], torch.zeros(H))
    top = torch.nn.functional.pad(x, (0, -H % 32)).unflatten(1, (-1, 32)).abs().amax(2)
    assert torch.equal(torch.nn.functional.pad(q.codes, (0, -H % 32)).unflatten(1, (-1, 32)).abs().amax(2),
                       torch.where(top > 0, 127, 0).to(torch.int8))


def test_codes_of_broken_and_tiny_groups():
    x = torch.ones(4, 64)
    x[0, 3] = float("nan")
    x[1, 40] = float("-inf")
    x[2, :32] = 1e-38
    back = quantize8(x).dequantize()
    assert back[0, :32].isnan().all() and torch.equal(back[0, 32:], x[0, 32:])
    assert back[1, 32:].isnan().all() and torch.equal(back[1, :32], x[1, :32])
    assert torch.equal(back[2, :32], torch.zeros(32)) and torch.equal(back[3], x[3])


def test_codes_keep_shape_type_and_refuse():
    x = torch.randn(2, 3, 5, 33).bfloat16()
    q = quantize8(x.transpose(0, 1))
    assert isinstance(q, Packed8) and q.dequantize().shape == (3, 2, 5, 33) and q.dequantize().dtype == torch.bfloat16
    assert q.nbytes == 30 * 33 + 30 * 2 * 4
    assert quantize8(torch.randn(0, 5)).dequantize().shape == (0, 5)
    for bad in (torch.randn(3, 0), torch.tensor(1.0), torch.ones(3, 4, dtype=torch.int32)):
        with pytest.raises(ValueError):
            quantize8(bad)


def test_saved8_gradients_come_from_the_codes():
    """A weight gradient inside the block is that of the packed input; leaves, small and marked tensors stay."""
    torch.manual_seed(7)
    x, w = torch.randn(64, 40), torch.randn(8, 40, requires_grad=True)
    inp = x * 1.0
    with saved8(min_numel=1):
        y = torch.nn.functional.linear(inp, w)
    g = torch.randn_like(y)
    gw, = torch.autograd.grad(y, w, g)
    torch.testing.assert_close(gw, g.t() @ quantize8(x).dequantize())
    with saved8():  # below min_numel
        gw, = torch.autograd.grad(torch.nn.functional.linear(inp, w), w, g)
    torch.testing.assert_close(gw, g.t() @ x)


def test_stack_steps_match_the_scan():
    """The blocks over a window equal the same blocks advanced token by token; absent rows keep their state."""
    from starry_unigraph.lib_stable import GatedRecurrentStack

    torch.manual_seed(8)
    m = GatedRecurrentStack(12, num_layers=2)
    x = torch.randn(7, 5, 12)
    n, last = m(x)
    state = m.init_state(9)
    rows = torch.tensor([8, 1, 0, 5, 3])
    for t in range(7):
        out = m.step(x[t], state, rows)
        torch.testing.assert_close(out, n[t], rtol=1e-5, atol=1e-5)
    for a, b in zip(state, last):
        torch.testing.assert_close(a[rows], b, rtol=1e-5, atol=1e-5)
    mask = torch.rand(7, 5) < 0.5
    mask[:, 2] = False
    x[~mask] = float("nan")
    n, last = m(x, mask=mask)
    (n.square().sum() + sum(s.sum() for s in last)).backward()
    assert all(torch.equal(s[2], torch.zeros(12)) for s in last)
    assert all(torch.isfinite(p.grad).all() for p in m.parameters())
    n2, mid = m(x[:4], mask=mask[:4])
    n3, end = m(x[4:], mid, mask[4:])
    for a, b in zip(end, last):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
    with pytest.raises(ValueError):
        m(torch.randn(2, 3, 11))
    with pytest.raises(ValueError):
        GatedRecurrentStack(8, checkpoint="int4")


def test_example_learns_and_int8_follows_fp32(tmp_path, monkeypatch):
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "train_gated_recurrence.py"
    spec = importlib.util.spec_from_file_location("train_gated_recurrence", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    monkeypatch.chdir(tmp_path)
    res = {}
    for keep in ("none", "int8"):
        res[keep] = ex.main(["--nodes", "300", "--edges", "1500", "--snapshots", "12", "--epochs", "2", "--checkpoint", keep,
                             "--artifact-root", str(tmp_path / keep)])
        assert res[keep]["train"][-1] < res[keep]["train"][0] and res[keep]["test"] > 0
    # 8-bit activations move a gradient by about half a percent
    assert abs(res["int8"]["train"][-1] - res["none"]["train"][-1]) < 0.02 * res["none"]["train"][-1]
