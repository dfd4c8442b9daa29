"""Edges of the gated recurrence, the norms around a block and 8-bit activations on CPU: what
8-bit saved tensors leave alone, values that are not finite, arguments that are refused."""
import copy
from contextlib import nullcontext

import pytest
import torch

from starry_unigraph.lib_stable import GatedRecurrentStack
from starry_unigraph.ops.checkpoint8 import quantize8, saved8
from starry_unigraph.ops.norm import norm_residual, rms_norm
from starry_unigraph.ops.recurrence import gated_scan, gated_scan_step


def test_saved8_leaves_weights_alone():
    """Gradients of the inputs go through the exact weights: biased linears (which save a transposed view),
    frozen ones, slices of a weight; the weight's own gradient is that of the packed input."""
    torch.manual_seed(0)
    lin, frozen = torch.nn.Linear(256, 300), torch.nn.Linear(300, 256).requires_grad_(False)
    leaf = torch.randn(512, 256, requires_grad=True)
    for f in (lin, lambda x: frozen(lin(x)), lambda x: x @ leaf[:256], lambda x: x @ leaf[100:356].t()):
        x = torch.randn(40, 256, requires_grad=True)
        want, = torch.autograd.grad(f(x).sin().sum(), x)
        with saved8(min_numel=1 << 14):  # above every activation, below the weights
            y = f(x).sin().sum()
        assert torch.equal(torch.autograd.grad(y, x)[0], want)
    x = torch.randn(300, 256)
    with saved8():
        y = lin(x * 1.0)
    g = torch.randn_like(y)
    gw, = torch.autograd.grad(y, lin.weight, g)
    torch.testing.assert_close(gw, g.t() @ quantize8(x).dequantize())


def test_saved8_leaves_sparse_tensors_alone():
    """A sparse adjacency has no rows to pack; its product is differentiated as without saved8."""
    torch.manual_seed(1)
    dense = (torch.rand(300, 300) < 0.05) * torch.randn(300, 300)
    x = torch.randn(300, 3)
    for adj in (dense.to_sparse(), dense.to_sparse_csr()):
        q = x.clone().requires_grad_()
        with saved8():
            y = torch.sparse.mm(adj, q)
        got, = torch.autograd.grad(y.sin().sum(), q)
        torch.testing.assert_close(got, dense.t() @ y.detach().cos())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("layout", ["dense", "packed", "no h0"])
def test_codes_and_states_are_not_packed_again(layout, dtype):
    """checkpoint="int8" inside saved8 gives the gradients that it gives outside."""
    torch.manual_seed(2)
    p, d, h0 = torch.randn(3, 40, 96), torch.randn(32) - 3, torch.randn(3, 32)
    p, h0 = p.to(dtype), h0.to(dtype)
    off = None
    if layout == "packed":
        p, off = p.flatten(0, 1), torch.tensor([0, 50, 50, 120])
    x, u, g = (torch.randn(30, 40).to(dtype) for _ in range(3))
    w = torch.randn(40)

    def grads(inside):
        a = [t.clone().requires_grad_() for t in (p, d, h0, x, u, g)]
        with saved8(min_numel=1) if inside else nullcontext():
            h, last = gated_scan(a[0] * 1, a[1], None if layout == "no h0" else a[2] * 1, offsets=off, checkpoint="int8")
            y, n = norm_residual(a[3] * 1, a[4] * 1, w, w, gate=a[5] * 1, checkpoint="int8")
        loss = h.double().sin().sum() + last.sum() + y.double().sin().sum() + n.double().cos().sum()
        return torch.autograd.grad(loss, a, allow_unused=True)

    for a, b in zip(grads(True), grads(False)):
        assert a is b is None or torch.equal(a, b)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_masked_steps_get_no_gradient_whatever_the_state(checkpoint):
    """A sequence without a valid step whose first state is NaN or infinite, and one whose state becomes so,
    with gradients at h that are not finite there: zeros at the masked steps, the decay's sum untouched by them."""
    torch.manual_seed(3)
    for bad in (float("nan"), float("inf")):
        p, d, h0 = torch.randn(3, 20, 12), torch.randn(4), torch.randn(3, 4)
        mask = torch.rand(3, 20) < 0.5
        mask[1], mask[2, 9], mask[2, 10:] = False, True, False
        h0[1] = bad
        a = [t.clone().requires_grad_() for t in (p, d, h0)]
        gh = torch.randn(3, 20, 4)
        gh[1] = bad
        h, _ = gated_scan(*a, mask=mask, checkpoint=checkpoint)
        dp, dd, d0 = torch.autograd.grad(h, a, gh)
        assert torch.equal(dp[~mask], torch.zeros_like(dp[~mask]))
        b = [t.clone().requires_grad_() for t in (p[[0, 2]], d, h0[[0, 2]])]
        want = torch.autograd.grad(gated_scan(*b, mask=mask[[0, 2]], checkpoint=checkpoint)[0], b, gh[[0, 2]])
        for x, y in zip((dp[[0, 2]], dd, d0[[0, 2]]), want):
            torch.testing.assert_close(x, y)
        assert torch.equal(h[1].detach().nan_to_num(1.0, 2.0), torch.full((20, 4), bad).nan_to_num(1.0, 2.0))
        p[2, 9, :4] = bad  # the state of the steps behind it
        a = [t.clone().requires_grad_() for t in (p, d)]
        dp, = torch.autograd.grad(gated_scan(*a, h0, mask=mask, checkpoint=checkpoint)[0].sum(), a[:1])
        assert torch.equal(dp[~mask], torch.zeros_like(dp[~mask]))


def test_rates_and_eps_that_fp32_cannot_hold_are_refused():
    p, d, x, w = torch.randn(2, 3, 12), torch.randn(4), torch.zeros(3, 8), torch.ones(8)
    for bad in (2.0 ** -150, 1e-60, 3.5e38, 1e300, float("inf"), float("nan"), 0.0, -1.0):
        for f in (lambda: gated_scan(p, d, rate=bad), lambda: gated_scan_step(p[0], d, torch.zeros(3, 4), rate=bad),
                  lambda: rms_norm(x, w, eps=bad), lambda: norm_residual(x, x, w, eps=bad)):
            with pytest.raises(ValueError):
                f()
    for good in (2.0 ** -149, 1e-40, 3.4e38):
        assert torch.equal(rms_norm(x, w, eps=good), x) and torch.isfinite(gated_scan(p, d - 50, rate=good)[0]).all()
    assert torch.equal(rms_norm(x.double(), w.double(), eps=1e-60), x.double())


def test_step_refuses_places_outside_the_table():
    """Nothing is written, of the valid places neither; -1 is no last row."""
    torch.manual_seed(4)
    p, d = torch.randn(3, 12), torch.randn(4)
    for rows in ([0, 1, -1], [0, 1, 5], [-5, 1, 2]):
        table = torch.ones(5, 4)
        with pytest.raises(IndexError):
            gated_scan_step(p, d, table, torch.tensor(rows))
        assert torch.equal(table, torch.ones(5, 4))
    for rows, decay in ((torch.tensor([True, True, True]), d), (torch.tensor([[0], [1], [2]]), d),
                        (torch.tensor([0, 1, 2]), d[:1])):
        with pytest.raises(ValueError):
            gated_scan_step(p, decay, table, rows)
    assert gated_scan_step(p[:0], d, table, torch.zeros(0, dtype=torch.long)).shape == (0, 4)


def test_scan_refuses_empty_offsets():
    for keep in (None, "int8"):
        for off in (torch.zeros(0, dtype=torch.long), torch.zeros(1, dtype=torch.long)):
            with pytest.raises(ValueError):
                gated_scan(torch.randn(3, 6), torch.randn(2), offsets=off, checkpoint=keep)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_stack_runs_in_the_type_of_its_parameters(checkpoint):
    """float64 blocks whole and token by token to 64 bits, and the fp32 blocks' results to 32."""
    torch.manual_seed(5)
    m = GatedRecurrentStack(12, num_layers=2, checkpoint=checkpoint)
    x = torch.randn(7, 5, 12)
    n, last = m(x)
    m64 = copy.deepcopy(m).double()
    n64, last64 = m64(x)
    assert n64.dtype == last64[0].dtype == torch.float64 and n.dtype == last[0].dtype == torch.float32
    torch.testing.assert_close(n64.float(), n, rtol=1e-4, atol=1e-5)
    state = m64.init_state(5)
    out = torch.stack([m64.step(row, state) for row in x])
    torch.testing.assert_close(out, n64, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(state, last64, rtol=1e-12, atol=1e-12)
    n64.square().sum().backward()
    assert all(torch.isfinite(p.grad).all() and p.grad.dtype == torch.float64 for p in m64.parameters() if p.grad is not None)
    assert m.bfloat16()(x)[0].dtype == torch.bfloat16
