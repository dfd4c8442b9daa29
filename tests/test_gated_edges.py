"""Edges of the gated recurrence, the norms around a block and 8-bit activations on CPU: what
8-bit saved tensors leave alone, values that are not finite, arguments that are refused."""
import pytest
import torch

from starry_unigraph.ops.checkpoint8 import quantize8, saved8


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
