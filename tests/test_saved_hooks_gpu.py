"""GPU: backward passes of the convolution path and the losses when saved-tensor hooks hand tensors back in another layout.

Memory formats are part of what the kernels assume, and no part of what a hook has to keep: torch.autograd.graph.save_on_cpu with pinned
memory hands channels_last tensors back in torch's default layout.  The gradients are the same bits.
"""
import pytest
import torch
import torch.nn as nn

from srmi import autograd as AG
from srmi import losses

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _transposed(t):
    """an equal tensor whose last two axes lie the other way round in memory"""
    return t.detach().transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t.detach().clone()


HOOKS = {"pinned": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True), "pageable": lambda: torch.autograd.graph.save_on_cpu(),
         "transposed": lambda: torch.autograd.graph.saved_tensors_hooks(_transposed, lambda t: t)}


def _same_gradients(f, leaves, hook):
    def run():
        y = f()
        gen = torch.Generator().manual_seed(3)
        return torch.autograd.grad(y, leaves, torch.randn(y.shape, generator=gen).to(DEV))

    want = run()
    with HOOKS[hook]():
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("hook", sorted(HOOKS))
@pytest.mark.parametrize("kind", ["prelu_bn", "relu", "residual", "shuffle", "thin", "strided"])
def test_convolutions(kind, hook):
    torch.manual_seed(1)
    cin, cout, stride, k = {"thin": (3, 64, 1, 3), "strided": (64, 128, 2, 3), "shuffle": (32, 64, 1, 3)}.get(kind, (64, 64, 1, 3))
    conv = nn.Conv2d(cin, cout, k, stride=stride, padding=1).to(DEV)
    bn = nn.BatchNorm2d(cout).to(DEV) if kind == "prelu_bn" else None
    act = nn.PReLU().to(DEV) if kind in ("prelu_bn", "shuffle") else nn.ReLU() if kind == "relu" else nn.LeakyReLU(0.2)
    x = torch.randn(2, cin, 10, 14, device=DEV, requires_grad=True)
    res = torch.randn(2, cout, 10, 14, device=DEV, requires_grad=True) if kind == "residual" else None
    leaves = [x, *conv.parameters()] + ([*bn.parameters()] if bn else []) + [*act.parameters()] + ([res] if res is not None else [])
    _same_gradients(lambda: AG.fused_conv(x, conv, bn, act, residual=res, shuffle=2 if kind == "shuffle" else 1), leaves, hook)


@pytest.mark.parametrize("hook", sorted(HOOKS))
def test_linear_and_pool(hook):
    torch.manual_seed(2)
    x = torch.randn(4, 32, 6, 8, device=DEV, requires_grad=True)
    lin = nn.Linear(32 * 6 * 8, 40).to(DEV)
    _same_gradients(lambda: AG.linear(x, lin, nn.LeakyReLU(0.2)), [x, *lin.parameters()], hook)
    _same_gradients(lambda: AG.maxpool2x2(x), [x], hook)


@pytest.mark.parametrize("hook", sorted(HOOKS))
@pytest.mark.parametrize("layout", [torch.contiguous_format, torch.channels_last])
def test_losses(layout, hook):
    torch.manual_seed(4)
    a, b = (torch.rand(2, 3, 9, 7, device=DEV).contiguous(memory_format=layout).requires_grad_() for _ in range(2))
    _same_gradients(lambda: losses.mse_loss(a, b), [a, b], hook)
    _same_gradients(lambda: losses.bce_loss(a, b.detach()), [a], hook)
    _same_gradients(lambda: losses.TVLoss()(a), [a], hook)
