"""modulated_layer_norm and layer_norm on the GPU: many batch entries, each gradient by itself, odd addresses."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_layer_norm import check, inputs, reference  # noqa: E402

DEV = "cuda:0"


@pytest.mark.parametrize("shape,both", [((65536, 1, 16), True), ((140000, 2, 24), True), ((70001, 1, 64), False)])
def test_many_entries(pkg, shape, both):
    """More batch entries than a grid's second dimension takes; ``both``: one shift and one scale an entry, otherwise one
    shift for all of them."""
    print(f"[norm entries] {shape}", flush=True)
    B, M, D = shape
    g = torch.Generator().manual_seed(B)
    x, dy = (torch.randn(shape, generator=g).to(torch.bfloat16) for _ in range(2))
    scale = (torch.randn(B, 1, D, generator=g) * 0.5).to(torch.bfloat16)
    shift = (torch.randn((B, 1, D) if both else (D,), generator=g) * 0.5).to(torch.bfloat16)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, shift, scale)]
    y = pkg.modulated_layer_norm(*leaves)
    assert y.shape == x.shape and y.dtype == x.dtype
    dx, dshift, dscale = torch.autograd.grad(y, leaves, dy.to(DEV))
    ref = reference(x, 1 + scale.double(), shift.double().expand(B, 1, D), dy, 1e-6)
    check(y, ref[0], "y")
    check(dx, ref[1], "dx")
    check(dscale, ref[2], "dscale")
    if both:
        check(dshift, ref[3], "dshift")
    else:
        # an entry's row is rounded, then torch adds them up: its sum of bf16 values in fp32 and rounds once
        want, mag = dy.double().sum((0, 1)), dy.double().abs().sum((0, 1))
        off = mag * (torch.finfo(torch.bfloat16).eps / 2 + B * 2.0 ** -24) + want.abs() * torch.finfo(torch.bfloat16).eps / 2
        assert ((dshift.cpu().double() - want).abs() <= off).all()
    if M == 1:                                     # a 2-D x with a row of the modulation each
        flat = pkg.modulated_layer_norm(x.to(DEV).view(B, D), leaves[1].detach().view(B, D) if both else leaves[1].detach(),
                                        scale.to(DEV).view(B, D))
        assert torch.equal(flat, y.detach().view(B, D))


@pytest.mark.parametrize("D", [256, 250, 2052, 5])
def test_each_gradient_by_itself(pkg, D):
    """The gradient of one of the leaves alone is that of all of them together (with no column sums for x's)."""
    x, dy, e = (t.to(DEV) for t in inputs((3, 10, D), torch.bfloat16, torch.bfloat16, 5))
    values = (x, e[:, 0:1].contiguous(), e[:, 1:2].contiguous())
    leaves = [t.clone().requires_grad_(True) for t in values]
    full = torch.autograd.grad(pkg.modulated_layer_norm(*leaves), leaves, dy)
    for k in range(3):
        one = [t.clone().requires_grad_(i == k) for i, t in enumerate(values)]
        g, = torch.autograd.grad(pkg.modulated_layer_norm(*one), one[k], dy)
        assert torch.equal(g, full[k]), k
    w, b = values[1][0, 0], values[2][0, 0]
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    full = torch.autograd.grad(pkg.layer_norm(*leaves), leaves, dy)
    for k in range(3):
        one = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        g, = torch.autograd.grad(pkg.layer_norm(*one), one[k], dy)
        assert torch.equal(g, full[k]), k


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [256, 250, 2052, 5])
def test_odd_addresses(pkg, D, dtype):
    """x, dy and the weights one element behind an aligned address: the same bits, by the same loads."""
    x, dy, e = (t.to(DEV) for t in inputs((3, 10, D), dtype, dtype, 6))
    values = (x, e[0, 0].contiguous(), e[0, 1].contiguous())

    def moved(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        buf[1:].copy_(t.reshape(-1))
        return buf[1:].view(t.shape)
    out = []
    for f in (torch.clone, moved):
        leaves = [f(t).requires_grad_(True) for t in values]
        y = pkg.layer_norm(*leaves)
        out.append([y.detach(), *torch.autograd.grad(y, leaves, f(dy))])
    assert all(torch.equal(a, b) for a, b in zip(*out))
