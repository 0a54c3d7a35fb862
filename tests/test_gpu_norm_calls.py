"""modulated_layer_norm and layer_norm on the GPU: many batch entries."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_layer_norm import check, reference  # noqa: E402

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
