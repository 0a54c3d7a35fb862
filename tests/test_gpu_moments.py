"""pack_moment on the GPU at the ends of its range: no elements, one, and more than 2^30."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_none_and_one(pkg):
    codes, scales = pkg.pack_moment(torch.zeros(0, 3, device=DEV))
    assert codes.shape == (0, 3) and codes.dtype == torch.float8_e4m3fn and scales.shape == (0,)
    assert pkg.unpack_moment((codes, scales)).shape == (0, 3)
    one = torch.tensor(0.375, device=DEV)
    codes, scales = pkg.pack_moment(one)
    assert codes.shape == () and scales.shape == (1,) and torch.equal(pkg.unpack_moment((codes, scales)), one)


@pytest.mark.parametrize("n", [129, 8192, 8193, (1 << 30) + 128 * 128 + 5])
def test_blocks_of_the_whole(pkg, n):
    """The codes and scale bytes are those of each 128 elements by themselves."""
    print(f"[pack_moment] {n}", flush=True)
    t = torch.empty(n, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(n))
    codes, scales = pkg.pack_moment(t)
    blocks = (n + 127) // 128
    assert codes.shape == (n,) and scales.shape == (blocks,)
    for first in {0, blocks // 2, max(0, blocks - 70)}:
        part = t[first * 128:(first + 70) * 128]
        p = torch.nn.functional.pad(part, (0, -part.numel() % 128)).view(-1, 128)
        q = pkg.fp8_quantize(p)
        assert torch.equal(codes[first * 128:(first + 70) * 128].view(torch.uint8), q.codes.view(torch.uint8).view(-1)[:part.numel()])
        assert torch.equal(scales[first:first + 70], q.scales[:, 0])
