"""The FP8 product with each tile size, in one range of k and in several, on whole numbers, whose sums are exact."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


# tiles of 256, of 128 with two stages and with three, of 64; sizes that end inside a tile, a block and 8 columns
@pytest.mark.parametrize("M,N,K,ranges", [(33683, 1111, 1439, False), (1530, 1533, 32001, True), (725, 5823, 190, False),
                                          (6887, 309, 28966, True), (309, 7373, 3, False), (210, 3063, 25769, True),
                                          (18, 131, 67, False), (17, 1530, 8961, True)])
def test_whole_numbers(pkg, M, N, K, ranges):
    print(f"[fp8 plan] {M} {N} {K}", flush=True)
    assert (pkg._lib.load().hif8_fp8_gemm_workspace_bytes(M, N, K) > 0) == ranges
    g = torch.Generator(device=DEV).manual_seed(M)
    a, b = (torch.empty(n, K, dtype=torch.bfloat16, device=DEV).random_(-2, 3, generator=g) for n in (M, N))
    bias = torch.empty(N, dtype=torch.float32, device=DEV).random_(-9, 10, generator=g)
    y = pkg.fp8_matmul(pkg.fp8_quantize(a), pkg.fp8_quantize(b, tile=True), bias, torch.float32)
    assert torch.equal(y, a.float() @ b.float().t() + bias)
