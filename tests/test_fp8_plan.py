"""The FP8 product's k ranges at sizes whose plans were timed: the workspace holds a float an output and range."""
from __future__ import annotations

import pytest

pytest.importorskip("torch")


@pytest.mark.parametrize("M,N,K,least,most", [
    # few rows: ranges where a long k has few tiles, none where the tiles suffice
    (16, 13824, 5120, 1, 1), (1, 13824, 5120, 1, 1), (128, 5120, 5120, 1, 1), (64, 1536, 1536, 1, 1),
    (1, 1536, 8960, 3, 8), (16, 1536, 8960, 3, 8), (64, 1536, 8960, 3, 8), (128, 1536, 8960, 3, 6),
    (16, 5120, 13824, 3, 3), (1, 5120, 5120, 2, 4),
    # a weight's gradient, and products that fill the GPU
    (1536, 1536, 32760, 5, 8), (512, 5120, 5120, 1, 1), (4680, 1536, 8960, 1, 1), (75600, 13824, 5120, 1, 1)])
def test_ranges(pkg, M, N, K, least, most):
    nbytes = pkg._lib.load().hif8_fp8_gemm_workspace_bytes(M, N, K)
    assert nbytes % (4 * M * N) == 0
    assert least <= max(1, nbytes // (4 * M * N)) <= most
