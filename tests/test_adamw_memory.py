"""AdamW refuses lists whose written tensors share memory before it changes any of them, also across types."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


def lists(*rows):
    return [[r[k] for r in rows] for k in range(4)]


def row(n, dtype, **given):
    return [given.get(k, torch.zeros(n, dtype=torch.float32 if k in "mv" else dtype)) for k in "pgmv"]


def call(pkg, *rows, **kw):
    pkg.adamw_step(*lists(*rows), torch.zeros(1, dtype=torch.int64), lr=1e-3, **kw)


def test_shared_across_types(pkg):
    b16, f32 = torch.bfloat16, torch.float32
    with pytest.raises(ValueError, match="GPU"):                            # nothing shared: refused for the device
        call(pkg, row(64, f32), row(64, b16))
    m = torch.zeros(64)
    with pytest.raises(ValueError, match="share"):                          # a moment of both
        call(pkg, row(64, f32, m=m), row(64, b16, m=m))
    with pytest.raises(ValueError, match="share"):                          # the fp32 parameter is the other's moment
        call(pkg, row(64, f32, p=m), row(64, b16, v=m))
    both = torch.zeros(65)
    with pytest.raises(ValueError, match="share"):                          # the last element of one, the first of the other
        call(pkg, row(64, f32, v=both[:64]), row(2, b16, m=both[63:]))
    with pytest.raises(ValueError, match="GPU"):                            # next to each other
        call(pkg, row(64, f32, v=both[:64]), row(1, b16, m=both[64:]))


def test_shared_in_8_bits(pkg):
    def packed(n):
        return torch.zeros(n, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros((n + 127) // 128, dtype=torch.uint8)
    a, b = packed(200), packed(200)
    rows = [row(200, torch.bfloat16, m=packed(200), v=a), row(200, torch.float32, m=packed(200), v=b)]
    with pytest.raises(ValueError, match="GPU"):
        call(pkg, *rows)
    rows[1][3] = (b[0], a[1])                                               # the scale bytes of both
    with pytest.raises(ValueError, match="share"):
        call(pkg, *rows)


def test_a_later_types_tensor_too_long(pkg):
    """(Addresses alone: nothing is read.)"""
    from ospnext_amd import optim

    def at(k, n):
        return (k, k + (1 << 39), k + (1 << 40), k + (1 << 41), 0, 0, 0, n, 0)
    rows = {torch.float32: [at(1 << 44, 64)], torch.bfloat16: [at(1 << 45, 1 << 34)]}
    optim._check_types(rows, False)
    rows[torch.bfloat16] = [at(1 << 45, (1 << 34) + 1)]
    with pytest.raises(ValueError, match="elements"):
        optim._check_types(rows, False)


def test_gradients(pkg):
    """A gradient may be shared by parameters, but not be what the step writes."""
    import numpy as np
    L = pkg._lib.load()
    at = 0x1000000                                          # never dereferenced: every call is refused

    def step(rows):
        t = np.array(rows, dtype=np.uint64)
        return L.hif8_adamw_step(t.ctypes.data, len(rows), 1, 32, at, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0, at, 64, None)

    def one(p, g, n=64):
        return (p, g, p + 0x1000, p + 0x2000, 0, 0, 0, n, 0)
    p, q, g = at + 0x10000, at + 0x20000, at + 0x30000
    assert step([one(p, p)]) == -1                          # its own parameter
    assert step([one(p, g), one(q, p + 252)]) == -1         # another's last element
    assert step([one(p, p + 0x1000 - 252)]) == -1           # the first of a moment
    assert step([one(p, g), one(q, q + 0x2080)]) == -1      # inside the other moment
    f32 = torch.float32
    shared = torch.zeros(64)
    with pytest.raises(ValueError, match="gradient"):       # across types
        call(pkg, row(64, f32, g=shared), row(64, torch.bfloat16, m=shared))
    with pytest.raises(ValueError, match="GPU"):            # of two parameters
        call(pkg, row(64, f32, g=shared), row(64, f32, g=shared), row(8, torch.bfloat16))
