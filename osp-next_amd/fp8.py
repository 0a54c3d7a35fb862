"""Linear layers in block-scaled FP8, forward and backward on the 8-bit matrix instructions.

Where ``HIF8Linear`` rounds its operands to HiF8 and multiplies them as bf16, ``FP8Linear`` multiplies
8-bit codes: 128 consecutive values (of a row of the activations or the gradient), or 128 x 128 of a
weight, share one power-of-two scale, which the matrix instruction applies.  With x_q, w_q and g_q the
quantised values::

    y  = x_q @ w_q.T + bias         blocks of x along the input features
    dx = g_q @ w_q                  blocks of g along the output features
    dw = g_q'.T @ x_q'              blocks of g and x along the tokens
    db = g.sum(0)                   the gradient as it came, summed in fp32

The weight's 128 x 128 tiles hold the same values read along either axis; activations and gradients are
quantised along both axes in one pass.

The matrix instruction cuts the terms of 8 values of k off towards zero, 13 bits below the largest of them; the sums of
8 are added in fp32 and rounded once.  Against the exact product of the same codes an fp32 result is off by 1.1e-5 to
1.5e-5 (in the norm) for values of one size, and by 4e-5 to 5e-5 where a few channels are 20 times the others.  An fp16
output, whose rounding alone is 2.07e-4, comes to 2.08e-4 and 2.13e-4 with that, a bf16 one stays at 1.66e-3.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from . import _lib

BLOCK = 128
FORMATS = {torch.float8_e4m3fn: _lib.FP8_E4M3, torch.float8_e5m2: _lib.FP8_E5M2}


def _round_up(v: int, m: int) -> int:
    return (v + m - 1) // m * m


def _format(dtype: torch.dtype) -> int:
    if dtype not in FORMATS:
        raise TypeError(f"FP8 blocks are float8_e4m3fn or float8_e5m2, got {dtype}")
    return FORMATS[dtype]


class FP8Blocks:
    """A matrix [R, cols] in FP8 blocks along its rows: ``codes`` [R, cols rounded up to 128] in a float8
    type, zeros behind the last column (NaN in a block that has one), and ``scales`` [R, blocks rounded up to 4] (uint8): block b of a row
    stands for its codes times 2^(scale - 127).  ``dtype``: the type of the matrix it was made from, if known."""

    def __init__(self, codes: Tensor, scales: Tensor, cols: int, dtype: Optional[torch.dtype] = None):
        _format(codes.dtype)
        if codes.dim() != 2 or scales.dim() != 2 or scales.dtype != torch.uint8:
            raise TypeError("FP8Blocks takes 2-D float8 codes and 2-D uint8 scales")
        R, cp = codes.shape
        if cols < 1 or cp != _round_up(cols, BLOCK) or tuple(scales.shape) != (R, _round_up(cp // BLOCK, 4)):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold {cols} columns")
        if scales.device != codes.device:
            raise ValueError("codes and scales lie on different devices")
        for t, name in ((codes, "codes"), (scales, "scales")):
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        self.codes, self.scales, self.shape, self.dtype = codes, scales, (R, int(cols)), dtype

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> Tensor:
        """The values held, rounded to ``dtype`` (fp32 and bf16 hold them exactly)."""
        R, cols = self.shape
        e = self.scales[:, :self.codes.shape[1] // BLOCK].to(torch.int32)
        # a byte of 0 stands for 2^-127, an fp32 subnormal
        s = torch.where(e > 0, e << 23, 1 << 22).view(torch.float32)
        v = self.codes.to(torch.float32).view(R, -1, BLOCK) * s.unsqueeze(-1)
        return v.view(R, -1)[:, :cols].to(dtype)


def _rows_2d(x: Tensor, name: str) -> Tensor:
    """x as the quantiser takes it: 2-D on the GPU, its rows contiguous (a row stride is kept)."""
    if x.dim() != 2:
        raise ValueError(f"{name} must be 2-D")
    if not x.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (the FP8 path has no CPU route)")
    _lib.float_code(x.dtype)
    if x.shape[1] > 1 and x.stride(1) != 1 or x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x


def _buffer(nbytes: int, device) -> Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _bias(bias: Optional[Tensor]):
    """(what has to live until the call, its address, its dtype code)"""
    if bias is None:
        return None, None, 0
    if not bias.is_contiguous():
        bias = bias.contiguous()
    return bias, bias.data_ptr(), _lib.float_code(bias.dtype)


def _quantize(x: Tensor, fmt: torch.dtype, tile: bool, cols: bool) -> Tuple[FP8Blocks, Optional[FP8Blocks]]:
    """(blocks along x's rows, with ``cols`` blocks of its transpose along its rows)."""
    f = _format(fmt)
    x = _rows_2d(x, "x")
    R, C = x.shape
    if R == 0 or C == 0:
        raise ValueError("FP8 blocks of an empty matrix")

    def blocks(r, c):
        cp = _round_up(c, BLOCK)
        return FP8Blocks(torch.empty((r, cp), dtype=fmt, device=x.device),
                         torch.empty((r, _round_up(cp // BLOCK, 4)), dtype=torch.uint8, device=x.device), c, x.dtype)

    with _lib.on(x.device):
        q, qt = blocks(R, C), blocks(C, R) if cols else None
        _lib.check(_lib.load().hif8_fp8_quantize(
            x.data_ptr(), _lib.float_code(x.dtype), R, C, max(x.stride(0), C), f, tile, q.codes.data_ptr(), q.scales.data_ptr(),
            qt.codes.data_ptr() if cols else None, qt.scales.data_ptr() if cols else None, None, 0, None, 0,
            _lib.stream_ptr(x.device)), "hif8_fp8_quantize")
    return q, qt


def fp8_quantize(x: Tensor, dtype: torch.dtype = torch.float8_e4m3fn, tile: bool = False) -> FP8Blocks:
    """A 2-D bf16, fp16 or fp32 x in FP8 blocks along its rows; ``tile``: one scale for each 128 x 128 values,
    as weights have it.  A block with an infinity or NaN becomes NaN."""
    return _quantize(x, dtype, tile, False)[0]


def fp8_quantize_both(x: Tensor, dtype: torch.dtype = torch.float8_e4m3fn,
                      tile: bool = False) -> Tuple[FP8Blocks, FP8Blocks]:
    """``fp8_quantize`` of x and of its transpose from one read of x."""
    return _quantize(x, dtype, tile, True)


def fp8_matmul(a: FP8Blocks, b: FP8Blocks, bias: Optional[Tensor] = None,
               out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """a [M, K] @ b [N, K]^T + bias -> [M, N], the matrix instruction's sums of 8 terms (see the head of this module: an
    fp32 result is 1e-5 to 5e-5 away from the exact one) added in fp32 and rounded once to ``out_dtype``."""
    (M, K), (N, Kb) = a.shape, b.shape
    if K != Kb:
        raise ValueError(f"a has {K} columns, b has {Kb}")
    if not a.codes.is_cuda:
        raise ValueError("fp8_matmul takes GPU operands (the FP8 path has no CPU route)")
    if a.device != b.device or (bias is not None and bias.device != a.device):
        raise ValueError("fp8_matmul: operands on different devices")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != N):
        raise ValueError(f"bias of shape {tuple(bias.shape)} for {N} output features")
    _lib.float_code(out_dtype)
    if M == 0 or N == 0:
        return torch.empty((M, N), dtype=out_dtype, device=a.device)
    L = _lib.load()
    with _lib.on(a.device):
        y = torch.empty((M, N), dtype=out_dtype, device=a.device)
        bias, bias_p, code = _bias(bias)
        nbytes = L.hif8_fp8_gemm_workspace_bytes(M, N, K)
        ws = _buffer(nbytes, a.device) if nbytes else None
        _lib.check(L.hif8_fp8_gemm(a.codes.data_ptr(), a.scales.data_ptr(), FORMATS[a.codes.dtype], b.codes.data_ptr(),
                                   b.scales.data_ptr(), FORMATS[b.codes.dtype], bias_p, code, y.data_ptr(),
                                   _lib.float_code(out_dtype), M, N, K, None if ws is None else ws.data_ptr(), nbytes,
                                   _lib.stream_ptr(a.device)), "hif8_fp8_gemm")
    return y


def _out_dtype(x: Tensor, weight) -> torch.dtype:
    return weight.dtype or x.dtype if x.dtype == torch.float32 else x.dtype


def _forward(x: Tensor, weight: Tensor, bias: Optional[Tensor], keep_x: bool, keep_w: bool):
    """(y, the blocks of x's transpose, of the weight's) of a weight that is quantised in the call."""
    N, K = weight.shape
    dev = x.device
    L = _lib.load()
    with _lib.on(dev):
        x2, w2 = _rows_2d(x if x.dim() == 2 else x.reshape(-1, K), "x"), _rows_2d(weight, "weight")
        M = x2.shape[0]
        out = _out_dtype(x, weight)
        y = torch.empty((M, N), dtype=out, device=dev)
        xt = _buffer(L.hif8_fp8_blocks_bytes(K, M), dev) if keep_x else None
        wt = _buffer(L.hif8_fp8_blocks_bytes(K, N), dev) if keep_w else None
        bias, bias_p, code = _bias(bias)
        nbytes = L.hif8_fp8_linear_fwd_workspace_bytes(M, N, K)
        ws = _buffer(nbytes, dev)
        _lib.check(L.hif8_fp8_linear_fwd(
            x2.data_ptr(), _lib.float_code(x2.dtype), max(x2.stride(0), K), w2.data_ptr(), _lib.float_code(w2.dtype),
            max(w2.stride(0), K), bias_p, code, y.data_ptr(), _lib.float_code(out), M, N, K,
            None if xt is None else xt.data_ptr(), None if wt is None else wt.data_ptr(), ws.data_ptr(), nbytes,
            _lib.stream_ptr(dev)), "hif8_fp8_linear_fwd")
    return (y if x.dim() == 2 else y.view(*x.shape[:-1], N)), xt, wt


class _FP8LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, grad_format):
        need_x, need_w, _ = ctx.needs_input_grad[:3]
        y, xt, wt = _forward(x, weight, bias, need_w, need_x)
        ctx.save_for_backward(xt, wt)
        ctx.rest = (*weight.shape, grad_format, x.shape, x.dtype, weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    def backward(ctx, gy):
        _lib.once(gy)
        N, K, fmt, x_shape, x_dtype, w_dtype, b_dtype = ctx.rest
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dev = gy.device
        xt, wt = ctx.saved_tensors
        L = _lib.load()
        with _lib.on(dev):
            g2 = _rows_2d(gy if gy.dim() == 2 else gy.reshape(-1, N), "grad")
            M = g2.shape[0]
            dx = torch.empty(x_shape, dtype=x_dtype, device=dev) if need_x else None
            dw = torch.empty((N, K), dtype=w_dtype, device=dev) if need_w else None
            db = torch.empty(N, dtype=b_dtype, device=dev) if need_b else None
            nbytes = L.hif8_fp8_linear_bwd_workspace_bytes(M, N, K)
            ws = _buffer(nbytes, dev)
            _lib.check(L.hif8_fp8_linear_bwd(
                g2.data_ptr(), _lib.float_code(g2.dtype), max(g2.stride(0), N), fmt, xt.data_ptr() if need_w else None,
                wt.data_ptr() if need_x else None, dx.data_ptr() if need_x else None, _lib.float_code(x_dtype),
                dw.data_ptr() if need_w else None, _lib.float_code(w_dtype), db.data_ptr() if need_b else None,
                _lib.float_code(b_dtype) if need_b else 0, M, N, K, ws.data_ptr(), nbytes, _lib.stream_ptr(dev)),
                "hif8_fp8_linear_bwd")
        return dx, dw, db, None


def fp8_linear(x: Tensor, weight, bias: Optional[Tensor] = None,
               grad_dtype: torch.dtype = torch.float8_e4m3fn) -> Tensor:
    """``x @ weight.T + bias`` in FP8 blocks, in x's dtype (bf16, fp16 or fp32).

    An fp32 x of a 16-bit weight (or blocks of one) gives the weight's type (the self-attention's o projection),
    with an fp32 dx.  The matrix instruction cuts small terms off, so that an fp32 result is 1e-5 to 5e-5 of its
    norm away from the exact product of the codes.

    ``weight`` [out, in] is a tensor, quantised in the call and differentiable, or the FP8Blocks that inference
    keeps (no gradient then).  ``grad_dtype``: the type of the gradient's codes in the backward pass.  Autocast
    changes nothing: the types are those of the operands."""
    fmt = _format(grad_dtype)
    _lib.float_code(x.dtype)
    packed = isinstance(weight, FP8Blocks)
    if x.dim() < 1 or len(weight.shape) != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} does not fit the weight {tuple(weight.shape)}")
    N, K = weight.shape
    dev = x.device
    if dev.type != "cuda":
        raise ValueError("x must be a GPU tensor (the FP8 path has no CPU route)")
    if dev != weight.device or (bias is not None and bias.device != dev):
        raise ValueError("fp8_linear: operands on different devices")
    if N == 0 or K == 0:
        raise ValueError(f"fp8_linear of an empty weight {tuple(weight.shape)}")
    if not packed:
        _lib.float_code(weight.dtype)
    if bias is not None:
        _lib.float_code(bias.dtype)
        if bias.dim() != 1 or bias.shape[0] != N:
            raise ValueError(f"bias of shape {tuple(bias.shape)} for {N} output features")
    if x.numel() == 0:                 # no rows: nothing to quantise
        out = _out_dtype(x, weight)
        w = x.new_zeros((N, K), dtype=out) if packed else weight.to(out)
        return torch.nn.functional.linear(x.to(out), w, None if bias is None else bias.to(out))
    if torch.is_grad_enabled() and (x.requires_grad or (not packed and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        if packed:
            raise RuntimeError("fp8_linear with a packed weight has no autograd; pass the weight tensor")
        return _FP8LinearFunction.apply(x, weight, bias, fmt)
    if not packed:
        return _forward(x, weight, bias, False, False)[0]
    L = _lib.load()
    with _lib.on(dev):
        # both steps in one call: 64 rows take 19 us, with a call each 22, of which the kernels take 10
        x2 = _rows_2d(x if x.dim() == 2 else x.reshape(-1, K), "x")
        M = x2.shape[0]
        out = _out_dtype(x, weight)
        y = torch.empty((M, N), dtype=out, device=dev)
        nbytes = L.hif8_fp8_linear_workspace_bytes(M, N, K)
        ws = _buffer(nbytes, dev)
        bias, bias_p, code = _bias(bias)
        _lib.check(L.hif8_fp8_linear(
            x2.data_ptr(), _lib.float_code(x2.dtype), max(x2.stride(0), K), weight.codes.data_ptr(), weight.scales.data_ptr(),
            FORMATS[weight.codes.dtype], bias_p, code, y.data_ptr(), _lib.float_code(out), M, N, K, ws.data_ptr(), nbytes,
            _lib.stream_ptr(dev)), "hif8_fp8_linear")
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


class FP8Linear(nn.Linear):
    """``nn.Linear`` on ``fp8_linear``.  ``prepack()`` keeps the weight's FP8 blocks for inference (with
    ``drop_weight`` in place of the weight); calls without gradients then take those, whatever becomes of the
    weight, until the next ``prepack()``, as with ``HIF8Linear``.  Without it they are made in every call, as
    training needs."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 grad_dtype: torch.dtype = torch.float8_e4m3fn, device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        _format(grad_dtype)
        self.grad_dtype = grad_dtype
        self._packed: Optional[FP8Blocks] = None

    @torch.no_grad()
    def prepack(self, drop_weight: bool = False) -> "FP8Linear":
        self._packed = fp8_quantize(self.weight.detach(), tile=True)
        if drop_weight:
            self.weight = nn.Parameter(torch.empty(0, device=self.weight.device, dtype=self.weight.dtype),
                                       requires_grad=False)
        return self

    def forward(self, x: Tensor) -> Tensor:
        w = self._packed
        if w is None or (torch.is_grad_enabled() and self.weight.numel()
                         and any(t is not None and t.requires_grad for t in (x, self.weight, self.bias))):
            w = self.weight
        return fp8_linear(x, w, self.bias, self.grad_dtype)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, grad_dtype={self.grad_dtype}"
