"""Producer fusion for the modulated LayerNorm in front of q/k/v and the FFN.

``block_forward`` (``ospnext/modules/osp_next.py:937-957``) feeds its self-attention and FFN
with ``norm(x) * (1 + e[1]) + e[0]`` and ``norm(x) * (1 + e[4]) + e[3]``, ``norm`` the
WanLayerNorm (``ospnext/modules/want2v.py:96-106``); every consuming HIF8Linear then runs
``_quant`` on that tensor (``hif8_linear.py:42-50``), so q, k and v quantise the same input
three times.  ``modulated_norm_quant`` produces the quantised input directly, in two passes
over x (``hif8_modln_amax`` and ``hif8_modln_fake_quant``), and ``qkv_from_modulated_norm``
feeds it to the three projections with one quantisation.  ``affine_norm_quant`` does the same
for the affine LayerNorm (norm3) in front of the cross-attention's q projection.

The fused route is inference-only (no autograd through the producer) and takes bf16 x with
``dim % 8 == 0`` and ``dim <= 8192``; anything else runs the reference's op sequence with the
library's ``_quant`` on the GPU.

``layer_norm`` and ``modulated_layer_norm`` are the norms with gradients, in one pass forward and one
backward: what a training step runs in place of the fp32 op sequence.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from . import _lib
from .hif8_linear import (GroupedWeight, HIF8Linear, QuantState, absmax_scale, fake_quant, grouped_ok,
                          linear_fwd_grouped)

MAX_DIM = 8192


class WanLayerNorm(nn.LayerNorm):
    """want2v.py:96-106: fp32 layer norm over the last dim, cast back to the input dtype."""

    def __init__(self, dim: int, eps: float = 1e-6, elementwise_affine: bool = False):
        super().__init__(dim, elementwise_affine=elementwise_affine, eps=eps)

    def forward(self, x: Tensor) -> Tensor:
        return super().forward(x.float()).type_as(x)


def modulate(n: Tensor, shift: Optional[Tensor], scale: Optional[Tensor]) -> Tensor:
    """``n * (1 + scale) + shift`` as block_forward writes it (osp_next.py:941, :954)."""
    y = n if scale is None else n * (1 + scale)
    return y if shift is None else y + shift


def _modulation_rows(t: Optional[Tensor], x: Tensor, name: str) -> Tuple[Optional[Tensor], int]:
    """[B, 1, D] / [B, D] / [1, D] / [D] modulation -> contiguous [batches, D] and rows per batch."""
    if t is None:
        return None, 0
    D = x.shape[-1]
    if t.shape[-1] != D:
        raise ValueError(f"{name} has last dim {t.shape[-1]}, x has {D}")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16 like x, got {t.dtype}")
    t2 = t.reshape(-1, D)
    batches = t2.shape[0]
    rows = x.numel() // D
    if batches == 1:
        rpb = rows
    else:
        if x.dim() < 3 or x.shape[0] != batches or any(s != 1 for s in t.shape[1:-1]):
            raise ValueError(f"{name} of shape {tuple(t.shape)} does not broadcast per batch over x {tuple(x.shape)}")
        rpb = rows // batches
    return t2.contiguous(), rpb


def fused_ok(x: Tensor) -> bool:
    return (x.is_cuda and x.dtype == torch.bfloat16 and x.dim() >= 1 and x.numel() > 0
            and x.shape[-1] % 8 == 0 and x.shape[-1] <= MAX_DIM)


def modulated_norm_quant(x: Tensor, shift: Optional[Tensor] = None, scale: Optional[Tensor] = None,
                         eps: float = 1e-6, scale_max: float = 15.0, semantics: int = _lib.SEM_NPU,
                         return_y: bool = False):
    """x_q = _quant(WanLayerNorm(x) * (1 + scale) + shift)[0] in bf16, the input every HIF8Linear
    fed by this modulated norm quantises to.  Returns ``(x_q, state)`` (``state`` holds amax,
    scale and decode tables of y), plus y itself with ``return_y``."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, shift, scale)):
        raise RuntimeError("modulated_norm_quant has no autograd; use WanLayerNorm, modulate and "
                           "HIF8Linear.forward when gradients are needed")
    if not fused_ok(x):
        y = modulate(WanLayerNorm(x.shape[-1], eps).to(x.device)(x), shift, scale).contiguous()
        st = absmax_scale(y, scale_max, QuantState(y.device))
        xq = fake_quant(y, st, semantics)
        return (xq, st, y) if return_y else (xq, st)
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    D = x.shape[-1]
    rows = x.numel() // D
    sh, rpb_s = _modulation_rows(shift, x, "shift")
    sc, rpb_c = _modulation_rows(scale, x, "scale")
    if sh is not None and sc is not None and rpb_s != rpb_c:
        raise ValueError("shift and scale have different batch counts")
    rpb = rpb_s or rpb_c or rows
    stats = torch.empty(rows * 2, dtype=torch.float32, device=x.device)
    st = QuantState(x.device)
    L = _lib.load()
    s = _lib.stream_ptr(x.device)
    sh_p = sh.data_ptr() if sh is not None else None
    sc_p = sc.data_ptr() if sc is not None else None
    _lib.check(L.hif8_modln_amax(x.data_ptr(), sh_p, sc_p, rows, D, rpb, float(eps), stats.data_ptr(),
                                 float(scale_max), st.ptr, s), "hif8_modln_amax")
    xq = torch.empty_like(x)
    y = torch.empty_like(x) if return_y else None
    _lib.check(L.hif8_modln_fake_quant(x.data_ptr(), sh_p, sc_p, rows, D, rpb, stats.data_ptr(), st.ptr,
                                       int(semantics), xq.data_ptr(), y.data_ptr() if y is not None else None, s),
               "hif8_modln_fake_quant")
    return (xq, st, y) if return_y else (xq, st)


STATIC_MAX_ROWS = 131072


def modulated_norm_quant_static(x: Tensor, shift: Optional[Tensor] = None, scale: Optional[Tensor] = None,
                                eps: float = 1e-6, scale_max: float = 15.0, semantics: int = _lib.SEM_NPU) -> Tensor:
    """``modulated_norm_quant(x, shift, scale, eps, scale_max)[0]`` through the allocation-free entry
    point ``hif8_modln_quant_static``: the row statistics and the state live in the library's static
    device workspace (at most STATIC_MAX_ROWS rows), so the library allocates nothing; only x_q is
    returned (it has no state object).  Calls overlapping on one GPU race on that workspace."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, shift, scale)):
        raise RuntimeError("modulated_norm_quant_static has no autograd")
    if not fused_ok(x):
        raise ValueError("modulated_norm_quant_static takes bf16 CUDA x with dim % 8 == 0 and dim <= 8192")
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    D = x.shape[-1]
    rows = x.numel() // D
    sh, rpb_s = _modulation_rows(shift, x, "shift")
    sc, rpb_c = _modulation_rows(scale, x, "scale")
    if sh is not None and sc is not None and rpb_s != rpb_c:
        raise ValueError("shift and scale have different batch counts")
    rpb = rpb_s or rpb_c or rows
    xq = torch.empty_like(x)
    _lib.check(_lib.load().hif8_modln_quant_static(x.data_ptr(), sh.data_ptr() if sh is not None else None,
                                                   sc.data_ptr() if sc is not None else None, rows, D, rpb, float(eps),
                                                   float(scale_max), int(semantics), xq.data_ptr(),
                                                   _lib.stream_ptr(x.device)), "hif8_modln_quant_static")
    return xq


AFFINE_MAX_DIM = 6144


def affine_fused_ok(x: Tensor, norm: nn.Module) -> bool:
    """The fused affine producer takes bf16 CUDA x with dim % 8 == 0, dim <= 6144, and a
    WanLayerNorm with fp32 weight and bias."""
    w, b = getattr(norm, "weight", None), getattr(norm, "bias", None)
    return (fused_ok(x) and x.shape[-1] <= AFFINE_MAX_DIM and isinstance(norm, nn.LayerNorm)
            and w is not None and b is not None and w.dtype == torch.float32 and b.dtype == torch.float32
            and tuple(norm.normalized_shape) == (x.shape[-1],) and w.device == x.device)


def affine_norm_quant(x: Tensor, norm: nn.Module, scale_max: float = 15.0, semantics: int = _lib.SEM_NPU,
                      return_y: bool = False):
    """x_q = _quant(norm(x))[0] in bf16 for the affine WanLayerNorm ``norm`` (norm3,
    osp_next.py:860-864, 949-951): the input the cross-attention's q projection quantises.
    Returns ``(x_q, state)``, plus y = norm(x) with ``return_y``.  Two passes over x
    (``hif8_ln_affine_amax`` and ``hif8_ln_affine_fake_quant``); other shapes and dtypes run
    the module and the library's ``_quant`` on the GPU."""
    if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in norm.parameters())):
        raise RuntimeError("affine_norm_quant has no autograd; use the norm module and HIF8Linear.forward "
                           "when gradients are needed")
    if not affine_fused_ok(x, norm):
        y = norm(x).contiguous()
        st = absmax_scale(y, scale_max, QuantState(y.device))
        xq = fake_quant(y, st, semantics)
        return (xq, st, y) if return_y else (xq, st)
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    w = norm.weight.detach().contiguous()
    b = norm.bias.detach().contiguous()
    D = x.shape[-1]
    rows = x.numel() // D
    stats = torch.empty(rows * 2, dtype=torch.float32, device=x.device)
    st = QuantState(x.device)
    L = _lib.load()
    s = _lib.stream_ptr(x.device)
    _lib.check(L.hif8_ln_affine_amax(x.data_ptr(), w.data_ptr(), b.data_ptr(), rows, D, float(norm.eps),
                                     stats.data_ptr(), float(scale_max), st.ptr, s), "hif8_ln_affine_amax")
    xq = torch.empty_like(x)
    y = torch.empty_like(x) if return_y else None
    _lib.check(L.hif8_ln_affine_fake_quant(x.data_ptr(), w.data_ptr(), b.data_ptr(), rows, D, stats.data_ptr(),
                                           st.ptr, int(semantics), xq.data_ptr(),
                                           y.data_ptr() if y is not None else None, s),
               "hif8_ln_affine_fake_quant")
    return (xq, st, y) if return_y else (xq, st)


def qkv_from_modulated_norm(x: Tensor, shift: Optional[Tensor], scale: Optional[Tensor], q: HIF8Linear,
                            k: HIF8Linear, v: HIF8Linear, eps: float = 1e-6) -> Tuple[Tensor, Tensor, Tensor]:
    """``q(y), k(y), v(y)`` for ``y = norm(x) * (1 + scale) + shift`` (osp_next.py:742-744 fed by :941)
    with y quantised once and the three products in one grouped launch when the shapes allow
    (each output bit-identical to the layer's own forward).  Inference only; the three layers
    must share ``scale_max_forward``."""
    smf = q.scale_max_forward
    if k.scale_max_forward != smf or v.scale_max_forward != smf:
        raise ValueError("q, k and v quantise their input with different scale_max_forward")
    xq, _ = modulated_norm_quant(x, shift, scale, eps, smf)
    gw = grouped_weight((q, k, v))
    if gw is None:
        return q.forward_quantized(xq), k.forward_quantized(xq), v.forward_quantized(xq)
    K = xq.shape[-1]
    ys = linear_fwd_grouped(xq.reshape(-1, K).contiguous(), gw)
    return tuple(y.view(*xq.shape[:-1], y.shape[-1]) for y in ys)


def grouped_weight(layers) -> Optional[GroupedWeight]:
    """The layers' weights concatenated for one grouped launch (cached on the first layer and
    rebuilt when any packed weight or bias changes), or None when they do not fit one."""
    packs = [m._packed_weight() for m in layers]
    if not grouped_ok(packs):
        return None
    key = tuple((id(p), None if m.bias is None else (m.bias.data_ptr(), m.bias._version))
                for p, m in zip(packs, layers))
    cached = getattr(layers[0], "_grouped_cache", None)
    if cached is not None and cached.key == key:
        return cached
    gw = GroupedWeight(packs, [m.bias for m in layers], key)
    layers[0]._grouped_cache = gw
    return gw


# ------------------------------------------------------------- with gradients


MAX_GROUPS = 65535            # of the entry points: a grid's second dimension


class _LayerNormFunction(torch.autograd.Function):
    """y = norm(x) * w + b over x's last dim; weight and bias hold ``groups`` rows of D (in any shape, with one
    row stride) or are None; ``plus``: w = 1 + weight."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps: float, plus: bool, groups: int):
        D = x.shape[-1]
        if not x.is_contiguous():
            x = x.contiguous()
        rows = x.numel() // D
        # the modulation's rows of a [B, 6, D] tensor are taken as they lie
        ld = D
        wp = bp = None
        code = 0
        given = weight if weight is not None else bias
        if given is not None:
            code = _lib.float_code(given.dtype)
            ld = given.stride(0) if groups > 1 else D
            for t in (weight, bias):
                if t is not None and (t.stride(-1) != 1 or (groups > 1 and (t.stride(0) != ld or ld < D))):
                    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
                    ld = D
                    break
            wp = None if weight is None else weight.data_ptr()
            bp = None if bias is None else bias.data_ptr()
        need = ctx.needs_input_grad
        keep = need[0] or need[1] or need[2]
        y = torch.empty_like(x)
        stats = torch.empty(rows * 2, dtype=torch.float32, device=x.device) if keep else None
        with _lib.on(x.device):
            _lib.check(_lib.load().hif8_layer_norm_fwd(
                x.data_ptr(), _lib.float_code(x.dtype), rows, D, groups, wp, bp, code, ld, plus, eps, y.data_ptr(),
                stats.data_ptr() if keep else None, _lib.stream_ptr(x.device)), "hif8_layer_norm_fwd")
        if keep:
            ctx.save_for_backward(x, weight, stats)
            ctx.rest = (rows, D, groups, ld, code, plus, None if weight is None else weight.shape,
                        None if bias is None else (bias.shape, bias.dtype))
        return y

    @staticmethod
    def backward(ctx, dy):
        _lib.once(dy)
        x, weight, stats = ctx.saved_tensors
        rows, D, groups, ld, code, plus, w_shape, b_info = ctx.rest
        if not dy.is_contiguous():
            dy = dy.contiguous()
        L = _lib.load()
        dev = x.device
        _, need_w, need_b = ctx.needs_input_grad[:3]
        with _lib.on(dev):
            dx = torch.empty_like(x)
            dw = torch.empty(w_shape, dtype=weight.dtype, device=dev) if need_w else None
            db = torch.empty(b_info[0], dtype=b_info[1], device=dev) if need_b else None
            ws, nbytes = None, 0
            if need_w or need_b:
                nbytes = L.hif8_layer_norm_bwd_workspace_bytes(rows, D, groups)
                ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            _lib.check(L.hif8_layer_norm_bwd(
                dy.data_ptr(), x.data_ptr(), _lib.float_code(x.dtype), rows, D, groups,
                None if weight is None else weight.data_ptr(), code, ld, plus, stats.data_ptr(), dx.data_ptr(),
                None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(),
                None if ws is None else ws.data_ptr(), nbytes, _lib.stream_ptr(dev)), "hif8_layer_norm_bwd")
        return dx, dw, db, None, None, None


def _norm_rows(x: Tensor, given, eps: float) -> int:
    """Checks of what both norms take; returns D."""
    _lib.float_code(x.dtype)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_DIM:
        raise ValueError(f"the norm takes a last dim of 1 to {MAX_DIM}, got x of shape {tuple(x.shape)}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    D = x.shape[-1]
    for name, t in given:
        if t is None:
            continue
        _lib.float_code(t.dtype)
        if t.dim() < 1 or t.shape[-1] != D:
            raise ValueError(f"{name} of shape {tuple(t.shape)} does not fit x {tuple(x.shape)}")
        if t.device != x.device:
            raise ValueError(f"{name} and x lie on different devices")
    if len({t.dtype for _, t in given if t is not None}) > 1:
        raise TypeError(" and ".join(name for name, _ in given) + " differ in dtype")
    if not x.is_cuda:
        raise ValueError("x must be a GPU tensor (the norm has no CPU route)")
    return D


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-6) -> Tensor:
    """LayerNorm over the last dim, as ``WanLayerNorm`` (want2v.py:96-106) computes it: fp32 statistics and
    arithmetic, rounded once to x's dtype (bf16, fp16 or fp32).  ``weight`` and ``bias`` [D] may have another
    dtype than x.  Differentiable; the gradients of weight and bias are summed in fp32 over all rows."""
    D = _norm_rows(x, (("weight", weight), ("bias", bias)), eps)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.dim() != 1:
            raise ValueError(f"{name} must have the shape [{D}], got {tuple(t.shape)}")
    if x.numel() == 0:
        y = x * 1.0 if weight is None else (x * weight).to(x.dtype)
        return y if bias is None else (y + bias).to(x.dtype)
    return _LayerNormFunction.apply(x, weight, bias, float(eps), False, 1)


def modulated_layer_norm(x: Tensor, shift: Optional[Tensor] = None, scale: Optional[Tensor] = None,
                         eps: float = 1e-6) -> Tensor:
    """``norm(x) * (1 + scale) + shift`` (osp_next.py:941, :954) with gradients for x, shift and scale, in fp32
    arithmetic and rounded once to x's dtype.  ``shift`` and ``scale`` are [D], or [B, 1, D] (as many ones as x
    has dims between) for x [B, ..., D], rows of a larger tensor included; their gradients are summed in fp32
    over a batch entry's rows.  More than 65535 entries are done in parts, which are put together by a copy."""
    D = _norm_rows(x, (("shift", shift), ("scale", scale)), eps)
    counts = [1, 1]
    for i, (name, t) in enumerate((("shift", shift), ("scale", scale))):
        if t is not None:
            counts[i] = n = t.numel() // D
            if n != 1 and (x.dim() < 2 or t.shape[0] != x.shape[0] or n != x.shape[0] or any(s != 1 for s in t.shape[1:-1])):
                raise ValueError(f"{name} of shape {tuple(t.shape)} does not broadcast per batch over x {tuple(x.shape)}")
    if x.numel() == 0:
        return (x * sum((t.sum() * 0 for t in (shift, scale) if t is not None), 1.0)).to(x.dtype)
    groups = max(counts)
    if groups > 1:       # one for all entries beside one for each: a row for each, whose gradients torch adds up
        shift, scale = (t if t is None or n == groups else t.reshape(1, D).expand(groups, D)
                        for t, n in zip((shift, scale), counts))
    if groups > MAX_GROUPS:
        parts = zip(*((None,) * -(-groups // MAX_GROUPS) if t is None else t.split(MAX_GROUPS) for t in (x, shift, scale)))
        return torch.cat([modulated_layer_norm(*part, eps) for part in parts])
    return _LayerNormFunction.apply(x, scale, shift, float(eps), True, groups)
