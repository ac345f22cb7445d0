"""The norms around a block fused with its gate and residual scale, forward and backward.

    n       = y / sqrt(mean(y^2) + eps) * w_post          (post_norm=False: n = y)
    res_out = residual + alpha * res_scale * act(gate) * n
    z       = res_out / sqrt(mean(res_out^2) + eps) * w_pre

One pass over the rows does what follows a block (its norm, gate and residual) and what precedes the next one (that
block's norm). No counterpart in the reference, whose BatchNorm is folded into the convolutions. Every call that is
refused raises a ``RuntimeError`` that names the reason. The gradients are a second call (``run_block_norm_backward``);
nothing here is recorded by autograd.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional

import torch

from .. import _lib
from ._common import ACT_DTYPES, Gate, dense_like, launch, raise_reasons, rows_2d

ACTS = {"none": _lib.ACT_NONE, "sigmoid": _lib.ACT_SIGMOID, "silu": _lib.ACT_SILU}
MAX_D = 16384


class BlockNormResult(NamedTuple):
    res_out: Optional[torch.Tensor]
    z: Optional[torch.Tensor]


class BlockNormGradients(NamedTuple):
    dy: Optional[torch.Tensor]
    dgate: Optional[torch.Tensor]
    dresidual: torch.Tensor
    dw_post: Optional[torch.Tensor]
    dres_scale: Optional[torch.Tensor]
    dw_pre: Optional[torch.Tensor]


def _number(v) -> Optional[float]:
    try:
        return None if isinstance(v, str) else float(v)
    except (TypeError, ValueError, RuntimeError):       # the last: a tensor of several values
        return None


def check_block_norm_support(y, gate, residual, w_post, res_scale, w_pre, gate_act, post_norm, pre_norm, eps, alpha=1.0,
                             **more) -> List[str]:
    """Reasons why the kernel cannot take this call (empty = it can). ``more``: further row tensors by name."""
    name, lead = ("y", y) if y is not None else ("residual", residual)
    g = Gate(name, lead)
    if not g:
        return g.why
    if lead.dim() < 1:
        g.add("unsupported_rank", f"{name} is a 0-dim tensor, the op is defined for rows of values")
        return g.why
    g.lead_is(rank=lead.dim())
    shape, D = lead.shape, int(lead.shape[-1])
    if not 1 <= D <= MAX_D:
        g.add("unsupported_shape", f"rows of {D} values, 1 to {MAX_D} are implemented")
    if not isinstance(gate_act, str) or gate_act not in ACTS:
        g.add("unsupported_gate", f"gate_act is {gate_act!r}, one of {sorted(ACTS)}")
    elif (gate is None) != (gate_act == "none"):
        g.add("unsupported_gate", f"gate_act is {gate_act!r} {'without a' if gate is None else 'with a'} gate")
    if y is None and (gate is not None or w_post is not None or res_scale is not None or post_norm):
        g.add("unsupported_form", "gate, w_post, res_scale and post_norm belong to y, which is None")
    if w_post is not None and not post_norm:
        g.add("unsupported_form", "w_post is given although post_norm is off")
    if w_pre is not None and not pre_norm:
        g.add("unsupported_form", "w_pre is given although pre_norm is off")
    number = _number(eps)
    if number is None or not number >= 0.0:
        g.add("unsupported_eps", f"eps is {eps}")
    if _number(alpha) is None:
        g.add("unsupported_alpha", f"alpha is {alpha}")
    for n, t in (("gate", gate), ("residual", residual), *more.items()):
        if t is None or t is lead:
            continue
        if not isinstance(t, torch.Tensor):
            g.add("", f"{n} is {type(t).__name__}, expected a Tensor")
        elif t.shape != shape:
            g.add("unsupported_shape", f"{n} is {tuple(t.shape)} while {name} is {tuple(shape)}")
        elif t.dtype != lead.dtype or t.device != lead.device:
            g.add("unsupported_dtype", f"{n} is {t.dtype} on {t.device} while {name} is {lead.dtype} on {lead.device}")
    w_dtype = None
    for n, t in (("w_post", w_post), ("res_scale", res_scale), ("w_pre", w_pre)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            g.add("", f"{n} is {type(t).__name__}, expected a Tensor")
        elif tuple(t.shape) != (D,):
            g.add("unsupported_shape", f"{n} is {tuple(t.shape)}, one value per column would be ({D},)")
        elif t.dtype not in (lead.dtype, torch.float32) or t.device != lead.device or t.dtype != (w_dtype or t.dtype):
            g.add("unsupported_dtype", f"{n} is {t.dtype} on {t.device}; the parameters share {lead.dtype} or torch.float32 "
                                       f"on {lead.device}")
        else:
            w_dtype = t.dtype
    return g.why


def _is_plain(y, rows, params, gate, w_post, w_pre, gate_act, post_norm, pre_norm, eps, alpha) -> bool:
    """Whether nothing needs a second look: what ``check_block_norm_support`` would say yes to, at the price that a decoding
    step can pay. Anything else goes through the full check."""
    if not (type(y) is torch.Tensor and y.is_cuda and y.dim() >= 1 and y.dtype in ACT_DTYPES
            and type(eps) in (float, int) and eps >= 0.0 and type(alpha) in (float, int)
            and type(gate_act) is str and (gate is None) == (gate_act == "none") and gate_act in ACTS
            and (post_norm or w_post is None) and (pre_norm or w_pre is None)):
        return False
    shape, dtype, device = y.shape, y.dtype, y.device
    D = shape[-1]
    if not 1 <= D <= MAX_D:
        return False
    for t in rows:
        if t is not None and not (type(t) is torch.Tensor and t.shape == shape and t.dtype == dtype and t.device == device):
            return False
    for w in params:
        if w is not None and not (type(w) is torch.Tensor and w.shape == (D,) and w.dtype == dtype and w.device == device):
            return False
    return True


def _params(lead, *ws):
    ws = [w.contiguous() if w is not None else None for w in ws]
    dtype = next((w.dtype for w in ws if w is not None), lead.dtype)
    return ws, _lib.dtype_code(dtype)


def _rows(t):
    """[..., D] -> (rows tensor kept alive, address, row stride)."""
    if t is None:
        return None, None, 0
    r = t if t.dim() == 2 and t.stride(1) == 1 else rows_2d(t)
    return r, r.data_ptr(), r.stride(0)


def run_block_norm(
    y: Optional[torch.Tensor],
    *,
    gate: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    w_post: Optional[torch.Tensor] = None,
    res_scale: Optional[torch.Tensor] = None,
    w_pre: Optional[torch.Tensor] = None,
    gate_act: str = "none",
    alpha: float = 1.0,
    post_norm: bool = True,
    pre_norm: bool = True,
    eps: float = 1e-6,
    res_inplace: bool = False,
    verbose: bool = False,
) -> BlockNormResult:
    """y, gate, residual [..., D] -> res_out and z (None without ``pre_norm``) of that shape, dense.

    ``y=None`` (with ``post_norm=False``) is the norm in front of the first block: z alone, res_out is None. ``residual``,
    ``w_post``, ``res_scale`` and ``w_pre`` may be None (zeros, ones, ones, ones); the parameters are [D] in y's dtype or
    fp32. ``res_inplace`` writes res_out over ``residual``, which must be contiguous and share no
    memory with y or gate then.
    """
    if not _is_plain(y, (gate, residual), (w_post, res_scale, w_pre), gate, w_post, w_pre, gate_act, post_norm, pre_norm, eps,
                     alpha):
        raise_reasons("block_norm", check_block_norm_support(y, gate, residual, w_post, res_scale, w_pre, gate_act, post_norm,
                                                             pre_norm, eps, alpha), False, verbose)
    lead = y if y is not None else residual
    if y is None and not pre_norm:
        raise RuntimeError("unsupported_form: neither y nor pre_norm, nothing to compute")
    if res_inplace and (y is None or residual is None or not residual.is_contiguous()):
        raise RuntimeError("unsupported_output: res_inplace needs y and a contiguous residual")
    D = int(lead.shape[-1])
    M = lead.numel() // D
    res_out = None
    if y is not None:
        res_out = residual if res_inplace else dense_like(lead)
    z = dense_like(lead) if pre_norm else None
    (w_post, res_scale, w_pre), w_code = _params(lead, w_post, res_scale, w_pre)
    if M > 0:
        y2, yp, ys = _rows(y)
        g2, gp, gs = _rows(gate)
        r2, rp, rs = _rows(residual)
        launch("snnb_block_norm", lead.device, yp, ys, gp, gs, rp, rs, _lib.ptr(w_post), _lib.ptr(res_scale),
               _lib.ptr(w_pre), _lib.ptr(res_out), _lib.ptr(z), M, D, float(alpha), float(eps), ACTS[gate_act],
               int(bool(post_norm)), _lib.dtype_code(lead.dtype), w_code)
    return BlockNormResult(res_out, z)


def run_block_norm_backward(
    dres_out: Optional[torch.Tensor],
    dz: Optional[torch.Tensor],
    y: Optional[torch.Tensor],
    *,
    gate: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    w_post: Optional[torch.Tensor] = None,
    res_scale: Optional[torch.Tensor] = None,
    w_pre: Optional[torch.Tensor] = None,
    gate_act: str = "none",
    alpha: float = 1.0,
    post_norm: bool = True,
    pre_norm: bool = True,
    eps: float = 1e-6,
    verbose: bool = False,
) -> BlockNormGradients:
    """Gradients for dres_out (of res_out) and dz (of z); one of them may be None (zeros), and dz is None without
    ``pre_norm``. The other arguments are those of the forward call, ``residual`` as it was before it.

    dy, dgate and dresidual are dense in y's dtype; the parameters' gradients are fp32, summed over the rows in a fixed
    order, and None for a parameter that is None.
    """
    if (dres_out is None and dz is None) or (dz is not None and not pre_norm) or not _is_plain(
            y, (gate, residual, dres_out, dz), (w_post, res_scale, w_pre), gate, w_post, w_pre, gate_act, post_norm, pre_norm, eps,
            alpha):
        why = check_block_norm_support(y, gate, residual, w_post, res_scale, w_pre, gate_act, post_norm, pre_norm, eps, alpha,
                                       dres_out=dres_out, dz=dz)
        if dres_out is None and dz is None:
            why.append("unsupported_form: neither dres_out nor dz")
        if dz is not None and not pre_norm:
            why.append("unsupported_form: dz is given although pre_norm is off")
        raise_reasons("block_norm_backward", why, False, verbose)
    lead = y if y is not None else residual
    D = int(lead.shape[-1])
    M = lead.numel() // D

    dy, dgate = dense_like(lead) if y is not None else None, dense_like(lead) if gate is not None else None
    dres = dense_like(lead)
    # without rows, or without a gradient of z, a sum is empty
    sums = (lead.new_empty if M > 0 and dz is not None else lead.new_zeros)((3, D), dtype=torch.float32).unbind(0)
    dw_post, dscale, dw_pre = (s if w is not None else None for s, w in zip(sums, (w_post, res_scale, w_pre)))
    if M > 0:
        (wp, sc, wr), w_code = _params(lead, w_post, res_scale, w_pre)
        ws = lead.new_empty(_lib.lib.snnb_block_norm_backward_workspace_bytes(M, D), dtype=torch.uint8)
        k0, dop, dos = _rows(dres_out)
        k1, dzp, dzs = _rows(dz)
        k2, yp, ys = _rows(y)
        k3, gp, gs = _rows(gate)
        k4, rp, rs = _rows(residual)
        has_z = dz is not None
        launch("snnb_block_norm_backward", lead.device, dop, dos, dzp, dzs, yp, ys, gp, gs, rp, rs,
               _lib.ptr(wp), _lib.ptr(sc), _lib.ptr(wr) if has_z else None, _lib.ptr(dy), _lib.ptr(dgate), _lib.ptr(dres),
               _lib.ptr(dw_post), _lib.ptr(dscale), _lib.ptr(dw_pre) if has_z else None, ws.data_ptr(), ws.numel(), M, D,
               float(alpha), float(eps), ACTS[gate_act], int(bool(post_norm)), _lib.dtype_code(lead.dtype), w_code)
    return BlockNormGradients(dy, dgate, dres, dw_post, dscale, dw_pre)
