"""Linear layer with 4-bit weights, for the few tokens of a decoding step.

    y[m][n] = sum_k x[m][k] * (q[n][k] - zero[n][k // G]) * scale[n][k // G] + bias[n]

The serving form of the linear layers in front of a neuron (``triton_temporal_linear_lif_backend`` is the 16- and 32-bit
one): a token's layer is bound by the bytes of its weights, which are a quarter here. No counterpart in the reference.
Every call that is refused raises a ``RuntimeError`` that names the reason.
"""
from __future__ import annotations

from numbers import Integral
from typing import List, NamedTuple, Optional

import torch

from .. import _lib
from ._common import ACT_DTYPES, Gate, launch, raise_reasons, rows_2d

GROUP_SIZES = (32, 64, 128)


class W4Weight(NamedTuple):
    q_weight: torch.Tensor              # [N, K // 2] uint8, weight k in the low (k even) or high half of byte k // 2
    scales: torch.Tensor                # [N, ceil(K / G)]
    zeros: Optional[torch.Tensor]       # [N, ceil(K / G)] uint8 (at most 127, see run_linear_w4), None = 8


def quantize_linear_w4(weight: torch.Tensor, group_size: int = 128, symmetric: bool = True) -> W4Weight:
    """Rounds a [N, K] weight to 4 bits with a scale (and, if not ``symmetric``, a zero point) for each group of
    ``group_size`` values along K. Done once when a model is loaded; plain torch operations on the weight's device."""
    if not isinstance(weight, torch.Tensor):
        raise RuntimeError(f"weight is {type(weight).__name__}, expected a Tensor")
    if weight.dim() != 2 or weight.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise RuntimeError(f"unsupported_dtype: weight is {weight.dtype} with {weight.dim()} dimensions")
    N, K = weight.shape
    if not isinstance(group_size, Integral) or group_size not in GROUP_SIZES or K % 32 != 0 or K == 0:
        raise RuntimeError(f"unsupported_shape: K = {K} (a multiple of 32), groups of {group_size} (one of {GROUP_SIZES})")
    if not bool(torch.isfinite(weight).all()):
        raise RuntimeError("unsupported_value: weight has infinite values or NaN")
    group_size = int(group_size)
    groups = -(-K // group_size)
    w = torch.nn.functional.pad(weight.detach().float(), (0, groups * group_size - K)).view(N, groups, group_size)
    largest = w.abs().amax(-1)
    if symmetric:
        exact = largest / 7
        zero = torch.full_like(exact, 8.0)
    else:
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        exact = torch.where((hi - lo).isinf(), hi / 15 - lo / 15, (hi - lo) / 15)
        zero = None
    scale = exact.to(weight.dtype)
    # a subnormal scale may have lost up to all of itself to rounding: the next larger one then
    lost = (scale.float() < exact * (1 - 2.0 ** -7)) | ((scale == 0) & (largest > 0))
    smallest = torch.finfo(weight.dtype).tiny * torch.finfo(weight.dtype).eps
    scale = torch.where(lost, (scale.float() + smallest).to(weight.dtype), scale)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    if zero is None:
        zero = (-lo / scale.float()).round().clamp(0, 15)
    q = ((w / scale.float()[..., None]).round() + zero[..., None]).clamp(0, 15).to(torch.uint8)
    q = q.view(N, groups * group_size)[:, :K]
    packed = (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous()
    return W4Weight(packed, scale.contiguous(), None if symmetric else zero.to(torch.uint8).contiguous())


def check_linear_w4_support(x, q_weight, scales, zeros, bias, group_size) -> List[str]:
    """Reasons why the kernel cannot take this call (empty = it can)."""
    g = Gate("x", x)
    if not g:
        return g.why
    if x.dim() < 1:
        g.add("unsupported_rank", "x is a 0-dim tensor, the op is defined for rows of features")
        return g.why
    g.lead_is(rank=x.dim())
    K = int(x.shape[-1])
    if not isinstance(group_size, Integral) or group_size not in GROUP_SIZES:
        g.add("unsupported_group_size", f"groups of {group_size} values, one of {GROUP_SIZES} is implemented")
        return g.why
    if K == 0 or K % 32 != 0:
        g.add("unsupported_shape", f"x has {K} features, a multiple of 32 is implemented")
        return g.why

    def has(name, t, dtype, shape):
        if not isinstance(t, torch.Tensor):
            g.add("", f"{name} is {type(t).__name__}, expected a Tensor")
        elif tuple(t.shape) != shape:
            g.add("unsupported_shape", f"{name} is {tuple(t.shape)}, expected {shape}")
        elif t.dtype != dtype or t.device != x.device:
            g.add("unsupported_dtype", f"{name} is {t.dtype} on {t.device}, expected {dtype} on {x.device}")

    if not isinstance(q_weight, torch.Tensor) or q_weight.dim() != 2:
        g.add("unsupported_weight_rank", "q_weight must be a rank-2 tensor")
        return g.why
    N, groups = int(q_weight.shape[0]), -(-K // group_size)
    if N < 1:
        g.add("unsupported_shape", "q_weight has no rows")
    has("q_weight", q_weight, torch.uint8, (N, K // 2))
    has("scales", scales, x.dtype, (N, groups))
    if zeros is not None:
        has("zeros", zeros, torch.uint8, (N, groups))
    if bias is not None:
        has("bias", bias, x.dtype, (N,))
    return g.why


def _is_plain(x, q, s, z, b, group_size) -> bool:
    """Whether nothing needs a second look: what ``check_linear_w4_support`` would say yes to, at the price that a decoding
    step can pay. Anything else goes through the full check."""
    if not (type(x) is torch.Tensor and type(q) is torch.Tensor and type(s) is torch.Tensor and x.is_cuda and x.dim() >= 1
            and q.dim() == 2 and x.dtype in ACT_DTYPES and type(group_size) is int and group_size in GROUP_SIZES):
        return False
    K, (N, half), dtype, device = x.shape[-1], q.shape, x.dtype, x.device
    if not (K > 0 and K % 32 == 0 and 2 * half == K and N > 0 and q.dtype == torch.uint8 and s.dtype == dtype
            and q.device == device and s.device == device):
        return False
    groups = (N, -(-K // group_size))
    return (s.shape == groups
            and (z is None or (type(z) is torch.Tensor and z.shape == groups and z.dtype == torch.uint8 and z.device == device))
            and (b is None or (type(b) is torch.Tensor and b.shape == (N,) and b.dtype == dtype and b.device == device)))


def run_linear_w4(
    x: torch.Tensor,
    q_weight: torch.Tensor,
    scales: torch.Tensor,
    zeros: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    *,
    group_size: int = 128,
    out: Optional[torch.Tensor] = None,
    verbose: bool = False,
) -> torch.Tensor:
    """x [..., K] -> [..., N] in x's dtype. ``q_weight``, ``scales`` and ``zeros`` as ``quantize_linear_w4`` lays them out;
    keep them contiguous (they are copied at every call otherwise). A zero point above 127, which no 4-bit weight needs, makes
    its output infinite or NaN for bf16 and fp32 tokens. ``out``: a contiguous tensor to write into, apart from x."""
    if not _is_plain(x, q_weight, scales, zeros, bias, group_size):
        raise_reasons("linear_w4", check_linear_w4_support(x, q_weight, scales, zeros, bias, group_size), False, verbose)
    K, N = int(x.shape[-1]), int(q_weight.shape[0])
    shape = (*x.shape[:-1], N)
    if out is None:
        out = x.new_empty(shape)
    elif not isinstance(out, torch.Tensor) or tuple(out.shape) != shape or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
        raise RuntimeError(f"unsupported_output: out must be a contiguous {x.dtype} tensor of shape {shape} on {x.device}")
    M = x.numel() // K
    if M > 0:
        x2 = rows_2d(x)
        w, s = q_weight.contiguous(), scales.contiguous()
        if w.data_ptr() % 16:
            w = w.clone()
        z = zeros.contiguous() if zeros is not None else None
        b = bias.contiguous() if bias is not None else None
        launch("snnb_linear_w4", x.device, x2.data_ptr(), x2.stride(0), w.data_ptr(), s.data_ptr(), _lib.ptr(z),
               _lib.ptr(b), out.data_ptr(), N, M, K, N, int(group_size), _lib.dtype_code(x.dtype))
    return out
