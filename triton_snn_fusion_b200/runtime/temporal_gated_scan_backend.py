"""Gated linear recurrence over time, forward and backward.

The leaky charge step of a LIF neuron without the spike, with the leak given per step and channel:

    a_t = sigmoid(gate_t) (``gate="sigmoid"``) or gate_t (``gate="value"``)
    h_t = a_t * h_{t-1} + (1 - a_t) * x_t (``leaky=True``) or a_t * h_{t-1} + x_t

No counterpart in the reference; the call conventions are those of the LIF scan (``triton_temporal_lif_backend``): a
carried state in and out, fp32 arithmetic inside, a ``RuntimeError`` that names the reason for every call that is
refused. One call over the whole sequence trains or prefills, a call with one step decodes. The gradients are a second
call (``run_temporal_gated_scan_backward``); nothing here is recorded by autograd.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional

import torch

from .. import _lib
from ._common import ACT_DTYPES, Gate, dense_like, launch, raise_reasons, rows_dense, state_or_none

GATES = {"value": _lib.GATE_VALUE, "sigmoid": _lib.GATE_SIGMOID}


class TemporalGatedScanResult(NamedTuple):
    h_seq: torch.Tensor
    h_last: torch.Tensor
    ckpt: Optional[torch.Tensor] = None     # states for the backward pass (save_for_backward=True)


class TemporalGatedScanGradients(NamedTuple):
    dx: torch.Tensor
    dgate: torch.Tensor
    dh_init: torch.Tensor


def _sizes(x_seq, batch_first):
    return (x_seq.shape[1], x_seq.shape[0], x_seq.shape[2]) if batch_first else tuple(x_seq.shape)


def _like(g: Gate, name: str, t, shape, dtype=None) -> None:
    if not isinstance(t, torch.Tensor):
        g.add("", f"{name} is {type(t).__name__}, expected a Tensor")
    elif tuple(t.shape) != tuple(shape):
        g.add("unsupported_shape", f"{name} is {tuple(t.shape)}, expected {tuple(shape)}")
    elif t.dtype != (dtype or g.lead.dtype) or t.device != g.lead.device:
        g.add("unsupported_dtype", f"{name} is {t.dtype} on {t.device}, expected {dtype or g.lead.dtype} on {g.lead.device}")


def _state(g: Gate, name: str, t):
    """A carried state, None where the call starts from zeros."""
    if t is not None and not isinstance(t, torch.Tensor):
        g.add("", f"{name} is {type(t).__name__}, expected a Tensor (0-dim or None for zeros)")
    return state_or_none(t)


def check_temporal_gated_scan_support(x_seq, gate_seq, h_init, gate, lengths=None, batch_first=False,
                                      state_dtype=None) -> List[str]:
    """Reasons why the scan cannot take this call (empty = it can)."""
    g = Gate("x_seq", x_seq)
    if not g:
        return g.why
    g.lead_is(rank=3)
    if not isinstance(gate, str) or gate not in GATES:
        g.add("unsupported_gate", f"gate is {gate!r}, one of {sorted(GATES)}")
    if x_seq.dim() == 3:
        _like(g, "gate_seq", gate_seq, x_seq.shape)
        _, B, D = _sizes(x_seq, batch_first)
        if state_dtype is not None and state_dtype not in (x_seq.dtype, torch.float32):
            g.add("unsupported_dtype", f"state_dtype is {state_dtype}, the state is {x_seq.dtype} or torch.float32")
        h0 = _state(g, "h_init", h_init)
        if h0 is not None:
            _like(g, "h_init", h0, (B, D), h0.dtype)
            if h0.dtype not in (x_seq.dtype, torch.float32) or state_dtype not in (None, h0.dtype):
                g.add("unsupported_dtype", f"h_init is {h0.dtype}, the state is {state_dtype or x_seq.dtype}"
                                           + ("" if state_dtype else " or torch.float32"))
        if lengths is not None:
            _like(g, "lengths", lengths, (B,), torch.int32)
    return g.why


def _is_plain(x, g, gate, h0, lengths, batch_first, state_dtype) -> bool:
    """Whether nothing needs a second look: what ``check_temporal_gated_scan_support`` would say yes to, at the price that a
    decoding step can pay. Anything else goes through the full check."""
    if not (type(x) is torch.Tensor and type(g) is torch.Tensor and x.is_cuda and x.dim() == 3 and x.dtype in ACT_DTYPES
            and g.shape == x.shape and g.dtype == x.dtype and g.device == x.device and type(gate) is str and gate in GATES
            and state_dtype in (None, torch.float32)):
        return False
    B, D = x.shape[0 if batch_first else 1], x.shape[2]
    return ((h0 is None or _is_f32(h0, (B, D), x.device))
            and (lengths is None or (type(lengths) is torch.Tensor and lengths.dtype == torch.int32
                                     and lengths.device == x.device and lengths.shape == (B,))))


def _is_f32(t, shape, device) -> bool:
    return type(t) is torch.Tensor and t.dtype == torch.float32 and t.device == device and t.shape == shape


def _strides(t, batch_first):
    s = t.stride()
    return (s[1], s[0]) if batch_first else (s[0], s[1])


def _state_out(name, t, B, D, dtype, x_seq, like=None):
    if t is None:
        return torch.empty_like(like) if like is not None else x_seq.new_empty((B, D), dtype=dtype)
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != (B, D) or t.dtype != dtype or t.device != x_seq.device or not t.is_contiguous():
        raise RuntimeError(f"unsupported_output: {name} must be a contiguous {dtype} tensor of shape {(B, D)} on {x_seq.device}")
    return t


def run_temporal_gated_scan(
    x_seq: torch.Tensor,
    gate_seq: torch.Tensor,
    h_init: Optional[torch.Tensor] = None,
    *,
    gate: str = "sigmoid",
    leaky: bool = True,
    lengths: Optional[torch.Tensor] = None,
    batch_first: bool = False,
    state_dtype: Optional[torch.dtype] = None,
    save_for_backward: bool = False,
    h_seq_out: Optional[torch.Tensor] = None,
    h_last_out: Optional[torch.Tensor] = None,
    verbose: bool = False,
) -> TemporalGatedScanResult:
    """The recurrence over x_seq, gate_seq [T,B,D] ([B,T,D] with ``batch_first``); returns h_seq of that shape and the
    last state [B,D].

    ``h_init``: state to start from, None or a 0-dim tensor for zeros. The state is fp32 unless ``h_init`` or
    ``state_dtype`` says it has x_seq's dtype. ``lengths`` (int32 [B], on the device): steps of each sequence; later rows
    are neither read nor counted, their h_seq is zero. ``h_seq_out`` / ``h_last_out``: tensors to write into;
    ``h_last_out`` may be ``h_init`` itself (a decoder's state updated in place); otherwise they share no memory with the
    inputs or each other. Rows may be parts of wider ones (x and
    gate as two halves of one projection); an innermost dimension that is not dense is copied first. The gates have x_seq's
    type. A state that has become infinite stays infinite or becomes NaN, in its channel alone.
    """
    if not _is_plain(x_seq, gate_seq, gate, h_init, lengths, batch_first, state_dtype):
        raise_reasons("temporal_gated_scan",
                      check_temporal_gated_scan_support(x_seq, gate_seq, h_init, gate, lengths, batch_first, state_dtype),
                      False, verbose)
    T, B, D = _sizes(x_seq, batch_first)
    x, g = rows_dense(x_seq), rows_dense(gate_seq)
    h0 = state_or_none(h_init)
    s_dt = h0.dtype if h0 is not None else (state_dtype or torch.float32)
    h0 = h0.contiguous() if h0 is not None else None
    lengths = lengths.contiguous() if lengths is not None else None
    if h_seq_out is None:
        h = dense_like(x)
    else:
        h = h_seq_out
        if not isinstance(h, torch.Tensor) or h.shape != x.shape or h.dtype != x.dtype or h.device != x.device or (D > 1 and h.stride(2) != 1):
            raise RuntimeError(f"unsupported_output: h_seq_out must be a {x.dtype} tensor of shape {tuple(x.shape)} with "
                               f"dense rows on {x.device}")
    h_last = _state_out("h_last_out", h_last_out, B, D, s_dt, x, h0)
    ckpt = None
    if save_for_backward:
        ckpt = torch.empty((_lib.lib.snnb_gated_scan_ckpt_rows(T), B, D), dtype=torch.float32, device=x.device)
    launch("snnb_gated_scan", x.device,
           x.data_ptr(), *_strides(x, batch_first), g.data_ptr(), *_strides(g, batch_first), _lib.ptr(h0), _lib.ptr(lengths),
           h.data_ptr(), *_strides(h, batch_first), h_last.data_ptr(), _lib.ptr(ckpt), T, B, D,
           GATES[gate], int(bool(leaky)), _lib.dtype_code(x.dtype), _lib.dtype_code(s_dt))
    return TemporalGatedScanResult(h, h_last, ckpt)


def _is_ckpt(ckpt, x, batch_first) -> bool:
    T, B, D = _sizes(x, batch_first)
    rows = _lib.lib.snnb_gated_scan_ckpt_rows(T)
    return (ckpt is None and rows == 0) or (_is_f32(ckpt, (rows, B, D), x.device) and ckpt.is_contiguous())


def _check_backward(dh_seq, x_seq, gate_seq, h_init, ckpt, dh_last, gate, lengths, batch_first) -> List[str]:
    why = check_temporal_gated_scan_support(x_seq, gate_seq, h_init, gate, lengths, batch_first)
    if isinstance(x_seq, torch.Tensor) and x_seq.dim() == 3:
        T, B, D = _sizes(x_seq, batch_first)
        g = Gate("x_seq", x_seq)
        _like(g, "dh_seq", dh_seq, x_seq.shape)
        h0, dl = state_or_none(h_init), _state(g, "dh_last", dh_last)
        if dl is not None:
            _like(g, "dh_last", dl, (B, D), h0.dtype if h0 is not None else dl.dtype)
            if dl.dtype not in (x_seq.dtype, torch.float32):
                g.add("unsupported_dtype", f"dh_last is {dl.dtype}, the state is {x_seq.dtype} or torch.float32")
        rows = _lib.lib.snnb_gated_scan_ckpt_rows(T)
        if ckpt is not None or rows > 0:
            _like(g, "ckpt", ckpt, (rows, B, D), torch.float32)
            if isinstance(ckpt, torch.Tensor) and not ckpt.is_contiguous():
                g.add("unsupported_layout", "ckpt is not contiguous")
        why += g.why
    return why


def run_temporal_gated_scan_backward(
    dh_seq: torch.Tensor,
    x_seq: torch.Tensor,
    gate_seq: torch.Tensor,
    h_init: Optional[torch.Tensor] = None,
    ckpt: Optional[torch.Tensor] = None,
    *,
    dh_last: Optional[torch.Tensor] = None,
    gate: str = "sigmoid",
    leaky: bool = True,
    lengths: Optional[torch.Tensor] = None,
    batch_first: bool = False,
    verbose: bool = False,
) -> TemporalGatedScanGradients:
    """Gradients of x_seq, gate_seq and h_init for the gradient dh_seq of h_seq (and dh_last of h_last).

    The other arguments are those of the forward call and the ``ckpt`` that it returned; x_seq, gate_seq and h_init must
    hold what they held then. dh_init has the state's dtype: h_init's, without one dh_last's, else fp32.
    """
    if not (_is_plain(x_seq, gate_seq, gate, h_init, lengths, batch_first, None) and type(dh_seq) is torch.Tensor
            and dh_seq.shape == x_seq.shape and dh_seq.dtype == x_seq.dtype and dh_seq.device == x_seq.device
            and (dh_last is None or _is_f32(dh_last, (x_seq.shape[0 if batch_first else 1], x_seq.shape[2]), x_seq.device))
            and _is_ckpt(ckpt, x_seq, batch_first)):
        raise_reasons("temporal_gated_scan_backward",
                      _check_backward(dh_seq, x_seq, gate_seq, h_init, ckpt, dh_last, gate, lengths, batch_first), False, verbose)
    T, B, D = _sizes(x_seq, batch_first)
    h0, dl = state_or_none(h_init), state_or_none(dh_last)
    dh, x, g = rows_dense(dh_seq), rows_dense(x_seq), rows_dense(gate_seq)
    s_dt = h0.dtype if h0 is not None else (dl.dtype if dl is not None else torch.float32)
    h0 = h0.contiguous() if h0 is not None else None
    dl = dl.contiguous() if dl is not None else None
    lengths = lengths.contiguous() if lengths is not None else None
    dx, dg = dense_like(x), dense_like(x)
    dh_init = _state_out("dh_init", None, B, D, s_dt, x, h0)
    launch("snnb_gated_scan_backward", x.device,
           dh.data_ptr(), *_strides(dh, batch_first), _lib.ptr(dl), x.data_ptr(), *_strides(x, batch_first),
           g.data_ptr(), *_strides(g, batch_first), _lib.ptr(h0), _lib.ptr(ckpt), _lib.ptr(lengths),
           dx.data_ptr(), *_strides(dx, batch_first), dg.data_ptr(), *_strides(dg, batch_first), dh_init.data_ptr(),
           T, B, D, GATES[gate], int(bool(leaky)), _lib.dtype_code(x.dtype), _lib.dtype_code(s_dt))
    return TemporalGatedScanGradients(dx, dg, dh_init)
