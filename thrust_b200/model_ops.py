"""Operators of language models that are scans and histograms: the gated linear recurrence of a recurrent layer, and the
statistics of routing its tokens to experts.

Like the rest of this package they take CUDA tensors, enqueue on the current stream of their device and, unless
``sync=False``, synchronise and check the device status before returning. Gradients are calls of their own; nothing
here records itself for autograd.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _capi as capi
from .algorithms import _On, _finish, _stream, _temp

_FLOATS = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}
_INDEX_BYTES = {torch.int32: 4, torch.int64: 8}


def _require_cuda(device, **tensors) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (thrust_b200 has no CPU path)")
        if t.device != device:
            raise ValueError(f"{name} lies on {t.device}, not on {device}")


def _float_code(t: torch.Tensor, name: str) -> int:
    try:
        return _FLOATS[t.dtype]
    except KeyError:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}") from None


def _rows(t: torch.Tensor, name: str) -> capi.Rows:
    """A [rows, channels] or [sequences, rows, channels] tensor whose channels are adjacent, by its strides."""
    stride = t.stride()
    if stride[-1] != 1 and t.shape[-1] > 1 and t.numel():
        raise ValueError(f"the channels of {name} must be adjacent in memory (its last stride is {stride[-1]})")
    return capi.Rows(t.data_ptr(), stride[-2], stride[0] if t.dim() == 3 else 0)


def _states(t: Optional[torch.Tensor], shape, name: str) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape {list(shape)}")
    return t.data_ptr()


def _offsets(t: Optional[torch.Tensor]) -> Tuple[int, Optional[int]]:
    if t is None:
        return 0, None
    if t.dtype not in _INDEX_BYTES or t.dim() != 1 or t.numel() < 1 or not t.is_contiguous():
        raise ValueError("offsets must be a contiguous 1-D tensor of sequences + 1 int32 or int64 elements")
    return _INDEX_BYTES[t.dtype], t.data_ptr()


def _shape(x: torch.Tensor, gate: torch.Tensor, offsets: Optional[torch.Tensor], log_gate: bool, fill: bool, name: str):
    """(shape structure, sequences) of a recurrence over x with these gates."""
    packed = offsets is not None
    if x.dim() != (2 if packed else 3):
        raise ValueError(f"{name} must be [rows, channels] with offsets, [sequences, rows, channels] without")
    if gate.shape[:-1] != x.shape[:-1] or gate.dim() != x.dim():
        raise ValueError(f"gate must have a row for each row of {name}")
    channels, heads = x.shape[-1], gate.shape[-1]
    if channels == 0 or heads == 0 or channels % heads:
        raise ValueError("a row must have a gate for each channel, or for each group of channels / gates neighbours")
    xd, gd = _float_code(x, name), _float_code(gate, "gate")
    if gd != xd and gd != capi.F32:
        raise TypeError(f"gate must have the type of {name} or float32")
    obytes, optr = _offsets(offsets)
    sequences = offsets.numel() - 1 if packed else x.shape[0]
    return capi.RecurrenceShape(sequences, x.shape[-2], channels, heads, xd, gd, int(bool(log_gate)), obytes,
                                int(fill)), sequences, optr


@lru_cache(maxsize=512)
def _recurrence_bytes(back: bool, *dims) -> int:
    need = C.c_size_t(0)
    s = capi.RecurrenceShape(*dims)
    if back:
        rc = capi.lib.tb200_linear_recurrence_backward(None, C.byref(need), C.byref(s), *(None,) * 10)
    else:
        rc = capi.lib.tb200_linear_recurrence(None, C.byref(need), C.byref(s), *(None,) * 7)
    capi.check(rc, "tb200_linear_recurrence(size)")
    return need.value


def _scratch(back: bool, s, device, temp: Optional[torch.Tensor]) -> torch.Tensor:
    need = _recurrence_bytes(back, s.sequences, s.rows, s.channels, s.heads, s.dtype, s.gate_dtype, s.log_gate,
                             s.offset_bytes, s.fill_outside)
    return _temp(need, device) if temp is None or temp.numel() < need else temp


def linear_recurrence(x: torch.Tensor, gate: torch.Tensor, initial: Optional[torch.Tensor] = None,
                      offsets: Optional[torch.Tensor] = None, log_gate: bool = False, out: Optional[torch.Tensor] = None,
                      sync: bool = True, temp: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """y[t] = a[t] * y[t-1] + x[t] by sequence and channel; returns (y, final states).

    x: [sequences, rows, channels], or packed [rows, channels] with ``offsets`` (sequences + 1 ascending int32 or int64
    from 0: sequence s owns rows offsets[s] to offsets[s+1] - 1, empty ones allowed). float32, float16 or bfloat16; any
    row and sequence strides, adjacent channels. gate: a[t] itself or, with ``log_gate``, its logarithm (-inf forgets);
    x's rows with a gate for each channel, or for each of ``heads`` groups of neighbouring channels; x's type or
    float32. initial: float32 [sequences, channels], y in front of the first row (None: zero). The final states have
    that shape and type; that of an empty sequence is its initial one. States are held in 32 bits, y is rounded once.
    ``out`` may be x. Packed rows behind the last sequence are left as they were in ``out``, and zero in a fresh y.
    Results are reproducible from run to run. A value that is not finite makes the rows behind it, in its sequence and
    channel, not finite."""
    _require_cuda(x.device, x=x, gate=gate, initial=initial, offsets=offsets, out=out)
    s, sequences, optr = _shape(x, gate, offsets, log_gate, out is None, "x")
    states = (sequences, x.shape[-1])
    iptr = _states(initial, states, "initial")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError("out must have the shape and type of x")
    rg, rx, ry = _rows(gate, "gate"), _rows(x, "x"), _rows(out, "out")
    final = torch.empty(states, dtype=torch.float32, device=x.device)
    with _On(x.device):
        stream = _stream(x)
        temp = _scratch(False, s, x.device, temp)
        have = C.c_size_t(temp.numel())
        capi.check(capi.lib.tb200_linear_recurrence(temp.data_ptr(), C.byref(have), C.byref(s), optr, C.byref(rg),
                                                    C.byref(rx), C.byref(ry), iptr, final.data_ptr(), stream),
                   "tb200_linear_recurrence")
        _finish(temp, stream, "tb200_linear_recurrence", sync)
    return out, final


def linear_recurrence_backward(gate: torch.Tensor, y: torch.Tensor, dy: torch.Tensor,
                               initial: Optional[torch.Tensor] = None, dfinal: Optional[torch.Tensor] = None,
                               offsets: Optional[torch.Tensor] = None, log_gate: bool = False, sync: bool = True,
                               temp: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of ``linear_recurrence`` from its gates and its output: returns (dx, dgate, dinitial).

    dy is the gradient of y, ``dfinal`` that of the final states (None: zero); ``initial``, ``offsets`` and ``log_gate``
    as in the forward call. dx has dy's type, dgate the gates' shape and type (summed over the channels that share a
    gate), dinitial is float32 [sequences, channels]. Packed rows behind the last sequence have zero gradients."""
    _require_cuda(dy.device, dy=dy, gate=gate, y=y, initial=initial, dfinal=dfinal, offsets=offsets)
    if y.shape != dy.shape or y.dtype != dy.dtype:
        raise ValueError("y and dy must have the same shape and type")
    s, sequences, optr = _shape(dy, gate, offsets, log_gate, True, "dy")
    states = (sequences, dy.shape[-1])
    iptr, fptr = _states(initial, states, "initial"), _states(dfinal, states, "dfinal")
    dx = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
    dgate = torch.empty(gate.shape, dtype=gate.dtype, device=dy.device)
    dinitial = torch.empty(states, dtype=torch.float32, device=dy.device)
    rg, ry, rdy = _rows(gate, "gate"), _rows(y, "y"), _rows(dy, "dy")
    rdx, rdg = _rows(dx, "dx"), _rows(dgate, "dgate")
    with _On(dy.device):
        stream = _stream(dy)
        temp = _scratch(True, s, dy.device, temp)
        have = C.c_size_t(temp.numel())
        capi.check(capi.lib.tb200_linear_recurrence_backward(
            temp.data_ptr(), C.byref(have), C.byref(s), optr, C.byref(rg), C.byref(ry), C.byref(rdy), C.byref(rdx),
            C.byref(rdg), iptr, fptr, dinitial.data_ptr(), stream), "tb200_linear_recurrence_backward")
        _finish(temp, stream, "tb200_linear_recurrence_backward", sync)
    return dx, dgate, dinitial


def linear_recurrence_step(state: torch.Tensor, x: torch.Tensor, gate: torch.Tensor,
                           slots: Optional[torch.Tensor] = None, log_gate: bool = False,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One row of many sequences, as in decoding: ``state`` = a * state + x in place; returns y, the new states rounded.

    state: float32 [slots, channels], a pool of states with adjacent channels. x: [rows, channels], gate: [rows,
    channels or heads], as in ``linear_recurrence``. Row r works on state slots[r] (int32 or int64, at most 65536 of
    them; None: state r). A row whose slot lies outside the pool (a negative one, say, where a batch is padded) gets a
    zero y and changes nothing; rows that name the same slot are applied in their order. Enqueues one kernel and
    returns without waiting."""
    _require_cuda(x.device, x=x, state=state, gate=gate, slots=slots, out=out)
    if x.dim() != 2 or state.dim() != 2 or state.dtype != torch.float32 or state.shape[1] != x.shape[1]:
        raise ValueError("x must be [rows, channels] and state float32 [slots, channels]")
    rows, channels = x.shape
    if gate.dim() != 2 or gate.shape[0] != rows or gate.shape[1] == 0 or channels == 0 or channels % gate.shape[1]:
        raise ValueError("gate must be [rows, channels], or [rows, heads] with a number of heads that divides the channels")
    xd, gd = _float_code(x, "x"), _float_code(gate, "gate")
    if gd != xd and gd != capi.F32:
        raise TypeError("gate must have the type of x or float32")
    sbytes, sptr = 0, None
    if slots is not None:
        if slots.dtype not in _INDEX_BYTES or slots.shape != (rows,) or not slots.is_contiguous():
            raise ValueError("slots must be a contiguous 1-D tensor of an int32 or int64 for each row")
        sbytes, sptr = _INDEX_BYTES[slots.dtype], slots.data_ptr()
    elif rows > state.shape[0]:
        raise ValueError("x has more rows than there are states")
    if state.shape[0] > 1 and state.stride(0) < channels:
        raise ValueError("the states of the pool overlap")
    if out is None:
        out = torch.empty((rows, channels), dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError("out must have the shape and type of x")
    rs, rg, rx, ry = _rows(state, "state"), _rows(gate, "gate"), _rows(x, "x"), _rows(out, "out")
    with _On(x.device):
        capi.check(capi.lib.tb200_linear_recurrence_step(
            rs.data, state.shape[0], max(rs.row_stride, channels), sptr, sbytes, C.byref(rg), C.byref(rx), C.byref(ry), rows,
            channels, gate.shape[1], xd, gd, int(bool(log_gate)), _stream(x)), "tb200_linear_recurrence_step")
    return out


def _ids(ids: torch.Tensor) -> Tuple[int, int, int, int]:
    """(rows, ids of a row, distance of rows, bytes of an id)"""
    if ids.dtype not in _INDEX_BYTES or ids.dim() not in (1, 2):
        raise ValueError("ids must be an int32 or int64 tensor [rows, k], or [rows]")
    if ids.dim() == 1:
        return ids.shape[0], 1, ids.stride(0) if ids.shape[0] > 1 else 1, _INDEX_BYTES[ids.dtype]
    rows, k = ids.shape
    if k == 0 or (rows and k > 1 and ids.stride(1) != 1) or (rows > 1 and ids.stride(0) < k):
        raise ValueError("the ids of a row must be adjacent in memory, at least one, and rows must not overlap")
    return rows, k, ids.stride(0) if rows > 1 else k, _INDEX_BYTES[ids.dtype]


def _mask(mask: Optional[torch.Tensor], rows: int) -> Optional[int]:
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8) or mask.shape != (rows,) or not mask.is_contiguous():
        raise ValueError("mask must be a contiguous 1-D tensor of a bool or uint8 for each row")
    return mask.data_ptr()


@lru_cache(maxsize=512)
def _counts_bytes(experts: int) -> int:
    need = C.c_size_t(0)
    capi.check(capi.lib.tb200_expert_counts(None, C.byref(need), None, 0, 1, 1, 8, None, experts, None, None, None),
               "tb200_expert_counts(size)")
    return need.value


@lru_cache(maxsize=512)
def _balance_bytes(dtype: int, offset_bytes: int, sequences: int, experts: int) -> int:
    need = C.c_size_t(0)
    capi.check(capi.lib.tb200_balance_loss(None, C.byref(need), None, dtype, None, 1, 1, 8, None, None, offset_bytes,
                                           sequences, 0, experts, None, None, None, None), "tb200_balance_loss(size)")
    return need.value


def expert_counts(ids: torch.Tensor, experts: int, mask: Optional[torch.Tensor] = None, sync: bool = True,
                  temp: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Tokens per expert: returns (counts [experts], begins [experts + 1]), int64.

    ids: the experts that each row (token) was routed to, int32 or int64, [rows, k] with the ids of a row adjacent, or
    [rows]. counts[e] is how often e occurs in rows whose mask (bool [rows], None: all) is set; ids outside
    [0, experts) are not counted. begins is the exclusive prefix sum of the counts: where each expert's tokens begin
    once (id, token) pairs are sorted with ``sort_by_key``. At most 8192 experts."""
    _require_cuda(ids.device, ids=ids, mask=mask)
    rows, k, stride, width = _ids(ids)
    mptr = _mask(mask, rows)
    need = _counts_bytes(experts)
    both = torch.empty(2 * experts + 1, dtype=torch.int64, device=ids.device)
    counts, begins = both[:experts], both[experts:]
    with _On(ids.device):
        stream = _stream(ids)
        if temp is None or temp.numel() < need:
            temp = _temp(need, ids.device)
        have = C.c_size_t(temp.numel())
        capi.check(capi.lib.tb200_expert_counts(temp.data_ptr(), C.byref(have), ids.data_ptr(), rows, k, stride, width,
                                                mptr, experts, counts.data_ptr(), begins.data_ptr(), stream),
                   "tb200_expert_counts")
        _finish(temp, stream, "tb200_expert_counts", sync)
    return counts, begins


def _logits(logits: torch.Tensor, offsets: Optional[torch.Tensor]):
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [rows, experts]")
    obytes, optr = _offsets(offsets)
    return _float_code(logits, "logits"), obytes, optr, 1 if offsets is None else offsets.numel() - 1


def balance_loss(logits: torch.Tensor, ids: torch.Tensor, mask: Optional[torch.Tensor] = None,
                 offsets: Optional[torch.Tensor] = None, sync: bool = True,
                 temp: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Balance loss of a router: returns (loss [sequences], counts [sequences, experts], weights [sequences, experts]).

    logits: [rows, experts], float32, float16 or bfloat16, at most 1024 experts; ids: the k experts chosen for each
    row, as in ``expert_counts``; mask: rows to look at. With ``offsets`` (as in ``linear_recurrence``) the loss of
    every packed sequence, without them one loss over all rows:

        experts / (k * n^2) * sum_e counts[e] * sum_t softmax(logits[t])[e],   n = unmasked rows

    which is 1 when both are balanced, and 0 without any rows. A logit of -inf is a disabled expert; a row of nothing
    else has no probabilities. weights is the derivative of a sequence's loss by each of its probabilities: what
    ``balance_loss_backward`` needs besides the logits. Results are reproducible from run to run."""
    _require_cuda(logits.device, logits=logits, ids=ids, mask=mask, offsets=offsets)
    dtype, obytes, optr, sequences = _logits(logits, offsets)
    rows, k, stride, width = _ids(ids)
    if rows != logits.shape[0]:
        raise ValueError("logits and ids differ in rows")
    experts = logits.shape[1]
    mptr, rz = _mask(mask, rows), _rows(logits, "logits")
    need = _balance_bytes(dtype, obytes, sequences, experts)
    loss = torch.empty(sequences, dtype=torch.float32, device=logits.device)
    counts = torch.empty((sequences, experts), dtype=torch.int64, device=logits.device)
    weights = torch.empty((sequences, experts), dtype=torch.float32, device=logits.device)
    with _On(logits.device):
        stream = _stream(logits)
        if temp is None or temp.numel() < need:
            temp = _temp(need, logits.device)
        have = C.c_size_t(temp.numel())
        capi.check(capi.lib.tb200_balance_loss(
            temp.data_ptr(), C.byref(have), C.byref(rz), dtype, ids.data_ptr(), k, stride, width, mptr, optr, obytes,
            sequences, rows, experts, loss.data_ptr(), counts.data_ptr(), weights.data_ptr(), stream),
            "tb200_balance_loss")
        _finish(temp, stream, "tb200_balance_loss", sync)
    return loss, counts, weights


def balance_loss_backward(logits: torch.Tensor, weights: torch.Tensor, dloss: torch.Tensor,
                          mask: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``balance_loss`` by the logits, in their type, from its weights and dloss (float32 [sequences], the
    gradient of the losses); mask and offsets as in the forward call. Zero for masked rows and rows of no sequence.
    ``out`` may be logits. Enqueues one kernel and returns without waiting."""
    _require_cuda(logits.device, logits=logits, weights=weights, dloss=dloss, mask=mask, offsets=offsets, out=out)
    dtype, obytes, optr, sequences = _logits(logits, offsets)
    rows, experts = logits.shape
    wptr = _states(weights, (sequences, experts), "weights")
    lptr = _states(dloss, (sequences,), "dloss")
    if out is None:
        out = torch.empty((rows, experts), dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype != logits.dtype:
        raise ValueError("out must have the shape and type of logits")
    mptr, rz, rd = _mask(mask, rows), _rows(logits, "logits"), _rows(out, "out")
    with _On(logits.device):
        capi.check(capi.lib.tb200_balance_loss_backward(C.byref(rz), dtype, wptr, lptr, mptr, optr, obytes, sequences, rows,
                                                        experts, C.byref(rd), _stream(logits)),
                   "tb200_balance_loss_backward")
    return out
