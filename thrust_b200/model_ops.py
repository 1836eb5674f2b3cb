"""Operators of language models that are scans and histograms: the gated linear recurrence of a recurrent layer, and the
statistics of routing its tokens to experts.

Like the rest of this package they take CUDA tensors, enqueue on the current stream of their device and, unless
``sync=False``, synchronise and check the device status before returning. Gradients are calls of their own; nothing
here records itself for autograd.
"""
from __future__ import annotations

import ctypes as C
import math
from functools import lru_cache
from typing import List, Optional, Tuple

import torch

from . import _capi as capi

_FLOATS = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}
_INDEX_BYTES = {torch.int32: 4, torch.int64: 8}

# A decoding step makes these calls for a few microseconds of work, so what they cost on the host is kept small: tensors
# are asked for little, arrays of rows go over as plain words, the current device is looked at only where there are
# several, and the current stream is asked for as a number.
_several_devices = lru_cache(maxsize=1)(lambda: torch.cuda.device_count() > 1)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(function, what: str, index: int, *args) -> None:
    if _several_devices() and torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            rc = function(*args)
    else:
        rc = function(*args)
    if rc:
        capi.check(rc, what)


def _status(temp: torch.Tensor, stream: int, what: str, index: int, sync: bool) -> None:
    if sync:
        _call(capi.lib.tb200_temp_status, what, index, temp.data_ptr(), stream)


def _device_of(name: str, t: torch.Tensor) -> int:
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor (thrust_b200 has no CPU path)")
    return index


def _same_device(index: int, name: str, t: Optional[torch.Tensor]) -> None:
    if t is not None and t.get_device() != index:
        _device_of(name, t)
        raise ValueError(f"{name} lies on {t.device}, not on cuda:{index}")


def _float_code(t: torch.Tensor, name: str) -> int:
    try:
        return _FLOATS[t.dtype]
    except KeyError:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}") from None


def _types(x: torch.Tensor, name: str, gate: torch.Tensor) -> Tuple[int, int]:
    xd, gd = _float_code(x, name), _float_code(gate, "gate")
    if gd != xd and gd != capi.F32:
        raise TypeError(f"gate must have the type of {name} or float32")
    return xd, gd


def _rows(t: torch.Tensor, name: str) -> Tuple[int, int, int]:
    """A [rows, channels] or [sequences, rows, channels] tensor with adjacent channels, as the words of a tb200_rows."""
    stride = t.stride()
    if stride[-1] != 1 and t.shape[-1] > 1 and t.numel():
        raise ValueError(f"the channels of {name} must be adjacent in memory (its last stride is {stride[-1]})")
    return t.data_ptr(), stride[-2], stride[0] if len(stride) == 3 else 0


class _Room:
    """Room for five tb200_rows one behind the other, as a call hands them over; it has read them when it returns."""

    def __init__(self):
        self.words = (C.c_uint64 * 15)()
        base = C.addressof(self.words)
        self.at = tuple(base + 24 * i for i in range(5))


# Rooms that no call is using. A call takes one for itself, so that neither another thread nor a finaliser or signal handler
# that makes such a call in between writes into it; pop and append are one step each.
_rooms: List[_Room] = []


def _arrays(*rows) -> Tuple[_Room, Tuple[int, ...]]:
    """These arrays of rows in a room of their own, and their addresses there. The caller gives the room back."""
    try:
        room = _rooms.pop()
    except IndexError:
        room = _Room()
    flat = [w for r in rows for w in r]
    room.words[:len(flat)] = flat
    return room, room.at[:len(rows)]


def _states(t: Optional[torch.Tensor], shape, name: str) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape {list(shape)}")
    return t.data_ptr()


def _offsets(t: Optional[torch.Tensor]) -> Tuple[int, Optional[int]]:
    if t is None:
        return 0, None
    if t.dtype not in _INDEX_BYTES or t.dim() != 1 or t.numel() < 1 or not t.is_contiguous():
        raise ValueError("offsets must be a contiguous 1-D tensor of sequences + 1 int32 or int64 elements")
    return _INDEX_BYTES[t.dtype], t.data_ptr()


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _new(shape, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A fresh contiguous tensor of one or two dimensions, the cheapest way there is."""
    return torch.empty_strided(shape, (1,) if len(shape) == 1 else (shape[1], 1), dtype=dtype, device=device)


def _lead(t: torch.Tensor) -> List[Tuple[int, int]]:
    """(bytes apart, how many) of the dimensions that rows of t are counted in, the largest distance first."""
    size = t.element_size()
    return sorted(((s * size, n) for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1), reverse=True)


def _rows_apart(t: torch.Tensor) -> bool:
    """Whether no two rows of t share memory: every distance reaches over all that is counted in smaller ones."""
    if t.is_contiguous():
        return True
    width = t.shape[-1] * t.element_size()
    for apart, n in reversed(_lead(t)):
        if apart < width:
            return False
        width += (n - 1) * apart
    return True


def _reach(t: torch.Tensor) -> int:
    """Bytes from the first element of t to behind its last one."""
    return t.nbytes if t.is_contiguous() else (sum(s * (n - 1) for s, n in zip(t.stride(), t.shape)) + 1) * t.element_size()


def _disjoint(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two arrays of rows share no memory. False also where they lie in one another's way in an order that does
    not show it."""
    at, bt = a.data_ptr(), b.data_ptr()
    if at + _reach(a) <= bt or bt + _reach(b) <= at or a.numel() == 0 or b.numel() == 0:
        return True
    la, lb = _lead(a), _lead(b)
    wa, wb = a.shape[-1] * a.element_size(), b.shape[-1] * b.element_size()
    # columns side by side: no two rows meet, whichever they are
    apart = math.gcd(*(s for s, _ in la + lb))
    if apart and (bt - at) % apart >= wa and (at - bt) % apart >= wb:
        return True
    if la != lb or any(s == 0 for s, _ in la):
        return False

    # the same distances: rows meet where b lies behind a by some of each distance and less than a row
    def meet(lead, p) -> bool:
        if not lead:
            return -wb < p < wa
        (s, n), reach = lead[0], sum(d * (m - 1) for d, m in lead[1:])
        first, last = -((reach + wa - p) // s), (p + reach + wb) // s
        return any(meet(lead[1:], p - i * s) for i in range(max(first, 1 - n), min(last, n - 1) + 1))

    return not meet(la, bt - at)


def _output(out: Optional[torch.Tensor], like: torch.Tensor, name: str, *others: Optional[torch.Tensor]) -> torch.Tensor:
    """A fresh output, or the caller's: it may be `like` itself, and shares memory with nothing else."""
    if out is None:
        return _empty_like(like)
    if out.shape != like.shape or out.dtype != like.dtype:
        raise ValueError(f"out must have the shape and type of {name}")
    if not _rows_apart(out):
        raise ValueError("the rows of out share memory")
    begin = out.data_ptr()
    end = begin + _reach(out)
    for t in others if out is like else (like, *others):
        if t is None:
            continue
        at = t.data_ptr()
        if end <= at or at + _reach(t) <= begin or _disjoint(out, t):
            continue
        if t is not like:
            raise ValueError(f"out must not share memory with other arguments than {name}")
        if at != begin or any(n > 1 and s != d for n, s, d in zip(out.shape, out.stride(), t.stride())):
            raise ValueError(f"out must be {name} itself or share no memory with it")
    return out


def _scratch(need: int, like: torch.Tensor, temp: Optional[torch.Tensor]) -> torch.Tensor:
    if temp is not None and temp.numel() >= need:
        if not temp.is_contiguous():
            raise ValueError("temp must be contiguous")
        return temp
    return _new((need,), torch.uint8, like.device)


@lru_cache(maxsize=512)
def _recurrence_bytes(back: bool, *dims) -> int:
    need = C.c_size_t(0)
    s = capi.RecurrenceShape(*dims)
    if back:
        rc = capi.lib.tb200_linear_recurrence_backward(None, C.byref(need), C.byref(s), *(None,) * 10)
    else:
        rc = capi.lib.tb200_linear_recurrence(None, C.byref(need), C.byref(s), *(None,) * 7)
    capi.check(rc, "tb200_linear_recurrence(size)")
    return max(need.value, 256)


def _shape(x: torch.Tensor, gate: torch.Tensor, offsets: Optional[torch.Tensor], log_gate: bool, fill: bool, name: str):
    """(the words of the shape, address of the offsets) of a recurrence over x with these gates."""
    xs, gs = x.shape, gate.shape
    if len(xs) != (3 if offsets is None else 2):
        raise ValueError(f"{name} must be [rows, channels] with offsets, [sequences, rows, channels] without")
    if gs[:-1] != xs[:-1] or len(gs) != len(xs):
        raise ValueError(f"gate must have a row for each row of {name}")
    channels, heads = xs[-1], gs[-1]
    if channels == 0 or heads == 0 or channels % heads:
        raise ValueError("a row must have a gate for each channel, or for each group of channels / gates neighbours")
    xd, gd = _types(x, name, gate)
    obytes, optr = _offsets(offsets)
    sequences = xs[0] if offsets is None else offsets.shape[0] - 1
    return (sequences, xs[-2], channels, heads, xd, gd, 1 if log_gate else 0, obytes, 1 if fill else 0), optr


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
    ``out`` may be x itself and shares no memory with anything else. Packed rows behind the last sequence are left as
    they were in ``out``, and zero in a fresh y. Results are reproducible from run to run. A value that is not finite makes the rows behind it, in its sequence and
    channel, not finite."""
    index = _device_of("x", x)
    for name, t in (("gate", gate), ("initial", initial), ("offsets", offsets), ("out", out), ("temp", temp)):
        _same_device(index, name, t)
    dims, optr = _shape(x, gate, offsets, log_gate, out is None, "x")
    states = (dims[0], dims[2])
    iptr = _states(initial, states, "initial")
    out = _output(out, x, "x", gate, initial)
    room, arrays = _arrays(_rows(gate, "gate"), _rows(x, "x"), _rows(out, "out"))
    final = _new(states, torch.float32, x.device)
    temp = _scratch(_recurrence_bytes(False, *dims), x, temp)
    shape, have, stream = capi.RecurrenceShape(*dims), C.c_size_t(temp.numel()), _raw_stream(index)
    _call(capi.lib.tb200_linear_recurrence, "tb200_linear_recurrence", index, temp.data_ptr(), C.byref(have),
          C.byref(shape), optr, *arrays, iptr, final.data_ptr(), stream)
    _rooms.append(room)
    _status(temp, stream, "tb200_linear_recurrence", index, sync)
    return out, final


def linear_recurrence_backward(gate: torch.Tensor, y: torch.Tensor, dy: torch.Tensor,
                               initial: Optional[torch.Tensor] = None, dfinal: Optional[torch.Tensor] = None,
                               offsets: Optional[torch.Tensor] = None, log_gate: bool = False, sync: bool = True,
                               temp: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of ``linear_recurrence`` from its gates and its output: returns (dx, dgate, dinitial).

    dy is the gradient of y, ``dfinal`` that of the final states (None: zero); ``initial``, ``offsets`` and ``log_gate``
    as in the forward call. dx has dy's type, dgate the gates' shape and type (summed over the channels that share a
    gate), dinitial is float32 [sequences, channels]. Packed rows behind the last sequence have zero gradients."""
    index = _device_of("dy", dy)
    for name, t in (("gate", gate), ("y", y), ("initial", initial), ("dfinal", dfinal), ("offsets", offsets), ("temp", temp)):
        _same_device(index, name, t)
    if y.shape != dy.shape or y.dtype != dy.dtype:
        raise ValueError("y and dy must have the same shape and type")
    dims, optr = _shape(dy, gate, offsets, log_gate, True, "dy")
    states = (dims[0], dims[2])
    iptr, fptr = _states(initial, states, "initial"), _states(dfinal, states, "dfinal")
    dx, dgate = _empty_like(dy), _empty_like(gate)
    dinitial = _new(states, torch.float32, dy.device)
    room, arrays = _arrays(_rows(gate, "gate"), _rows(y, "y"), _rows(dy, "dy"), _rows(dx, "dx"), _rows(dgate, "dgate"))
    temp = _scratch(_recurrence_bytes(True, *dims), dy, temp)
    shape, have, stream = capi.RecurrenceShape(*dims), C.c_size_t(temp.numel()), _raw_stream(index)
    _call(capi.lib.tb200_linear_recurrence_backward, "tb200_linear_recurrence_backward", index, temp.data_ptr(),
          C.byref(have), C.byref(shape), optr, *arrays, iptr, fptr, dinitial.data_ptr(), stream)
    _rooms.append(room)
    _status(temp, stream, "tb200_linear_recurrence_backward", index, sync)
    return dx, dgate, dinitial


def linear_recurrence_step(state: torch.Tensor, x: torch.Tensor, gate: torch.Tensor,
                           slots: Optional[torch.Tensor] = None, log_gate: bool = False,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One row of many sequences, as in decoding: ``state`` = a * state + x in place; returns y, the new states rounded.

    state: float32 [slots, channels], a pool of states with adjacent channels. x: [rows, channels], gate: [rows,
    channels or heads], as in ``linear_recurrence``. Row r works on state slots[r] (int32 or int64, at most 65536 of
    them; None: state r). A row whose slot lies outside the pool (a negative one, say, where a batch is padded) gets a
    zero y and changes nothing; rows that name the same slot are applied in their order. ``out`` may be x itself and
    shares no memory with anything else. Enqueues one kernel and returns without waiting."""
    index = _device_of("x", x)
    _same_device(index, "state", state)
    _same_device(index, "gate", gate)
    _same_device(index, "slots", slots)
    _same_device(index, "out", out)
    xs, ss, gs = x.shape, state.shape, gate.shape
    if len(xs) != 2 or len(ss) != 2 or state.dtype != torch.float32 or ss[1] != xs[1]:
        raise ValueError("x must be [rows, channels] and state float32 [slots, channels]")
    rows, channels = xs
    if len(gs) != 2 or gs[0] != rows or gs[1] == 0 or channels == 0 or channels % gs[1]:
        raise ValueError("gate must be [rows, channels], or [rows, heads] with a number of heads that divides the channels")
    xd, gd = _types(x, "x", gate)
    sbytes, sptr = 0, None
    if slots is not None:
        if slots.dtype not in _INDEX_BYTES or slots.shape != (rows,) or not slots.is_contiguous():
            raise ValueError("slots must be a contiguous 1-D tensor of an int32 or int64 for each row")
        sbytes, sptr = _INDEX_BYTES[slots.dtype], slots.data_ptr()
    elif rows > ss[0]:
        raise ValueError("x has more rows than there are states")
    pool, apart, _ = _rows(state, "state")
    if ss[0] <= 1:
        apart = channels
    elif apart < channels:
        raise ValueError("the states of the pool overlap")
    out = _output(out, x, "x", gate, state)
    room, arrays = _arrays(_rows(gate, "gate"), _rows(x, "x"), _rows(out, "out"))
    _call(capi.lib.tb200_linear_recurrence_step, "tb200_linear_recurrence_step", index, pool, ss[0], apart, sptr, sbytes,
          *arrays, rows, channels, gs[1], xd, gd, 1 if log_gate else 0, _raw_stream(index))
    _rooms.append(room)
    return out


def _ids(ids: torch.Tensor) -> Tuple[int, int, int, int]:
    """(rows, ids of a row, distance of rows, bytes of an id)"""
    width, shape = _INDEX_BYTES.get(ids.dtype), ids.shape
    if width is None or len(shape) not in (1, 2):
        raise ValueError("ids must be an int32 or int64 tensor [rows, k], or [rows]")
    stride = ids.stride()
    if len(shape) == 1:
        return shape[0], 1, stride[0] if shape[0] > 1 else 1, width
    rows, k = shape
    if k == 0 or k >> 32 or (rows and k > 1 and stride[1] != 1) or (rows > 1 and stride[0] < k):
        raise ValueError("the ids of a row must be adjacent in memory, at least one, less than 2^32, and rows must not overlap")
    return rows, k, stride[0] if rows > 1 else k, width


def _mask(mask: Optional[torch.Tensor], rows: int) -> Optional[int]:
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8) or mask.shape != (rows,) or not mask.is_contiguous():
        raise ValueError("mask must be a contiguous 1-D tensor of a bool or uint8 for each row")
    return mask.data_ptr()


@lru_cache(maxsize=512)
def _counts_bytes(experts: int) -> int:
    if experts >> 32:  # the library would see the lower 32 bits
        raise ValueError("at most 8192 experts")
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
    index = _device_of("ids", ids)
    _same_device(index, "mask", mask)
    _same_device(index, "temp", temp)
    rows, k, stride, width = _ids(ids)
    mptr = _mask(mask, rows)
    temp = _scratch(_counts_bytes(experts), ids, temp)
    device = ids.device
    counts, begins = _new((experts,), torch.int64, device), _new((experts + 1,), torch.int64, device)
    have, raw = C.c_size_t(temp.numel()), _raw_stream(index)
    _call(capi.lib.tb200_expert_counts, "tb200_expert_counts", index, temp.data_ptr(), C.byref(have), ids.data_ptr(), rows,
          k, stride, width, mptr, experts, counts.data_ptr(), begins.data_ptr(), raw)
    _status(temp, raw, "tb200_expert_counts", index, sync)
    return counts, begins


def _logits(logits: torch.Tensor, offsets: Optional[torch.Tensor]):
    shape = logits.shape
    if len(shape) != 2 or shape[1] == 0 or shape[1] >> 32:
        raise ValueError("logits must be [rows, experts]")
    obytes, optr = _offsets(offsets)
    return _float_code(logits, "logits"), obytes, optr, 1 if offsets is None else offsets.shape[0] - 1, shape[0], shape[1]


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
    index = _device_of("logits", logits)
    for name, t in (("ids", ids), ("mask", mask), ("offsets", offsets), ("temp", temp)):
        _same_device(index, name, t)
    dtype, obytes, optr, sequences, rows, experts = _logits(logits, offsets)
    id_rows, k, stride, width = _ids(ids)
    if id_rows != rows:
        raise ValueError("logits and ids differ in rows")
    mptr, (room, arrays) = _mask(mask, rows), _arrays(_rows(logits, "logits"))
    temp = _scratch(_balance_bytes(dtype, obytes, sequences, experts), logits, temp)
    device, cells = logits.device, (sequences, experts)
    loss, counts, weights = _new((sequences,), torch.float32, device), _new(cells, torch.int64, device), _new(cells, torch.float32, device)
    have, stream = C.c_size_t(temp.numel()), _raw_stream(index)
    _call(capi.lib.tb200_balance_loss, "tb200_balance_loss", index, temp.data_ptr(), C.byref(have), arrays[0], dtype,
          ids.data_ptr(), k, stride, width, mptr, optr, obytes, sequences, rows, experts, loss.data_ptr(),
          counts.data_ptr(), weights.data_ptr(), stream)
    _rooms.append(room)
    _status(temp, stream, "tb200_balance_loss", index, sync)
    return loss, counts, weights


def balance_loss_backward(logits: torch.Tensor, weights: torch.Tensor, dloss: torch.Tensor,
                          mask: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``balance_loss`` by the logits, in their type, from its weights and dloss (float32 [sequences], the
    gradient of the losses); mask and offsets as in the forward call. Zero for masked rows and rows of no sequence.
    ``out`` may be logits itself and shares no memory with anything else. Enqueues one kernel and returns without waiting."""
    index = _device_of("logits", logits)
    for name, t in (("weights", weights), ("dloss", dloss), ("mask", mask), ("offsets", offsets), ("out", out)):
        _same_device(index, name, t)
    dtype, obytes, optr, sequences, rows, experts = _logits(logits, offsets)
    wptr = _states(weights, (sequences, experts), "weights")
    lptr = _states(dloss, (sequences,), "dloss")
    out = _output(out, logits, "logits", weights)
    mptr, (room, arrays) = _mask(mask, rows), _arrays(_rows(logits, "logits"), _rows(out, "out"))
    _call(capi.lib.tb200_balance_loss_backward, "tb200_balance_loss_backward", index, arrays[0], dtype, wptr, lptr, mptr,
          optr, obytes, sequences, rows, experts, arrays[1], _raw_stream(index))
    _rooms.append(room)
    return out
