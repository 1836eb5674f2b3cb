"""Refusals of the recurrence's entry points: nothing here touches a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import thrust_b200 as tb
from thrust_b200 import _capi as capi


def shape(sequences=2, rows=10, channels=8, heads=8, dtype=capi.F32, gate_dtype=capi.F32, log=0, offset_bytes=0, fill=0):
    return capi.RecurrenceShape(sequences, rows, channels, heads, dtype, gate_dtype, log, offset_bytes, fill)


def size(s, back=False):
    need = C.c_size_t(0)
    call = capi.lib.tb200_linear_recurrence_backward if back else capi.lib.tb200_linear_recurrence
    return call(None, C.byref(need), C.byref(s), *(None,) * (10 if back else 7)), need.value


def test_size_queries_answer_without_a_gpu():
    for back in (False, True):
        rc, need = size(shape(), back)
        assert rc == 0 and need >= 256
        for bad in (dict(dtype=capi.F64), dict(dtype=capi.BF16, gate_dtype=capi.F16), dict(dtype=capi.I32)):
            assert size(shape(**bad), back)[0] == capi.ERR_UNSUPPORTED
        for bad in (dict(channels=0), dict(heads=0), dict(heads=3), dict(offset_bytes=2)):
            assert size(shape(**bad), back)[0] == capi.ERR_INVALID_ARGUMENT
        for bad in (dict(channels=1 << 25, heads=1), dict(sequences=1 << 40), dict(rows=1 << 50)):
            assert size(shape(**bad), back)[0] == capi.ERR_UNSUPPORTED
    assert capi.lib.tb200_linear_recurrence(None, None, C.byref(shape()), *(None,) * 7) == capi.ERR_INVALID_ARGUMENT


def test_rows_of_all_sequences_stay_in_range():
    """Their number is a product: one that passes 64 bits must not come back as a small scratch."""
    for back in (False, True):
        for sequences, rows in (((1 << 31) - 1, 1 << 40), (1 << 30, 1 << 34), (1 << 20, (1 << 20) + 1), (3, 1 << 39)):
            assert size(shape(sequences=sequences, rows=rows), back)[0] == capi.ERR_UNSUPPORTED
        for sequences, rows, offsets in ((1 << 20, 1 << 20, 0), (1, 1 << 40, 0), ((1 << 31) - 1, 1 << 40, 8), ((1 << 31) - 1, 0, 0)):
            rc, need = size(shape(sequences=sequences, rows=rows, offset_bytes=offsets), back)
            # a tile of 64 rows of 8 channels takes 12 bytes a channel at least
            assert rc == 0 and need >= (rows if offsets else rows * sequences) // 64 * 8 * 12


def test_arguments_are_checked_before_any_device_work():
    s, need = shape(), C.c_size_t(1 << 20)
    fake = 0x7f0000000100  # never dereferenced
    good, odd = capi.Rows(fake, 8, 80), capi.Rows(fake + 2, 8, 80)
    call = capi.lib.tb200_linear_recurrence

    def run(temp=fake, bytes_=need, shp=s, off=None, g=good, x=good, y=good):
        return call(temp, C.byref(bytes_), C.byref(shp), off, C.byref(g), C.byref(x), C.byref(y), None, None, None)

    assert run(temp=fake + 8) == capi.ERR_INVALID_ARGUMENT
    assert run(bytes_=C.c_size_t(16)) == capi.ERR_TEMP_TOO_SMALL
    assert run(x=odd) == capi.ERR_INVALID_ARGUMENT
    assert run(y=capi.Rows(None, 8, 80)) == capi.ERR_INVALID_ARGUMENT
    assert run(shp=shape(offset_bytes=4)) == capi.ERR_INVALID_ARGUMENT           # no offsets
    assert run(shp=shape(offset_bytes=8), off=fake + 4) == capi.ERR_INVALID_ARGUMENT
    step = capi.lib.tb200_linear_recurrence_step

    def one(state=fake, slots=4, stride=8, idx=None, bytes_=0, rows=3, channels=8, heads=8, dt=capi.F32, gd=capi.F32, x=good):
        return step(state, slots, stride, idx, bytes_, C.byref(good), C.byref(x), C.byref(good), rows, channels, heads, dt, gd,
                    0, None)

    assert one(rows=0) == 0
    assert one(dt=capi.F64) == capi.ERR_UNSUPPORTED and one(dt=capi.F16, gd=capi.BF16) == capi.ERR_UNSUPPORTED
    assert one(rows=5) == capi.ERR_INVALID_ARGUMENT and one(stride=7) == capi.ERR_INVALID_ARGUMENT
    assert one(bytes_=4) == capi.ERR_INVALID_ARGUMENT and one(bytes_=3) == capi.ERR_INVALID_ARGUMENT
    assert one(heads=5) == capi.ERR_INVALID_ARGUMENT and one(x=odd) == capi.ERR_INVALID_ARGUMENT
    assert one(idx=fake, bytes_=4, rows=65537) == capi.ERR_UNSUPPORTED
    assert one(state=fake + 2) == capi.ERR_INVALID_ARGUMENT


def test_states_off_their_boundary_are_refused():
    s, need, fake = shape(), C.c_size_t(1 << 20), 0x7f0000000100  # never dereferenced
    # an array that is refused later on, so that nothing reaches a device whichever check comes first
    good, none = C.byref(capi.Rows(fake, 8, 80)), C.byref(capi.Rows(None, 8, 80))
    for rows in (10, 0):
        s = shape(rows=rows)
        for which in range(2):
            states = [None, None]
            states[which] = fake + 2
            assert capi.lib.tb200_linear_recurrence(fake, C.byref(need), C.byref(s), None, good, good, none, *states,
                                                    None) == capi.ERR_INVALID_ARGUMENT
        for which in range(3):
            states = [None] * 3
            states[which] = fake + 1
            assert capi.lib.tb200_linear_recurrence_backward(fake, C.byref(need), C.byref(s), None, good, good, good, good, none,
                                                             *states, None) == capi.ERR_INVALID_ARGUMENT


def test_python_front_end_refuses_cpu_tensors():
    z = torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="CUDA"):
        tb.linear_recurrence(z, z)
    with pytest.raises(ValueError, match="CUDA"):
        tb.linear_recurrence_backward(z, z, z)
    with pytest.raises(ValueError, match="CUDA"):
        tb.linear_recurrence_step(z[0], z[0], z[0])
    with pytest.raises(TypeError):  # no other algorithm takes the 16-bit floating types
        tb.tb200_dtype(torch.zeros(2, dtype=torch.bfloat16))
    assert capi.lib.tb200_scan(None, C.byref(C.c_size_t(0)), None, None, 4, capi.BF16, 0, None, None) == capi.ERR_UNSUPPORTED


def rows_at(address):
    r = capi.Rows.from_address(address)
    return r.data, r.row_stride, r.sequence_stride


@pytest.mark.parametrize("interrupted", ["_new", "_scratch", "_raw_stream", "_call"])
def test_a_call_within_a_call_keeps_its_arrays(monkeypatch, interrupted):
    """A finaliser or a signal handler may make one of these calls while another one is being put together."""
    ops = tb.model_ops
    seen, armed = [], []
    small = torch.zeros(1, 2, 3)
    inner = {"recurrence": lambda: ops.linear_recurrence(small, small, sync=False),
             "balance": lambda: ops.balance_loss_backward(small[0], small[0, :1].contiguous(), torch.zeros(1))}

    def record(function, what, index, *args):
        seen.append((what, [rows_at(a) for a in args if isinstance(a, int) and a in rooms()]))

    def rooms():
        return {address for room in all_rooms for address in room.at}

    all_rooms, room_init = [], ops._Room.__init__
    monkeypatch.setattr(ops._Room, "__init__", lambda self: (room_init(self), all_rooms.append(self))[0])
    monkeypatch.setattr(ops, "_rooms", [])
    monkeypatch.setattr(ops, "_device_of", lambda name, t: 0)
    monkeypatch.setattr(ops, "_same_device", lambda index, name, t: None)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(ops, "_call", record)
    plain = getattr(ops, interrupted)

    def interrupt(*args):
        if armed:
            armed.pop()()
        return plain(*args)

    monkeypatch.setattr(ops, interrupted, interrupt)
    x, gate = torch.zeros(2, 50, 8), torch.zeros(2, 50, 4)
    state, row = torch.zeros(7, 8), torch.zeros(5, 8)
    z, ids = torch.zeros(40, 16), torch.zeros(40, 2, dtype=torch.int64)
    calls = {"tb200_linear_recurrence": (lambda: ops.linear_recurrence(x, gate, sync=False), [gate, x]),
             "tb200_linear_recurrence_backward": (lambda: ops.linear_recurrence_backward(gate, x, x, sync=False), [gate, x, x]),
             "tb200_linear_recurrence_step": (lambda: ops.linear_recurrence_step(state, row, row), [row, row]),
             "tb200_balance_loss": (lambda: ops.balance_loss(z, ids, sync=False), [z]),
             "tb200_balance_loss_backward": (lambda: ops.balance_loss_backward(z, z[:1].contiguous(), torch.zeros(1)), [z])}
    for what, (call, inputs) in calls.items():
        for other in inner.values():
            del seen[:]
            armed[:] = [other]
            call()
            found = [arrays for name, arrays in seen if name == what and len(arrays) >= len(inputs) and
                     arrays[0][0] == inputs[0].data_ptr()]
            assert len(found) == 1, (what, interrupted, seen)
            for got, t in zip(found[0], inputs):
                assert got == (t.data_ptr(), t.stride(-2), t.stride(0) if t.dim() == 3 else 0), (what, interrupted)
    assert 1 <= len(all_rooms) <= 2  # given back and used again


def cells(t):
    """The bytes of a tensor, one by one."""
    at = np.array([t.data_ptr()])
    for s, n in zip(t.stride(), t.shape):
        at = (at[:, None] + np.arange(n) * s * t.element_size()).reshape(-1)
    return (at[:, None] + np.arange(t.element_size())).reshape(-1)


def test_arrays_that_share_memory_are_found():
    """Against the sets of bytes: never called apart when they are not, and slices as they are made are called apart."""
    ops, rng = tb.model_ops, np.random.default_rng(0)
    buffer = torch.zeros(4000)
    shared = apart = known = 0
    for _ in range(4000):
        a, b = (torch.as_strided(buffer, (int(rng.integers(1, 4)), int(rng.integers(1, 6)), int(rng.integers(1, 7))),
                                 (int(rng.integers(0, 40)), int(rng.integers(0, 12)), 1), int(rng.integers(0, 60))) for _ in range(2))
        if rng.random() < 0.4:
            b = torch.as_strided(buffer, (*a.shape[:2], b.shape[2]), a.stride(), b.storage_offset())
        if rng.random() < 0.3:
            b = b.view(torch.float16)
        ca, cb = cells(a), cells(b)
        if ops._rows_apart(a):
            assert len(set(ca)) == len(ca)
        together = bool(set(ca) & set(cb))
        shared += together
        apart += not together
        if ops._disjoint(a, b):
            known += 1
            assert not together, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
    assert shared > 500 and known > 0.7 * apart
    wide = torch.zeros(3, 20, 24)
    for a, b in ((wide[:, :, :8], wide[:, :, 8:16]), (wide[:, :10, :8], wide[:, 10:, :8]), (wide[:, ::2], wide[:, 1::2]),
                 (wide[0], wide[1]), (wide[:, :, :8].transpose(0, 1), wide[:, :, 16:].transpose(0, 1)), (wide[:, :5], wide[:, 10:15]),
                 (wide[:, :, :4], wide[:, :, 4:12]), (wide[:2, :, :8], wide[1:, :, 8:16]), (wide[:, :0], wide[:, :0])):
        assert ops._disjoint(a, b) and ops._disjoint(b, a) and ops._rows_apart(a) and ops._rows_apart(b)
    for a, b in ((wide[:, :-1], wide[:, 1:]), (wide[..., :8], wide[..., 7:15]), (wide, wide), (wide[:2], wide[1:])):
        assert not ops._disjoint(a, b) and not ops._disjoint(b, a)


def test_outputs_that_race_are_refused():
    ops = tb.model_ops
    buffer = torch.zeros(2, 30, 16)
    x = buffer[:, :20, :8]
    assert ops._output(x, x, "x") is x and ops._output(None, x, "x").shape == x.shape
    same = buffer[:, :20, :8]
    assert ops._output(same, x, "x") is same
    one = torch.as_strided(x, (1, 20, 8), (7, 16, 1))  # the distance of one sequence means nothing
    assert ops._output(one, x[:1], "x") is one
    assert ops._output(buffer[:, 5:25, 8:], x, "x", buffer[:, 6:26, :8], None) is not None
    square = torch.zeros(3, 3, 4)
    for out, like, others in ((buffer[:, 1:21, :8], x, ()), (buffer[:, :20, 4:12], x, ()), (square.transpose(0, 1), square, ()),
                              (torch.as_strided(torch.zeros(400), (2, 20, 8), (200, 7, 1)), x, ()),
                              (torch.as_strided(torch.zeros(400), (2, 20, 8), (0, 8, 1)), x, ()),
                              (torch.as_strided(torch.zeros(400), (2, 20, 8), (159, 8, 1)), x, ()),
                              (buffer[:, :20, 8:], x, (buffer[..., 7:9],)), (buffer[:, :20, 8:], x, (None, buffer[0, 3:5]))):
        with pytest.raises(ValueError, match="share"):
            ops._output(out, like, "x", *others)


def test_scratch_with_gaps_is_refused():
    """The library writes to all bytes from the first one on: an expanded tensor has one of them."""
    ops, like = tb.model_ops, torch.zeros(1)
    whole = torch.zeros(4096, dtype=torch.uint8)
    assert ops._scratch(4096, like, whole) is whole
    assert ops._scratch(5000, like, whole).numel() == 5000 and ops._scratch(300, like, None).numel() == 300
    for temp in (whole[:1].expand(4096), whole[::2], whole.view(64, 64).T):
        with pytest.raises(ValueError, match="contiguous"):
            ops._scratch(1000, like, temp)
