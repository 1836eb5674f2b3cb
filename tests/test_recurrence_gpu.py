"""The gated linear recurrence against a row-by-row evaluation in 64 bits.

Tolerances. A state is advanced in 32 bits by one fused multiply-add (and one more addition near a gate of one): two
roundings a row of at most 2^-24 each of the largest state, kept by the gates for the memory m = 1 / (1 - max a) rows at
most, or for the length of the sequence where that is shorter; the gate itself is off by at most 2^-22 of it (away from
one) or of 1 - a (near one), and the products over stretches by a rounding a row. Together less than
8 * 2^-24 * min(m, rows) * max|state|, to which an output of fewer bits adds half a step of its own. Gradients of gates
are products of two such values, summed over the channels that share a gate.
"""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

import thrust_b200 as tb
from thrust_b200 import _capi as capi

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 2.0 ** -24


def spans_of(x, offsets):
    """[(flat rows as an index, sequence)] of every sequence over x viewed as [.., rows, channels]."""
    if offsets is None:
        return [(b, slice(None)) for b in range(x.shape[0])]
    return [(slice(int(a), int(b)),) for a, b in zip(offsets[:-1], offsets[1:])]


def reference(x, gate, initial, offsets, log_gate):
    x, gate = x.double().cpu(), gate.double().cpu()
    a = gate.exp() if log_gate else gate
    a = a.repeat_interleave(x.shape[-1] // gate.shape[-1], -1)
    spans = spans_of(x, offsets)
    h0 = torch.zeros(len(spans), x.shape[-1], dtype=torch.float64) if initial is None else initial.double().cpu()
    y, final = torch.zeros_like(x), h0.clone()
    for i, at in enumerate(spans):
        h = h0[i]
        for t in range(x[at].shape[0]):
            h = (a[at][t] * h if t or initial is not None else 0.0) + x[at][t]
            y[at][t] = h
        final[i] = h
    return y, final


def reference_backward(gate, y, dy, initial, dfinal, offsets, log_gate):
    gate, y, dy = gate.double().cpu(), y.double().cpu(), dy.double().cpu()
    a = gate.exp() if log_gate else gate
    per = y.shape[-1] // gate.shape[-1]
    a = a.repeat_interleave(per, -1)
    spans = spans_of(y, offsets)
    zeros = torch.zeros(len(spans), y.shape[-1], dtype=torch.float64)
    h0 = zeros if initial is None else initial.double().cpu()
    p0 = zeros.clone() if dfinal is None else dfinal.double().cpu().clone()
    dx, da = torch.zeros_like(y), torch.zeros_like(y)
    for i, at in enumerate(spans):
        p = p0[i]
        for t in reversed(range(y[at].shape[0])):
            g = dy[at][t] + p
            dx[at][t] = g
            da[at][t] = g * (y[at][t - 1] if t else h0[i])
            p = a[at][t] * g
        p0[i] = p
    if log_gate:
        da = da * a
    size = da.abs().unflatten(-1, (-1, per)).sum(-1)
    return dx, da.unflatten(-1, (-1, per)).sum(-1), p0, size


def make(rng, lead, channels, heads, dtype, gate_dtype, log_gate, device, dmin=2e-3):
    rate = np.exp(rng.uniform(np.log(dmin), np.log(3.0), size=(*lead, heads)))
    gate = -rate if log_gate else np.exp(-rate) * rng.choice([1.0, -1.0], p=[0.9, 0.1], size=rate.shape)
    x = rng.standard_normal((*lead, channels))
    return (torch.from_numpy(x).to(device, TYPES[dtype]), torch.from_numpy(gate).to(device, TYPES[gate_dtype]))


def close(got, want, dtype, memory, scale=None, what=""):
    """|got - want| within the derived bound, element by element."""
    got = got.double().cpu()
    scale = want.abs().max().item() if scale is None else scale
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bound = 8 * EPS * memory * scale + half * want.abs() * (1 + 1e-6) + tiny
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= bound).all(), (what, float((off / bound).max()))


CASES = [
    # sequences (or lengths of packed ones), rows, channels, heads, x, gate, log
    (1, 1, 1, 1, "f32", "f32", False),
    (3, 5, 7, 7, "bf16", "f32", True),
    (2, 64, 128, 128, "f32", "f32", True),
    (2, 65, 132, 132, "bf16", "bf16", False),
    (1, 700, 256, 256, "bf16", "f32", True),
    (2, 333, 136, 136, "f16", "f16", True),
    (3, 129, 96, 6, "bf16", "bf16", False),      # heads of 16
    (2, 140, 200, 5, "f32", "f32", True),        # heads of 40: three to a block of 128 channels
    (1, 90, 960, 10, "f16", "f32", True),        # heads of 96
    (2, 70, 512, 2, "bf16", "f32", False),       # heads of 256: two blocks each
    (1, 66, 300, 1, "f32", "f32", True),         # one gate for a row
    (2, 75, 51, 17, "bf16", "bf16", True),       # heads of 3, odd rows
    (2, 75, 70, 2, "f16", "f32", False),         # heads of 35
    (300, 3, 40, 40, "bf16", "bf16", False),     # many short sequences
    ([5, 0, 1, 130, 0, 64, 3], None, 128, 128, "bf16", "f32", True),
    ([0, 0, 257, 1, 1, 1], None, 260, 260, "f32", "f32", False),
    ([40, 64, 24, 100, 0], None, 160, 4, "f16", "f32", True),
    ([1], None, 33, 33, "bf16", "bf16", True),
    ([31, 600], None, 768, 3, "bf16", "f32", True),
]


def build(case, device, seed, strided=False, int_dtype=torch.int32):
    seqs, rows, channels, heads, dtype, gate_dtype, log_gate = case
    rng = np.random.default_rng(seed)
    packed = isinstance(seqs, list)
    count = len(seqs) if packed else seqs
    lead = (sum(seqs),) if packed else (seqs, rows)
    x, gate = make(rng, lead, channels, heads, dtype, gate_dtype, log_gate, device)
    offsets = torch.from_numpy(np.cumsum([0, *seqs])).to(device, int_dtype) if packed else None
    initial = torch.from_numpy(rng.standard_normal((count, channels)).astype(np.float32)).to(device)
    return x, gate, initial, offsets, rng


def memory_of(gate, log_gate, rows):
    a = gate.double().exp() if log_gate else gate.double().abs()
    top = float(a.max()) if a.numel() else 0.0
    return min(rows, 1.0 / max(1e-9, 1.0 - top)) + 1


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
@pytest.mark.parametrize("with_initial", [False, True])
def test_forward(cuda_device, case, with_initial):
    x, gate, initial, offsets, _ = build(case, cuda_device, 11, int_dtype=torch.int64 if with_initial else torch.int32)
    initial = initial if with_initial else None
    y, final = tb.linear_recurrence(x, gate, initial=initial, offsets=offsets, log_gate=case[6])
    wy, wf = reference(x, gate, initial, offsets, case[6])
    m = memory_of(gate, case[6], x.shape[-2])
    scale = max(float(wy.abs().max()), float(wf.abs().max()))
    close(y, wy, x.dtype, m, scale, "y")
    close(final, wf, torch.float32, m, scale, "final")
    again, final2 = tb.linear_recurrence(x, gate, initial=initial, offsets=offsets, log_gate=case[6])
    assert torch.equal(y, again) and torch.equal(final, final2)  # reproducible to the bit


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
@pytest.mark.parametrize("with_states", [False, True])
def test_backward(cuda_device, case, with_states):
    x, gate, initial, offsets, rng = build(case, cuda_device, 12)
    initial = initial if with_states else None
    y = reference(x, gate, initial, offsets, case[6])[0].to(cuda_device, x.dtype)
    dy = torch.from_numpy(rng.standard_normal(tuple(x.shape))).to(cuda_device, x.dtype)
    count = offsets.numel() - 1 if offsets is not None else x.shape[0]
    dfinal = None
    if with_states:
        dfinal = torch.from_numpy(rng.standard_normal((count, x.shape[-1])).astype(np.float32)).to(cuda_device)
    got = tb.linear_recurrence_backward(gate, y, dy, initial=initial, dfinal=dfinal, offsets=offsets, log_gate=case[6])
    wx, wg, wi, size = reference_backward(gate, y, dy, initial, dfinal, offsets, case[6])
    m = memory_of(gate, case[6], x.shape[-2])
    scale = max(float(wx.abs().max()), float(wi.abs().max()))
    close(got[0], wx, dy.dtype, m, scale, "dx")
    per = x.shape[-1] // gate.shape[-1]
    before = float(y.abs().max()) if initial is None else max(float(y.abs().max()), float(initial.abs().max()))
    # a product with y, and the sum over a head's channels in a tree of at most per roundings of its absolute sum
    close(got[1], wg, gate.dtype, m, scale * before * per + float(size.max()), "dgate")
    close(got[2], wi, torch.float32, m, scale, "dinitial")
    again = tb.linear_recurrence_backward(gate, y, dy, initial=initial, dfinal=dfinal, offsets=offsets, log_gate=case[6])
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_gradients_agree_with_differences(cuda_device):
    """The whole backward call against central differences of the definition in 64 bits."""
    rng = np.random.default_rng(3)
    for log_gate, heads in ((True, 2), (False, 8)):
        x, gate = make(rng, (7,), 8, heads, "f32", "f32", log_gate, cuda_device, dmin=0.05)
        offsets = torch.tensor([0, 3, 3, 7], dtype=torch.int32, device=cuda_device)
        initial = torch.from_numpy(rng.standard_normal((3, 8)).astype(np.float32)).to(cuda_device)
        wy = torch.from_numpy(rng.standard_normal((7, 8)).astype(np.float32))
        wf = torch.from_numpy(rng.standard_normal((3, 8)).astype(np.float32))

        def loss(x, gate, initial):
            y, f = reference(x, gate, initial, offsets, log_gate)
            return float((y * wy.double()).sum() + (f * wf.double()).sum())

        y, _ = tb.linear_recurrence(x, gate, initial=initial, offsets=offsets, log_gate=log_gate)
        got = tb.linear_recurrence_backward(gate, y, wy.to(cuda_device), initial=initial, dfinal=wf.to(cuda_device),
                                            offsets=offsets, log_gate=log_gate)
        args = [x.double().cpu(), gate.double().cpu(), initial.double().cpu()]
        for which, g in enumerate(got):
            for _ in range(12):
                at = tuple(int(rng.integers(n)) for n in g.shape)
                step = 1e-5
                hi, lo = [a.clone() for a in args], [a.clone() for a in args]
                hi[which][at] += step
                lo[which][at] -= step
                diff = (loss(*hi) - loss(*lo)) / (2 * step)
                # differences: cubes of the step times third derivatives (at most of order 7!), and 64-bit roundings
                assert abs(diff - float(g[at])) <= 1e-4 * max(1.0, float(g.abs().max())), (log_gate, which, at)


@pytest.mark.parametrize("dtype,channels,heads", [("bf16", 128, 128), ("f32", 36, 9), ("f16", 13, 13)])
def test_strides_and_orders(cuda_device, dtype, channels, heads):
    """Slices of a fused projection, time-major batches, rows that begin at odd elements, broadcast gates."""
    rng = np.random.default_rng(5)
    wide = torch.from_numpy(rng.standard_normal((3, 70, 2 * channels + 5))).to(cuda_device, TYPES[dtype])
    rate = torch.from_numpy(rng.uniform(0.01, 1.0, size=(70, 3, heads))).to(cuda_device, torch.float32)
    x, gate = wide[:, :, 1:1 + channels], (-rate).transpose(0, 1)
    plain = tb.linear_recurrence(x.contiguous(), gate.contiguous(), log_gate=True)
    other = torch.empty_like(wide)  # a slice that begins at the allocation, and an output slice of the same array
    other[:, :, :channels].copy_(x)
    for xv, out in ((x, None), (x, torch.empty(70, 3, channels, dtype=x.dtype, device=cuda_device).transpose(0, 1)),
                    (x.transpose(0, 1).contiguous().transpose(0, 1), None),
                    (other[:, :, :channels], other[:, :, channels + 1:2 * channels + 1])):
        y, final = tb.linear_recurrence(xv, gate, log_gate=True, out=out)
        tol = 8 * EPS * 71 * float(plain[1].abs().max()) + torch.finfo(x.dtype).eps * float(plain[0].float().abs().max())
        assert float((y.float() - plain[0].float()).abs().max()) <= tol
        assert float((final - plain[1]).abs().max()) <= tol
    x = wide[:, :, :channels]
    decay = (-rate[0, 0]).expand(3, 70, heads)  # one decay for all rows
    a = tb.linear_recurrence(x, decay, log_gate=True)
    b = tb.linear_recurrence(x.contiguous(), decay.contiguous(), log_gate=True)
    assert float((a[1] - b[1]).abs().max()) <= 8 * EPS * 71 * float(b[1].abs().max())
    dy = wide[:, :, channels:2 * channels]
    ga = tb.linear_recurrence_backward(decay, a[0].transpose(0, 1).contiguous().transpose(0, 1), dy, log_gate=True)
    gb = tb.linear_recurrence_backward(decay.contiguous(), a[0], dy.contiguous(), log_gate=True)
    for u, v in zip(ga, gb):
        assert float((u.float() - v.float()).abs().max()) <= (torch.finfo(u.dtype).eps + 1e-4) * float(v.float().abs().max())


def test_in_place_and_rows_behind_the_last_sequence(cuda_device):
    rng = np.random.default_rng(6)
    x, gate = make(rng, (150,), 64, 64, "bf16", "f32", True, cuda_device)
    offsets = torch.tensor([0, 70, 70, 101], dtype=torch.int64, device=cuda_device)
    want, wf = tb.linear_recurrence(x, gate, offsets=offsets, log_gate=True)
    assert not want[101:].any()
    work = x.clone()
    y, final = tb.linear_recurrence(work, gate, offsets=offsets, log_gate=True, out=work)
    assert y is work and torch.equal(work[:101], want[:101]) and torch.equal(work[101:], x[101:])
    assert torch.equal(final, wf) and not final[1].any()
    garbage_x, garbage_g = x.clone(), gate.clone()
    garbage_x[101:] = float("nan")
    garbage_g[101:] = float("inf")
    got, gf = tb.linear_recurrence(garbage_x, garbage_g, offsets=offsets, log_gate=True)
    assert torch.equal(got, want) and torch.equal(gf, wf)
    dy = torch.randn_like(x)
    dy_g = dy.clone()
    dy_g[101:] = float("nan")
    y_g = want.clone()
    y_g[101:] = float("nan")
    a = tb.linear_recurrence_backward(gate, want, dy, offsets=offsets, log_gate=True)
    b = tb.linear_recurrence_backward(garbage_g, y_g, dy_g, offsets=offsets, log_gate=True)
    assert all(torch.equal(u, v) for u, v in zip(a, b)) and not a[0][101:].any() and not a[1][101:].any()


def test_sequences_do_not_touch_each_other(cuda_device):
    """NaN and infinities of one sequence stay in it, also where it shares a tile with others."""
    x = torch.ones(200, 8, device=cuda_device)
    gate = torch.full((200, 8), 0.5, device=cuda_device)
    offsets = torch.tensor([0, 10, 20, 150, 200], dtype=torch.int32, device=cuda_device)
    clean, cf = tb.linear_recurrence(x, gate, offsets=offsets)
    x[12, 3], x[60, 4] = float("nan"), float("inf")
    y, final = tb.linear_recurrence(x, gate, offsets=offsets)
    for s, (b, e) in enumerate(((0, 10), (10, 20), (20, 150), (150, 200))):
        for c in range(8):
            bad = {(1, 3): 12, (2, 4): 60}.get((s, c))
            if bad is None:
                assert torch.equal(y[b:e, c], clean[b:e, c]) and final[s, c] == cf[s, c]
            else:
                assert torch.equal(y[b:bad, c], clean[b:bad, c]) and not torch.isfinite(y[bad:e, c]).any()
    gate[30:] = 0.5
    gate[40, 2] = 0.0  # a gate of zero forgets
    y, _ = tb.linear_recurrence(x, gate, offsets=offsets)
    assert y[40, 2] == 1.0
    y, _ = tb.linear_recurrence(torch.ones(1, 3, 4, device=cuda_device), torch.tensor([-1.0, float("-inf"), -1.0], device=cuda_device)
                                .view(1, 3, 1), log_gate=True)
    assert (y[0, 1] == 1.0).all()


def test_memory_near_one(cuda_device):
    """Gates so close to one that a rounding of the gate, or a leaning exponential, would show: constant decays."""
    rows = 20000
    for log_gate in (True, False):
        rate = torch.tensor([1e-4, 3e-4, 1e-3, 1e-2], device=cuda_device)
        gate = (-rate if log_gate else 1 - rate).expand(1, rows, 4)
        x = torch.ones(1, rows, 4, device=cuda_device)
        y, final = tb.linear_recurrence(x, gate, log_gate=log_gate)
        a = gate[0, 0].double().exp() if log_gate else gate[0, 0].double()
        want = (1 - a ** rows) / (1 - a)
        # the state's own roundings, half a step a row at random: far below this; a gate off by 2^-25 gives 3e-4
        assert float(((final[0].double() - want) / want).abs().max()) <= 2e-5


def test_empty_shapes(cuda_device):
    z = torch.zeros(3, 0, 8, device=cuda_device)
    initial = torch.randn(3, 8, device=cuda_device)
    y, final = tb.linear_recurrence(z, z, initial=initial)
    assert y.shape == z.shape and torch.equal(final, initial)
    assert not tb.linear_recurrence(z, z)[1].any()
    dx, dg, di = tb.linear_recurrence_backward(z, z, z, dfinal=initial)
    assert torch.equal(di, initial) and dx.shape == dg.shape == z.shape
    none = torch.zeros(0, 4, 8, device=cuda_device)
    assert tb.linear_recurrence(none, none)[1].shape == (0, 8)
    offsets = torch.zeros(4, dtype=torch.int32, device=cuda_device)  # only empty sequences in front of some rows
    x = torch.randn(5, 8, device=cuda_device)
    y, final = tb.linear_recurrence(x, x, initial=initial, offsets=offsets)
    assert not y.any() and torch.equal(final, initial)
    y, final = tb.linear_recurrence(x, x, offsets=offsets[:1])
    assert not y.any() and final.shape == (0, 8)


def test_bad_offsets_are_reported(cuda_device):
    x = torch.randn(100, 8, device=cuda_device)
    for bad in ([0, 50, 40, 100], [1, 100], [0, 101], [-1, 100], [0, -5, 100]):
        offsets = torch.tensor(bad, dtype=torch.int32, device=cuda_device)
        with pytest.raises(tb.Tb200Error) as e:
            tb.linear_recurrence(x, x, offsets=offsets)
        assert e.value.code == capi.ERR_INVALID_ARGUMENT
        with pytest.raises(tb.Tb200Error):
            tb.linear_recurrence_backward(x, x, x, offsets=offsets)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_bad_offsets_without_rows_or_sequences(cuda_device, dtype):
    some, none = torch.randn(5, 8, device=cuda_device), torch.zeros(0, 8, device=cuda_device)
    cases = [(none, [0, 3], True), (none, [0, 0, 1, 0], True), (none, [-1, 0], True), (none, [1], True), (some, [7], True),
             (some, [-2], True), (some, [3], True), (none, [0, 0, 0], False), (none, [0], False), (some, [0], False),
             (none, [0] * 700, False), (none, [0] * 600 + [1] + [0] * 99, True)]
    for x, values, bad in cases:
        offsets = torch.tensor(values, dtype=dtype, device=cuda_device)
        ids = torch.zeros(x.shape[0], 2, dtype=torch.int64, device=cuda_device)
        for call in (lambda: tb.linear_recurrence(x, x, offsets=offsets), lambda: tb.balance_loss(x, ids, offsets=offsets),
                     lambda: tb.linear_recurrence(x, x, offsets=offsets, out=torch.empty_like(x)),
                     lambda: tb.linear_recurrence_backward(x, x, x, offsets=offsets)):
            if bad:
                with pytest.raises(tb.Tb200Error) as e:
                    call()
                assert e.value.code == capi.ERR_INVALID_ARGUMENT
            else:
                call()


@pytest.mark.parametrize("rows,slots,channels,heads,dtype,gate_dtype,log_gate", [
    (1, 1, 1, 1, "f32", "f32", False), (5, 9, 128, 128, "bf16", "f32", True), (33, 40, 1000, 25, "f16", "f16", False),
    (7, 7, 51, 17, "bf16", "bf16", True), (130, 300, 2048, 8, "bf16", "f32", False)])
def test_step(cuda_device, rows, slots, channels, heads, dtype, gate_dtype, log_gate):
    rng = np.random.default_rng(rows)
    x, gate = make(rng, (rows,), channels, heads, dtype, gate_dtype, log_gate, cuda_device)
    state = torch.from_numpy(rng.standard_normal((slots, channels)).astype(np.float32)).to(cuda_device)
    at = torch.from_numpy(rng.permutation(slots)[:rows]).to(cuda_device, torch.int32 if rows % 2 else torch.int64)
    before = state.clone()
    y = tb.linear_recurrence_step(state, x, gate, slots=at, log_gate=log_gate)
    wy, wf = reference(x[:, None], gate[:, None], before[at.long()], None, log_gate)
    close(y, wy[:, 0], x.dtype, 2, what="y")
    close(state[at.long()], wf, torch.float32, 2, what="state")
    rest = torch.ones(slots, dtype=torch.bool, device=cuda_device)
    rest[at.long()] = False
    assert torch.equal(state[rest], before[rest])
    again = before.clone()
    assert torch.equal(tb.linear_recurrence_step(again[:rows], x, gate, log_gate=log_gate),
                       tb.linear_recurrence_step(before.clone(), x, gate, log_gate=log_gate,
                                                 slots=torch.arange(rows, device=cuda_device)))


def test_step_padding_and_repeated_slots(cuda_device):
    rng = np.random.default_rng(2)
    x, gate = make(rng, (6,), 300, 300, "f32", "f32", False, cuda_device)
    state = torch.randn(4, 300, device=cuda_device)
    before = state.clone()
    slots = torch.tensor([2, -1, 0, 2, 4, 2], device=cuda_device)
    y = tb.linear_recurrence_step(state, x, gate, slots=slots)
    assert not y[1].any() and not y[4].any()
    assert torch.equal(state[1], before[1]) and torch.equal(state[3], before[3])
    one = before.clone()
    for r in (0, 2, 3, 5):  # the same rows one call at a time
        yr = tb.linear_recurrence_step(one, x[r:r + 1], gate[r:r + 1], slots=slots[r:r + 1])
        assert torch.equal(yr[0], y[r])
    assert torch.equal(one, state)
    padded = torch.randn(4, 300 + 20, device=cuda_device)  # a pool with gaps between its states
    view = padded[:, :300].copy_(before)
    tail = padded[:, 300:].clone()
    assert torch.equal(tb.linear_recurrence_step(view, x, gate, slots=slots), y)
    assert torch.equal(view, state) and torch.equal(padded[:, 300:], tail)


def test_prefill_then_steps_is_one_recurrence(cuda_device):
    rng = np.random.default_rng(9)
    x, gate = make(rng, (2, 90), 64, 4, "f32", "f32", True, cuda_device)
    whole, final = tb.linear_recurrence(x, gate, log_gate=True)
    _, state = tb.linear_recurrence(x[:, :80], gate[:, :80], log_gate=True)
    for t in range(80, 90):
        y = tb.linear_recurrence_step(state, x[:, t], gate[:, t], log_gate=True)
        assert float((y - whole[:, t]).abs().max()) <= 8 * EPS * 90 * float(whole.abs().max())
    assert float((state - final).abs().max()) <= 8 * EPS * 90 * float(whole.abs().max())


def test_streams_and_graphs(cuda_device):
    """Two recurrences at once on two streams, and a captured forward and backward pass replayed on new data."""
    rng = np.random.default_rng(4)
    x, gate = make(rng, (4, 300), 256, 256, "bf16", "f32", True, cuda_device)
    want, wf = tb.linear_recurrence(x, gate, log_gate=True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            got.append(tb.linear_recurrence(x, gate, log_gate=True, sync=False))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) and torch.equal(f, wf) for y, f in got)
    sx, sdy = x.clone(), torch.randn_like(x)
    tb.linear_recurrence_backward(gate, want, sdy, log_gate=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, f = tb.linear_recurrence(sx, gate, log_gate=True, sync=False)
        grads = tb.linear_recurrence_backward(gate, y, sdy, log_gate=True, sync=False)
    for k in range(3):
        sx.copy_(x * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        y2, f2 = tb.linear_recurrence(sx, gate, log_gate=True)
        g2 = tb.linear_recurrence_backward(gate, y2, sdy, log_gate=True)
        assert torch.equal(y, y2) and torch.equal(f, f2) and all(torch.equal(a, b) for a, b in zip(grads, g2))


def test_short_sequences_that_lie_apart(cuda_device):
    """Sequences of a few rows in a time-major batch: no two of them lie behind one another."""
    rng = np.random.default_rng(12)
    for rows, channels in ((5, 64), (1, 20), (32, 136)):
        x, gate = make(rng, (40, rows), channels, channels, "bf16", "f32", True, cuda_device)
        apart = x.transpose(0, 1).contiguous().transpose(0, 1)
        a, b = tb.linear_recurrence(x, gate, log_gate=True), tb.linear_recurrence(apart, gate, log_gate=True)
        wy, wf = reference(x, gate, None, None, True)
        for y, final in (a, b):
            close(y, wy, x.dtype, rows, what="y")
            close(final, wf, torch.float32, rows, what="final")
        ga = tb.linear_recurrence_backward(gate, a[0], x, log_gate=True)
        gb = tb.linear_recurrence_backward(gate, a[0], apart, log_gate=True)
        wx, wg, wi, size = reference_backward(gate, a[0], x, None, None, None, True)
        for g in (ga, gb):
            close(g[0], wx, x.dtype, rows, what="dx")
            close(g[1], wg, gate.dtype, rows, float(wx.abs().max() * a[0].float().abs().max().cpu()) + float(size.max()), "dgate")


@pytest.mark.parametrize("case", [
    (400, 40, 520, 520, "bf16", "bf16", True),         # tiles that wait for none: each is a whole sequence
    (400, 40, 523, 523, "bf16", "f32", False),         # the same with one channel a lane
    (300, 33, 640, 20, "f16", "f32", True),            # heads of 32
    (300, 31, 1001, 1001, "f32", "f32", True),         # short ones behind one another, a chain of hundreds of tiles
    (1, 20011, 301, 301, "bf16", "bf16", False),       # one channel a lane in long chains: values through registers
    (1, 20011, 299, 299, "f32", "f32", True),          # and by asynchronous copies
    (2, 9001, 350, 10, "f16", "f16", True),            # heads of 35, over two blocks of channels each
    (1, 15013, 306, 102, "bf16", "f32", False),        # heads of 3
    (1, 15013, 640, 16, "f32", "f32", True),           # heads of 40 in boxes
    ([3000, 0, 1, 64, 4001, 0, 7, 6000, 31], None, 333, 333, "bf16", "f32", True),
    ([1000] * 16 + [0] * 40 + [3] * 50, None, 520, 520, "f32", "f32", False),
], ids=lambda c: "-".join(map(str, c)).replace(" ", "")[:60])
def test_many_tiles_for_each_cta(cuda_device, case):
    """Nine tiles and more for every one of 148 CTAs, so that all rings of the pipeline wrap: against 64 bits, and the same to
    the bit every time."""
    x, gate, initial, offsets, rng = build(case, cuda_device, 21)
    log_gate, per = case[6], case[2] // case[3]
    y, final = tb.linear_recurrence(x, gate, initial=initial, offsets=offsets, log_gate=log_gate)
    wy, wf = reference(x, gate, initial, offsets, log_gate)
    m = memory_of(gate, log_gate, x.shape[-2])
    scale = max(float(wy.abs().max()), float(wf.abs().max()))
    close(y, wy, x.dtype, m, scale, "y")
    close(final, wf, torch.float32, m, scale, "final")
    dy = torch.from_numpy(rng.standard_normal(tuple(x.shape))).to(cuda_device, x.dtype)
    dfinal = torch.from_numpy(rng.standard_normal(tuple(final.shape)).astype(np.float32)).to(cuda_device)
    args = dict(initial=initial, dfinal=dfinal, offsets=offsets, log_gate=log_gate)
    got = tb.linear_recurrence_backward(gate, y, dy, **args)
    wx, wg, wi, size = reference_backward(gate, y, dy, initial, dfinal, offsets, log_gate)
    back = max(float(wx.abs().max()), float(wi.abs().max()))
    close(got[0], wx, dy.dtype, m, back, "dx")
    close(got[1], wg, gate.dtype, m, back * max(float(y.abs().max()), float(initial.abs().max())) * per + float(size.max()), "dgate")
    close(got[2], wi, torch.float32, m, back, "dinitial")
    for _ in range(3):
        again = tb.linear_recurrence(x, gate, initial=initial, offsets=offsets, log_gate=log_gate)
        assert torch.equal(again[0], y) and torch.equal(again[1], final)
        assert all(torch.equal(a, b) for a, b in zip(got, tb.linear_recurrence_backward(gate, y, dy, **args)))


def test_arrays_of_more_than_32_bits(cuda_device):
    """More than 2^32 elements an array: the last rows are those of a run over the last rows alone, since decays of at most
    exp(-0.02) leave nothing of what lies 6000 rows back. Both runs are within the bound of an exact one, and round once."""
    channels, far, near = 2048, (1 << 32) // 2048 + 5000, 6000
    block = torch.randn(1, 4099, channels, device=cuda_device).bfloat16()
    rate = torch.empty(1, 4099, channels, device=cuda_device).uniform_(0.02, 1.0)

    def many(rows):
        return rows.repeat(1, -(-far // rows.shape[1]), 1)[:, :far].contiguous()

    x, gate = many(block), many(torch.exp(-rate).clamp(max=0.98).bfloat16())
    y, final = tb.linear_recurrence(x, gate)
    ly, lf = tb.linear_recurrence(x[:, -2 * near:], gate[:, -2 * near:])

    def agree(a, b, scale):
        bound = 2 * (8 * EPS * 60 * scale + torch.finfo(a.dtype).eps / 2 * (1 + 1e-6) * b.float().abs())
        return bool(((a.float() - b.float()).abs() <= bound).all())

    top = float(ly.abs().max())
    assert agree(y[:, -near:], ly[:, -near:], top) and agree(final, lf, top)
    dx, dgate, dinitial = tb.linear_recurrence_backward(gate, y, x)
    lx, lg, _ = tb.linear_recurrence_backward(gate[:, -2 * near:], y[:, -2 * near:], x[:, -2 * near:])
    assert agree(dx[:, -near:], lx[:, -near:], float(lx.abs().max()))
    assert agree(dgate[:, -near:], lg[:, -near:], float(lx.abs().max()) * top)
    fx, fg, fi = tb.linear_recurrence_backward(gate[:, :2 * near], y[:, :2 * near], x[:, :2 * near])
    assert agree(dx[:, :near], fx[:, :near], float(fx.abs().max())) and agree(dinitial, fi, float(fx.abs().max()))
    assert agree(dgate[:, :near], fg[:, :near], float(fx.abs().max()) * top)
    del x, gate, y, dx, dgate
    pool = torch.zeros((1 << 32) // channels + 3, channels, device=cuda_device)  # and a pool of such states
    pool[-2:] = 1.0
    slots = torch.tensor([pool.shape[0] - 1, 0, pool.shape[0] - 2, 1], device=cuda_device)
    step = torch.arange(4.0, device=cuda_device)[:, None].expand(4, channels).contiguous()
    out = tb.linear_recurrence_step(pool, step, torch.full_like(step, 0.5), slots=slots)
    assert torch.equal(out[:, 0], torch.tensor([0.5, 1.0, 2.5, 3.0], device=cuda_device)) and torch.equal(pool[slots], out)


def test_calls_from_several_threads(cuda_device):
    """Four threads with a stream each, all operators of a layer over arrays of different strides: nobody's arguments or
    results are another one's."""
    def layer(i):
        rng = np.random.default_rng(i)
        channels, experts = 64 + 8 * i, 8 + i
        wide = torch.from_numpy(rng.standard_normal((200 + 30 * i, channels + 8 * i))).to(cuda_device, torch.float32)
        x, gate = wide[:, :channels], -wide[:, :channels].abs() - 0.01
        offsets = torch.tensor([0, 50 + i, 190 + i], dtype=torch.int32, device=cuda_device)
        ids = torch.from_numpy(rng.integers(0, experts, size=(x.shape[0], 2))).to(cuda_device)
        dloss = torch.ones(2, device=cuda_device)
        pool = torch.zeros(4 + i, channels, device=cuda_device)

        def run():
            pool.zero_()
            y, final = tb.linear_recurrence(x, gate, offsets=offsets, log_gate=True)
            grads = tb.linear_recurrence_backward(gate, y, x, offsets=offsets, log_gate=True)
            z = y[:, :experts]
            loss, counts, weights = tb.balance_loss(z, ids, offsets=offsets)
            dz = tb.balance_loss_backward(z, weights, dloss, offsets=offsets)
            step = tb.linear_recurrence_step(pool, x[:3], gate[:3], log_gate=True)
            return [y, final, *grads, loss, counts, weights, dz, step, pool.clone(), *tb.expert_counts(ids, experts)]
        return run

    layers = [layer(i) for i in range(4)]
    want = [run() for run in layers]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.device(cuda_device), torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                for a, b in zip(layers[i](), want[i]):
                    if not torch.equal(a, b):
                        return f"thread {i}"
        return None

    with ThreadPoolExecutor(4) as pool:
        assert list(pool.map(work, range(4))) == [None] * 4


@pytest.mark.parametrize("heads", [96, 3])
def test_one_long_sequence(cuda_device, heads):
    """Hundreds of tiles in a row, most of them in work at once: against 64 bits, and the same to the bit every time."""
    rng = np.random.default_rng(13)
    x, gate = make(rng, (1, 20011), 96, heads, "f32", "f32", True, cuda_device)
    y, final = tb.linear_recurrence(x, gate, log_gate=True)
    wy, wf = reference(x, gate, None, None, True)
    m = memory_of(gate, True, 20011)
    close(y, wy, torch.float32, m, what="y")
    close(final, wf, torch.float32, m, float(wy.abs().max()), "final")
    dy = torch.from_numpy(rng.standard_normal((1, 20011, 96))).to(cuda_device, torch.float32)
    grads = tb.linear_recurrence_backward(gate, y, dy, log_gate=True)
    wx, wg, wi, size = reference_backward(gate, y, dy, None, None, None, True)
    close(grads[0], wx, torch.float32, m, what="dx")
    close(grads[1], wg, torch.float32, m, float(wx.abs().max() * wy.abs().max()) * (96 // heads) + float(size.max()), "dgate")
    for _ in range(5):
        again = tb.linear_recurrence(x, gate, log_gate=True)
        g2 = tb.linear_recurrence_backward(gate, y, dy, log_gate=True)
        assert torch.equal(again[0], y) and torch.equal(again[1], final) and all(torch.equal(a, b) for a, b in zip(grads, g2))


@pytest.mark.parametrize("sequences,rows,channels,heads,dtype", [
    (700, 40, 136, 136, "bf16"), (700, 40, 135, 135, "bf16"), (900, 30, 64, 4, "f32"), (3, 900, 64, 64, "bf16")])
def test_scratch_of_a_call_that_gave_up(cuda_device, sequences, rows, channels, heads, dtype):
    """What an earlier call left in the scratch, a time-out in its status among it, means nothing to the next one."""
    rng = np.random.default_rng(17)
    x, gate = make(rng, (sequences, rows), channels, heads, dtype, "f32", True, cuda_device)
    temp = torch.empty(8 << 20, dtype=torch.uint8, device=cuda_device)
    want = tb.linear_recurrence(x, gate, log_gate=True)
    grads = tb.linear_recurrence_backward(gate, want[0], x, log_gate=True)
    for word in (capi.ERR_WAIT_TIMEOUT, capi.ERR_INVALID_ARGUMENT, -1):
        for _ in range(3):
            temp.view(torch.int32).fill_(word)
            got = tb.linear_recurrence(x, gate, log_gate=True, temp=temp)
            temp.view(torch.int32).fill_(word)
            g2 = tb.linear_recurrence_backward(gate, want[0], x, log_gate=True, temp=temp)
            assert all(torch.equal(a, b) for a, b in zip(got + g2, want + grads))


def test_refusals_of_tensors(cuda_device):
    x = torch.zeros(2, 5, 8, device=cuda_device)
    offsets = torch.tensor([0, 5], device=cuda_device)
    bad = [dict(x=x[0]), dict(offsets=offsets), dict(gate=x[:1]), dict(gate=x[..., :3]), dict(x=x.double()),
           dict(gate=x.half()), dict(initial=torch.zeros(2, 4, device=cuda_device)), dict(out=x[:1].expand(2, 5, 8)),
           dict(initial=torch.zeros(2, 8)), dict(x=torch.zeros(2, 8, 5, device=cuda_device).transpose(1, 2)),
           dict(out=torch.zeros(2, 5, 8, device=cuda_device, dtype=torch.half)), dict(gate=x[..., :0])]
    for change in bad:
        with pytest.raises((ValueError, TypeError)):
            tb.linear_recurrence(**{"x": x, "gate": x, **change})
    with pytest.raises(ValueError):
        tb.linear_recurrence_backward(x, x, x[:, :4])
    state = torch.zeros(3, 8, device=cuda_device)
    for change in (dict(state=state.half()), dict(slots=torch.zeros(2, device=cuda_device)), dict(gate=x[0, :1]),
                   dict(slots=torch.zeros(2, dtype=torch.int32)), dict(state=state[:, :4]), dict(state=state[:1].expand(3, 8))):
        with pytest.raises((ValueError, TypeError)):
            tb.linear_recurrence_step(**{"state": state, "x": x[0], "gate": x[0], "slots": torch.zeros(5, dtype=torch.int32, device=cuda_device), **change})
    with pytest.raises(ValueError):
        tb.linear_recurrence_step(state, x[0], x[0])  # more rows than states
