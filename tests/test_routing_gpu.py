"""Tokens per expert and the balance loss against plain evaluations: whole numbers exactly, the loss and its gradient in
64 bits.

Tolerances. A probability is exp of a difference that is rounded (2^-24 of it) and an exponential that is off by
2 + 1.2 |difference| units of 2^-23, divided by a sum of such: with logits within 20 of the largest, below 40 * 2^-23 of
the probability. Sums of non-negative terms keep that and add a rounding a term, at most `rows of a CTA` of them in
32 bits. The gradient p * (w - p.w) adds the cancellation: the same share of p * (|w| + p.|w|). 16-bit outputs add half a
step.
"""
import numpy as np
import pytest
import torch

import thrust_b200 as tb
from thrust_b200 import _capi as capi

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
REL = 40 * 2.0 ** -23


def plain_counts(ids, experts, mask):
    ids = ids.cpu().long()
    if mask is not None:
        ids = ids[mask.cpu().bool()]
    ids = ids.reshape(-1)
    return torch.bincount(ids[(ids >= 0) & (ids < experts)], minlength=experts)


def softmax64(z):
    z = z.double().cpu()
    top = z.amax(1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    s = p.sum(1, keepdim=True)
    return torch.where(s > 0, p / torch.where(s > 0, s, torch.ones_like(s)), p)


def spans_of(rows, offsets):
    return [(0, rows)] if offsets is None else list(zip(offsets[:-1].tolist(), offsets[1:].tolist()))


def plain_loss(z, ids, mask, offsets):
    p, experts = softmax64(z), z.shape[1]
    k = ids.shape[1] if ids.dim() == 2 else 1
    keep = torch.ones(z.shape[0], dtype=torch.bool) if mask is None else mask.cpu().bool()
    loss, counts, weights = [], [], []
    for b, e in spans_of(z.shape[0], offsets):
        m = keep[b:e]
        n = int(m.sum())
        c = plain_counts(ids[b:e], experts, m)
        w = c.double() * experts / (k * n * n) if n else torch.zeros(experts, dtype=torch.float64)
        loss.append((w * p[b:e][m].sum(0)).sum())
        counts.append(c)
        weights.append(w)
    return torch.stack(loss), torch.stack(counts), torch.stack(weights)


@pytest.mark.parametrize("rows,k,experts", [(0, 2, 8), (1, 1, 1), (1, 8, 64), (37, 4, 64), (1000, 1, 3), (4097, 6, 160),
                                            (70001, 8, 256), (3000, 2, 8192), (50000, 3, 5000)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("masked", [False, True])
def test_counts(cuda_device, rows, k, experts, dtype, masked):
    rng = np.random.default_rng(rows + k)
    ids = torch.from_numpy(rng.integers(-1, experts + 1, size=(rows, k))).to(cuda_device, dtype)  # -1 and E: no expert
    mask = torch.from_numpy(rng.random(rows) < 0.7).to(cuda_device) if masked else None
    counts, begins = tb.expert_counts(ids, experts, mask=mask)
    want = plain_counts(ids, experts, mask)
    assert torch.equal(counts.cpu(), want)
    assert torch.equal(begins.cpu(), torch.cat([torch.zeros(1, dtype=torch.int64), want.cumsum(0)]))
    if rows > 2:  # a slice of wider rows, that does not begin at the allocation
        wide = torch.zeros(rows, 2 * k + 3, dtype=dtype, device=cuda_device)
        wide[:, 1:1 + k] = ids
        assert torch.equal(tb.expert_counts(wide[:, 1:1 + k], experts, mask=mask)[0].cpu(), want)
        assert torch.equal(tb.expert_counts(ids[:, 0], experts)[0].cpu(), plain_counts(ids[:, :1], experts, None))


def test_all_tokens_to_one_expert(cuda_device):
    ids = torch.full((300000, 2), 5, dtype=torch.int32, device=cuda_device)
    counts, begins = tb.expert_counts(ids, 7)
    assert counts.tolist() == [0, 0, 0, 0, 0, 600000, 0] and begins.tolist() == [0] * 6 + [600000] * 2
    counts, begins = tb.expert_counts(ids, 7, mask=torch.zeros(300000, dtype=torch.bool, device=cuda_device))
    assert not counts.any() and not begins.any()


LOSS_CASES = [  # rows or lengths, experts, k, type
    (1, 1, 1, "f32"), (1, 8, 2, "bf16"), (2, 5, 1, "f16"), (1024, 8, 2, "f32"), (333, 60, 4, "bf16"),
    (5000, 64, 6, "f16"), (3001, 160, 6, "bf16"), (9000, 256, 8, "bf16"), (700, 384, 8, "f32"), (300, 512, 3, "f16"),
    (130, 1000, 8, "bf16"), (77, 1024, 2, "f32"), ([3, 0, 1, 4000, 0, 59], 64, 4, "bf16"), ([0, 700], 24, 2, "f32"),
    ([1] * 50, 16, 1, "f16"), ([0, 0], 8, 1, "bf16"),
]


def build(case, device, masked, seed=3):
    rows, experts, k, dtype = case
    rng = np.random.default_rng(seed)
    offsets = None
    if isinstance(rows, list):
        offsets = torch.from_numpy(np.cumsum([0, *rows])).to(device, torch.int32 if masked else torch.int64)
        rows = sum(rows)
    z = rng.standard_normal((rows, experts)) * 2 + rng.standard_normal(experts)
    ids = rng.permuted(np.tile(np.arange(experts), (rows, 1)), axis=1)[:, :k] if rows else np.zeros((0, k), dtype=np.int64)
    if rows > 4 and experts > 2:
        z[2, 1:] = -np.inf  # one expert left
        z[3, 0] = -np.inf
    mask = torch.from_numpy(rng.random(rows) < 0.8).to(device) if masked else None
    return (torch.from_numpy(z).to(device, TYPES[dtype]), torch.from_numpy(ids.copy()).to(device), mask, offsets, rng)


@pytest.mark.parametrize("case", LOSS_CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", "")[:40])
@pytest.mark.parametrize("masked", [False, True])
def test_loss_and_gradient(cuda_device, case, masked):
    z, ids, mask, offsets, rng = build(case, cuda_device, masked)
    loss, counts, weights = tb.balance_loss(z, ids, mask=mask, offsets=offsets)
    wl, wc, ww = plain_loss(z, ids, mask, offsets)
    assert torch.equal(counts.cpu(), wc)
    assert ((weights.cpu().double() - ww).abs() <= 2 ** -23 * ww).all()
    per_cta = 64 + z.shape[0] / 100
    assert ((loss.cpu().double() - wl).abs() <= (REL + per_cta * 2 ** -24) * wl).all()
    again = tb.balance_loss(z, ids, mask=mask, offsets=offsets)
    assert torch.equal(loss, again[0]) and torch.equal(weights, again[2])

    sequences = loss.numel()
    scale = 1.0 if z.dtype == torch.float32 else 64.0 * max(1, z.shape[0])  # 16-bit gradients are scaled into range
    dloss = torch.from_numpy((rng.random(sequences) + 0.5).astype(np.float32) * scale).to(cuda_device)
    got = tb.balance_loss_backward(z, weights, dloss, mask=mask, offsets=offsets).cpu().double()
    p, w64, d64 = softmax64(z), weights.cpu().double(), dloss.cpu().double()
    want, size = torch.zeros_like(p), torch.zeros_like(p)
    for i, (b, e) in enumerate(spans_of(z.shape[0], offsets)):
        q, w = p[b:e], w64[i]
        want[b:e] = d64[i] * q * (w - (q @ w)[:, None])
        size[b:e] = d64[i] * q * (w + (q @ w)[:, None])
    if mask is not None:
        want[~mask.cpu()] = 0
        assert not got[~mask.cpu()].any()
    half = 0.0 if z.dtype == torch.float32 else torch.finfo(z.dtype).eps / 2
    tiny = torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps
    top = torch.finfo(z.dtype).max
    inside = want.abs() < top / 2
    assert ((got - want).abs() <= 2 * REL * size + half * want.abs() * (1 + 1e-5) + tiny)[inside].all()


@pytest.mark.parametrize("lengths,experts,k", [
    ([16] * 256, 8, 8), ([1, 0, 2] * 150, 64, 6), ([2000, 2096], 8, 2), ([4096], 8, 2), ([1024], 8, 8), ([1025], 8, 8), ([31] * 33, 32, 1)])
def test_small_calls_on_one_cta_and_on_many(cuda_device, lengths, experts, k):
    """Either side of what one CTA takes alone, as one sequence and as many: the same counts, losses within the bound."""
    z, ids, mask, offsets, _ = build((lengths, experts, k, "bf16"), cuda_device, True)
    loss, counts, weights = tb.balance_loss(z, ids, mask=mask, offsets=offsets)
    wl, wc, ww = plain_loss(z, ids, mask, offsets)
    assert torch.equal(counts.cpu(), wc)
    assert ((weights.cpu().double() - ww).abs() <= 2 ** -23 * ww).all()
    bound = REL + (64 + z.shape[0] / 100) * 2 ** -24
    assert ((loss.cpu().double() - wl).abs() <= bound * wl).all()
    whole, per_expert, _ = tb.balance_loss(z, ids, mask=mask)
    assert torch.equal(per_expert[0], counts.sum(0))
    assert abs(float(whole) - float(plain_loss(z, ids, mask, None)[0])) <= bound * float(whole)


@pytest.mark.parametrize("lengths,experts", [
    ([0] * 700 + [50] + [0] * 300, 64), ([0, 0, 9000, 0] * 3 + [0] * 70, 160), ([0] * 33, 8), ([0] * 31 + [1], 1000), ([3] * 40 + [0] * 4000, 24)])
def test_outputs_of_empty_sequences(cuda_device, lengths, experts):
    """Many of them, in front, between and behind, over one CTA and over many: zeros, in outputs that held something else."""
    z, ids, mask, offsets, _ = build((lengths, experts, 2, "bf16"), cuda_device, False)
    for _ in range(2):  # what these blocks held is what the next outputs begin with
        full = [torch.full((len(lengths), experts), 7, dtype=t, device=cuda_device) for t in (torch.int64, torch.float32)]
        del full
        loss, counts, weights = tb.balance_loss(z, ids, offsets=offsets)
    wl, wc, ww = plain_loss(z, ids, None, offsets)
    assert torch.equal(counts.cpu(), wc)
    assert ((weights.cpu().double() - ww).abs() <= 2 ** -23 * ww).all()
    assert ((loss.cpu().double() - wl).abs() <= (REL + (64 + z.shape[0] / 100) * 2 ** -24) * wl).all()


def test_gradient_agrees_with_differences(cuda_device):
    z, ids, mask, offsets, rng = build(([5, 0, 8], 6, 2, "f32"), cuda_device, True)
    z = torch.where(torch.isinf(z), torch.zeros_like(z), z)
    loss, counts, weights = tb.balance_loss(z, ids, mask=mask, offsets=offsets)
    dloss = torch.tensor([0.5, 3.0, 2.0], device=cuda_device)
    got = tb.balance_loss_backward(z, weights, dloss, mask=mask, offsets=offsets).cpu()
    for r in range(13):
        for e in range(6):
            hi, lo = z.double().cpu(), z.double().cpu()
            hi[r, e] += 1e-5
            lo[r, e] -= 1e-5
            d = sum(float(((plain_loss(a, ids, mask, offsets)[0]) * dloss.cpu().double()).sum()) * s
                    for a, s in ((hi, 1), (lo, -1))) / 2e-5
            assert abs(d - float(got[r, e])) <= 1e-5 * max(1.0, float(got.abs().max()))


def test_masked_rows_are_not_looked_at(cuda_device):
    z, ids, _, _, _ = build((500, 40, 3, "bf16"), cuda_device, False)
    mask = torch.arange(500, device=cuda_device) % 3 != 0
    want = tb.balance_loss(z, ids, mask=mask)
    dloss = torch.ones(1, device=cuda_device)
    grad = tb.balance_loss_backward(z, want[2], dloss, mask=mask)
    z[~mask] = float("nan")
    ids[~mask] = 10 ** 12
    got = tb.balance_loss(z, ids, mask=mask)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(tb.balance_loss_backward(z, got[2], dloss, mask=mask), grad) and not grad[~mask].any()
    work = z.clone()
    assert tb.balance_loss_backward(work, got[2], dloss, mask=mask, out=work) is work and torch.equal(work, grad)
    z[4] = float("nan")  # an unmasked one shows
    loss, counts, _ = tb.balance_loss(z, ids, mask=mask)
    assert torch.isnan(loss).all() and torch.equal(counts, got[1])


def test_disabled_experts_and_rows_without_any(cuda_device):
    z = torch.randn(64, 8, device=cuda_device)
    ids = torch.randint(0, 8, (64, 2), device=cuda_device)
    z[10] = float("-inf")
    z[:, 7] = float("-inf")
    loss, counts, weights = tb.balance_loss(z, ids)
    wl, wc, ww = plain_loss(z, ids, None, None)
    assert torch.equal(counts.cpu(), wc) and abs(float(loss) - float(wl)) <= 1e-5
    grad = tb.balance_loss_backward(z, weights, torch.ones(1, device=cuda_device))
    assert torch.isfinite(grad).all() and not grad[10].any() and not grad[:, 7].any()
    low = z.clone()
    low[torch.isinf(low)] = torch.finfo(torch.float32).min
    l2, _, _ = tb.balance_loss(low, ids)  # masks of the lowest value: the empty row is uniform
    p = softmax64(low)
    assert abs(float(l2) - float((ww[0] * p.sum(0)).sum())) <= 1e-5


def test_strided_logits_and_sequences_without_rows(cuda_device):
    rng = np.random.default_rng(1)
    for experts in (16, 13):
        wide = torch.from_numpy(rng.standard_normal((90, 40))).to(cuda_device, torch.bfloat16)
        z, ids = wide[:, 3:3 + experts], torch.from_numpy(rng.integers(0, experts, size=(90, 2))).to(cuda_device)
        a, b = tb.balance_loss(z, ids), tb.balance_loss(z.contiguous(), ids)
        assert torch.equal(a[1], b[1]) and abs(float(a[0]) - float(b[0])) <= 1e-5
        d = torch.full((1,), 90.0, device=cuda_device)
        out = torch.zeros_like(wide)
        tb.balance_loss_backward(z, a[2], d, out=out[:, 5:5 + experts])
        want = tb.balance_loss_backward(z.contiguous(), a[2], d)
        assert float((out[:, 5:5 + experts].float() - want.float()).abs().max()) <= 2 ** -7 * float(want.float().abs().max())
        assert not out[:, :5].any() and not out[:, 5 + experts:].any()
    offsets = torch.tensor([0, 4, 4], dtype=torch.int32, device=cuda_device)  # rows behind the last sequence
    loss, counts, weights = tb.balance_loss(z, ids, offsets=offsets)
    first = tb.balance_loss(z[:4], ids[:4])
    assert torch.equal(loss[:1], first[0]) and torch.equal(counts[0], first[1][0]) and not counts[1].any() and loss[1] == 0
    grad = tb.balance_loss_backward(z, weights, torch.ones(2, device=cuda_device), offsets=offsets)
    assert grad[:4].any() and not grad[4:].any()
    empty = torch.zeros(0, 8, device=cuda_device)
    loss, counts, weights = tb.balance_loss(empty, torch.zeros(0, 2, dtype=torch.int64, device=cuda_device))
    assert loss.tolist() == [0.0] and not counts.any() and not weights.any()
    assert tb.balance_loss_backward(empty, weights, loss).shape == (0, 8)
    for bad in ([0, 50, 40, 90], [1, 90], [0, 91], [0, -5, 90]):
        with pytest.raises(tb.Tb200Error) as e:
            tb.balance_loss(z, ids, offsets=torch.tensor(bad, dtype=torch.int32, device=cuda_device))
        assert e.value.code == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("experts", [8, 13, 64, 256, 600])
def test_rows_behind_the_last_sequence_are_not_looked_at(cuda_device, dtype, experts):
    """The tail of a padded buffer holds anything: NaN, infinities, whatever. Its gradients are zero, masked or not."""
    rng = np.random.default_rng(experts)
    lengths, tail = [0, 30, 0, 70, 0], 41
    rows = sum(lengths) + tail
    z = torch.from_numpy(rng.standard_normal((rows, experts))).to(cuda_device, TYPES[dtype])
    ids = torch.from_numpy(rng.integers(0, experts, size=(rows, 2))).to(cuda_device)
    offsets = torch.from_numpy(np.cumsum([0, *lengths])).to(cuda_device, torch.int32)
    garbage, garbage_ids = z.clone(), ids.clone()
    end = rows - tail
    garbage[end::4] = float("nan")
    garbage[end + 1::4] = float("inf")
    garbage[end + 2::4, 1] = float("inf")
    garbage[end + 3::4, -1] = float("nan")
    garbage_ids[end:] = -(10 ** 12)
    odd = torch.arange(rows, device=cuda_device) % 3 != 0
    dloss = torch.full((len(lengths),), 1000.0, device=cuda_device)
    for mask in (None, odd):
        want = tb.balance_loss(z, ids, mask=mask, offsets=offsets)
        got = tb.balance_loss(garbage, garbage_ids, mask=mask, offsets=offsets)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        grad = tb.balance_loss_backward(z, want[2], dloss, mask=mask, offsets=offsets)
        out = torch.full_like(z, 3.0)
        tb.balance_loss_backward(garbage, want[2], dloss, mask=mask, offsets=offsets, out=out)
        assert torch.equal(out, grad) and not out[end:].any() and out[:end].any()
        none = tb.balance_loss_backward(garbage, want[2][:0].contiguous(), dloss[:0], mask=mask, offsets=offsets[:1])
        assert none.shape == z.shape and not none.any()  # no sequences at all
    # what belongs to one sequence alone does not reach another: its weights, its dloss, its rows
    dloss[1] = float("inf")
    weights = want[2].clone()
    weights[1, 0] = float("nan")
    garbage[:lengths[1]] = float("nan")
    out = tb.balance_loss_backward(garbage, weights, dloss, mask=odd, offsets=offsets)
    assert torch.equal(out[lengths[1]:], grad[lengths[1]:]) and not out[~odd].any()
    assert torch.isnan(out[:lengths[1]][odd[:lengths[1]]]).all()


def test_captured_and_replayed(cuda_device):
    z, ids, mask, _, _ = build((5000, 128, 4, "bf16"), cuda_device, True)
    dloss = torch.full((1,), 100.0, device=cuda_device)

    def step():
        loss, counts, weights = tb.balance_loss(z, ids, mask=mask, sync=False)
        many, begins = tb.expert_counts(ids, 128, mask=mask, sync=False)
        return loss, counts, weights, many, begins, tb.balance_loss_backward(z, weights, dloss, mask=mask)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        z.mul_(0.9)
        ids.add_(1).remainder_(128)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        assert torch.equal(got[1][0], got[3])


def test_logits_of_more_than_32_bits(cuda_device):
    """More than 2^32 logits, the same 4096 rows over and over: their loss and counts, and the gradient of the last rows."""
    times, experts = (1 << 32) // (4096 * 256) + 3, 256
    z, ids, _, _, _ = build((4096, experts, 2, "bf16"), cuda_device, False)
    wl, wc, _ = plain_loss(z, ids, None, None)
    many, all_ids = z.repeat(times, 1), ids.to(torch.int32).repeat(times, 1)
    loss, counts, weights = tb.balance_loss(many, all_ids)
    assert torch.equal(counts.cpu(), wc * times)
    assert torch.equal(tb.expert_counts(all_ids, experts)[0].cpu(), wc[0] * times)
    # a lane adds a row in eight of a CTA's, of at least 132 SMs with a CTA each, in 32 bits
    assert abs(float(loss) - float(wl[0])) <= (REL + many.shape[0] / 132 / 8 * 2 ** -24) * float(wl[0])
    dloss = torch.full((1,), float(many.shape[0]), device=cuda_device)
    grad = tb.balance_loss_backward(many, weights, dloss)
    want = tb.balance_loss_backward(z, weights, dloss)
    assert want.any() and torch.equal(grad[-4096:], want) and torch.equal(grad[:4096], want)


def test_two_streams_at_once(cuda_device):
    """The same calls under way on two streams: scratch and outputs of their own."""
    z, ids, mask, offsets, _ = build(([4000, 0, 9000, 70, 2000], 160, 6, "bf16"), cuda_device, True)
    dloss = torch.full((5,), 1000.0, device=cuda_device)

    def step():
        loss, counts, weights = tb.balance_loss(z, ids, mask=mask, offsets=offsets, sync=False)
        return (loss, counts, weights, *tb.expert_counts(ids, 160, mask=mask, sync=False),
                tb.balance_loss_backward(z, weights, dloss, mask=mask, offsets=offsets))

    want = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams * 10:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_layer_of_recurrence_and_routing(cuda_device):
    """A training step of one layer on packed sequences: recurrence, router, dispatch order, balance loss, and back."""
    rng = np.random.default_rng(8)
    lengths, channels, experts, k = [40, 0, 90, 1, 61], 64, 8, 2
    rows = sum(lengths)
    offsets = torch.from_numpy(np.cumsum([0, *lengths])).to(cuda_device, torch.int32)
    x = torch.from_numpy(rng.standard_normal((rows, channels)).astype(np.float32)).to(cuda_device)
    gate = torch.from_numpy(-rng.uniform(0.01, 1, size=(rows, 4)).astype(np.float32)).to(cuda_device)
    router = torch.from_numpy(rng.standard_normal((channels, experts)).astype(np.float32) / 8).to(cuda_device)
    y, final = tb.linear_recurrence(x, gate, offsets=offsets, log_gate=True)
    z = y @ router
    ids = z.topk(k, dim=1).indices
    counts, begins = tb.expert_counts(ids, experts)
    # dispatch: (expert, slot) pairs in order of experts, by the library's own stable sort
    keys, slots = ids.reshape(-1).to(torch.int32).clone(), torch.arange(rows * k, dtype=torch.int32, device=cuda_device)
    tb.stable_sort_by_key(keys, slots)
    for e in range(experts):
        b, n = int(begins[e]), int(counts[e])
        assert (keys[b:b + n] == e).all() and torch.equal(slots[b:b + n].long().cpu(), (ids.reshape(-1) == e).nonzero()[:, 0].cpu())
    loss, per_sequence, weights = tb.balance_loss(z, ids, offsets=offsets)
    assert torch.equal(per_sequence.sum(0), counts)
    dloss = torch.full((5,), 1.0, device=cuda_device)
    dz = tb.balance_loss_backward(z, weights, dloss, offsets=offsets)
    dx, dgate, dinitial = tb.linear_recurrence_backward(gate, y, dz @ router.T, offsets=offsets, log_gate=True)

    # the same by autograd in 64 bits, choices held
    x64, g64, r64 = (t.double().cpu().requires_grad_() for t in (x, gate, router))
    a = g64.exp().repeat_interleave(channels // 4, 1)
    out = []
    for b, e in spans_of(rows, offsets.cpu()):
        h = torch.zeros(channels, dtype=torch.float64)
        for t in range(b, e):
            h = a[t] * h + x64[t]
            out.append(h)
    z64 = torch.stack(out) @ r64
    total = torch.zeros((), dtype=torch.float64)
    p = torch.softmax(z64, 1)
    for i, (b, e) in enumerate(spans_of(rows, offsets.cpu())):
        total = total + (weights[i].double().cpu() * p[b:e]).sum()
    total.backward()
    total = total.detach()
    assert abs(float(total) - float(loss.sum())) <= 1e-4 * float(total)
    for got, want in ((dx, x64.grad), (dgate, g64.grad), (y.T @ dz, r64.grad)):
        # single-precision products of 64 channels in front and behind: a few hundred roundings of 2^-24
        assert float((got.double().cpu() - want).abs().max()) <= 1e-4 * float(want.abs().max())


def test_refusals_of_tensors(cuda_device):
    z, ids = torch.zeros(6, 8, device=cuda_device), torch.zeros(6, 2, dtype=torch.int64, device=cuda_device)
    mask = torch.ones(6, dtype=torch.bool, device=cuda_device)
    for call in (lambda: tb.expert_counts(ids.float(), 8), lambda: tb.expert_counts(ids, 8, mask=mask[:5]),
                 lambda: tb.expert_counts(ids, 8, mask=mask.float()), lambda: tb.expert_counts(ids.T, 8), lambda: tb.expert_counts(ids, 8, mask=mask.cpu()),
                 lambda: tb.balance_loss(z, ids[:5]), lambda: tb.balance_loss(z.double(), ids), lambda: tb.balance_loss(z[0], ids),
                 lambda: tb.balance_loss(z, ids, offsets=torch.zeros(2, device=cuda_device)), lambda: tb.balance_loss(z.T, ids),
                 lambda: tb.balance_loss_backward(z, z, torch.zeros(1, device=cuda_device)),
                 lambda: tb.balance_loss_backward(z, z[:1].contiguous(), torch.zeros(2, device=cuda_device)),
                 lambda: tb.balance_loss_backward(z, z[:1].contiguous(), torch.zeros(1, device=cuda_device), out=z[:1].expand(6, 8))):
        with pytest.raises((ValueError, TypeError)):
            call()
    for experts in (0, 8193):
        with pytest.raises(tb.Tb200Error):
            tb.expert_counts(ids, experts)
    with pytest.raises(tb.Tb200Error):
        tb.balance_loss(torch.zeros(6, 1025, device=cuda_device), ids)
