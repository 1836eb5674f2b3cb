"""Cases of the operators of recurrent mixture-of-experts models: the gated linear recurrence (forward, backward, one
token of many requests) and the routing statistics (tokens per expert, balance loss forward and backward).

`run` computes an operator with elementary torch operations, or, where `own` is true, with this framework's calls.

Recurrence, for every sequence and channel: y[t] = a[t] * y[t-1] + x[t], y[-1] the initial state or zero, a the gate or
exp(gate), one gate for each channel or one shared by the channels of a head. Balance loss of a sequence with n
unmasked tokens that choose k of E experts: E / (k n^2) * sum_e count[e] * sum_t softmax(logits[t])[e].
"""
import math

import torch

own = False
DEVICE = "cuda:0"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4, "i64": 8}


def listed():
    return [
        # training or prefill of one long document: a single sequence, a log decay for every channel in 32 bits
        dict(name="recurrence_long", op="recurrence", batch=1, rows=65536, channels=2048, heads=2048, dtype="bf16", gates="f32",
             log=True, packed=False, initial=False),
        # prefill of a few prompts of different lengths behind one another, states carried in and out, a decay per head
        dict(name="recurrence_prompts", op="recurrence", batch=9, rows=4133, channels=1536, heads=24, dtype="bf16", gates="f32",
             log=True, packed=True, initial=True),
        # the backward pass of a training batch, gates of the activations' type
        dict(name="recurrence_backward_batch", op="recurrence_backward", batch=8, rows=4096, channels=2048, heads=2048,
             dtype="bf16", gates="bf16", log=False, packed=False, initial=False),
        # the backward pass over packed documents in full precision, odd sizes, a decay per head
        dict(name="recurrence_backward_packed", op="recurrence_backward", batch=13, rows=10007, channels=1000, heads=25,
             dtype="f32", gates="f32", log=True, packed=True, initial=True),
        # one token of one request
        dict(name="step_one", op="step", rows=1, slots=64, channels=2048, heads=2048, dtype="bf16", gates="f32", log=True),
        # one token of every request of a full server
        dict(name="step_server", op="step", rows=512, slots=2048, channels=4096, heads=64, dtype="bf16", gates="bf16", log=False),
        # where the tokens of a decoding batch go
        dict(name="counts_decode", op="counts", rows=37, experts=64, k=4, ids="i32", masked=True),
        # the expert loads of a large training batch
        dict(name="counts_batch", op="counts", rows=262144, experts=256, k=8, ids="i64", masked=False),
        # balance loss of a small model
        dict(name="balance_small", op="balance", batch=1, rows=1024, experts=8, k=2, dtype="f32", ids="i64", masked=False),
        # balance loss of a training batch, padding masked out
        dict(name="balance_batch", op="balance", batch=1, rows=65536, experts=256, k=8, dtype="bf16", ids="i32", masked=True),
        # its gradient for each of many packed sequences, an odd number of rows
        dict(name="balance_backward_packed", op="balance_backward", batch=23, rows=30011, experts=160, k=6, dtype="bf16",
             ids="i64", masked=True),
        # its gradient over a large batch
        dict(name="balance_backward_batch", op="balance_backward", batch=1, rows=131072, experts=128, k=8, dtype="bf16",
             ids="i64", masked=False),
    ]


def _size(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "recurrence_backward", "recurrence_backward", "step", "counts", "balance",
                     "balance_backward"])
    if op in ("recurrence", "recurrence_backward", "step"):
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        gates = rng.choice([dtype, "f32"])
        if rng.random() < 0.5:  # a gate for every channel
            channels = _size(rng, 16, 8192)
            channels -= channels % 8 if rng.random() < 0.7 and channels > 8 else 0
            heads = channels
        else:
            size = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128, 256])
            heads = _size(rng, 1, 8192 // size)
            channels = size * heads
        log = rng.random() < 0.5
        if op == "step":
            rows = _size(rng, 1, 1024)
            return dict(op=op, rows=rows, slots=_size(rng, rows, 4096), channels=channels, heads=heads, dtype=dtype, gates=gates,
                        log=log)
        packed = rng.random() < 0.5
        # a drawn case stays below the largest listed one: 2^27 elements forward, 2^26 backward
        most = (1 << 26) // channels // (2 if dtype == "f32" else 1) if op == "recurrence" else (1 << 25) // channels
        rows = _size(rng, 1, min(65536, most))
        if packed:
            batch = _size(rng, 1, max(1, min(256, rows)))
        else:
            batch = _size(rng, 1, max(1, min(64, most // rows)))
        return dict(op=op, batch=batch, rows=rows, channels=channels, heads=heads, dtype=dtype, gates=gates, log=log,
                    packed=packed, initial=rng.random() < 0.5)
    experts = rng.choice([8, 16, 32, 60, 64, 128, 160, 256, 384, 512])
    k = rng.choice([1, 2, 4, 6, 8])
    ids = rng.choice(["i32", "i64"])
    if op == "counts":
        return dict(op=op, rows=_size(rng, 1, 262144), experts=experts, k=k, ids=ids, masked=rng.random() < 0.5)
    rows = _size(rng, 1, min(131072, (1 << 24) // experts))
    return dict(op=op, batch=rng.choice([1, 1, _size(rng, 1, min(256, rows))]), rows=rows, experts=experts, k=k,
                dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), ids=ids, masked=rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------
def _cuts(total, parts, g):
    """Begins of `parts` packed sequences of `total` rows: uneven lengths, some of them perhaps empty."""
    cut = torch.randint(0, total + 1, (parts - 1,), device=DEVICE, generator=g).sort().values
    ends = torch.tensor([0, total], device=DEVICE)
    return torch.cat([ends[:1], cut, ends[1:]]).to(torch.int32)


def _gates(shape, case, g):
    """Decays as trained models have them: memories from a few tokens to a thousand, moving with the data."""
    near = torch.exp(torch.empty(shape[-1], device=DEVICE).uniform_(math.log(2e-3), 0.0, generator=g))
    rate = near * torch.sigmoid(torch.randn(shape, device=DEVICE, generator=g))
    return (-rate if case["log"] else torch.exp(-rate)).to(_TYPES[case["gates"]])


def _scores(rows, experts, g):
    """Router logits: some experts preferred by all tokens, the rest of the token."""
    return torch.randn(rows, experts, device=DEVICE, generator=g) * 1.5 + torch.randn(experts, device=DEVICE, generator=g)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] in ("recurrence", "recurrence_backward"):
        rows, d = case["rows"], case["channels"]
        lead = (rows,) if case["packed"] else (case["batch"], rows)
        s["gate"] = _gates((*lead, case["heads"]), case, g)
        s["x"] = torch.randn(*lead, d, device=DEVICE, generator=g).to(_TYPES[case["dtype"]])
        s["offsets"] = _cuts(rows, case["batch"], g) if case["packed"] else None
        s["initial"] = torch.randn(case["batch"], d, device=DEVICE, generator=g) if case["initial"] else None
        if case["op"] == "recurrence_backward":
            s["y"] = _recurrence(s)[0]
            del s["x"]
            s["dy"] = torch.randn(*lead, d, device=DEVICE, generator=g).to(_TYPES[case["dtype"]])
            s["dfinal"] = torch.randn(case["batch"], d, device=DEVICE, generator=g) if case["initial"] else None
    elif case["op"] == "step":
        rows, d = case["rows"], case["channels"]
        s["gate"] = _gates((rows, case["heads"]), case, g)
        s["x"] = torch.randn(rows, d, device=DEVICE, generator=g).to(_TYPES[case["dtype"]])
        s["state"] = torch.randn(case["slots"], d, device=DEVICE, generator=g)
        s["slots"] = torch.randperm(case["slots"], device=DEVICE, generator=g)[:rows].to(torch.int32)
    else:
        scores = _scores(case["rows"], case["experts"], g)
        s["ids"] = scores.topk(case["k"], dim=1).indices.to(torch.int32 if case["ids"] == "i32" else torch.int64)
        s["mask"] = torch.rand(case["rows"], device=DEVICE, generator=g) < 0.9 if case["masked"] else None
        if case["op"] != "counts":
            s["logits"] = scores.to(_TYPES[case["dtype"]])
            s["offsets"] = _cuts(case["rows"], case["batch"], g) if case["batch"] > 1 else None
        if case["op"] == "balance_backward":
            s["weights"] = _balance(s)[2]
            s["dloss"] = torch.rand(case["batch"], device=DEVICE, generator=g) + 0.5
            if case["dtype"] == "f16":  # the loss scale that keeps gradients of this type in range
                s["dloss"] *= max(1.0, case["rows"] / case["batch"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------
def _flat(s, t):
    """The rows of all sequences one behind the other, in 32 bits."""
    return t.reshape(-1, t.shape[-1]).float()


def _ends(s, rows):
    """First and last row of every sequence, and which of them have rows."""
    if s["packed"]:
        first, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    else:
        first = torch.arange(s["batch"], device=DEVICE) * s["rows"]
        end = first + s["rows"]
    return first, end, end > first


def _decays(s, gate):
    """A gate for every channel. exp in 64 bits: a decay next to one acts a thousand times over, and a rounding that
    leans to one side with it."""
    a = torch.exp(gate.double()).float() if s["log"] else gate.float()
    return a.repeat_interleave(s["channels"] // s["heads"], 1)


def _scan(a, b, longest):
    """b[t] + a[t] * (b[t-1] + a[t-1] * ...), by doubling the reach of every row."""
    reach = 1
    while reach < longest:
        b[reach:] = b[reach:] + a[reach:] * b[:-reach]
        a[reach:] = a[reach:] * a[:-reach]
        reach *= 2
    return b


def _recurrence(s):
    a, x = _decays(s, _flat(s, s["gate"])), _flat(s, s["x"])
    first, end, some = _ends(s, x.shape[0])
    at = first[some]
    h = torch.zeros(s["batch"], s["channels"], device=DEVICE) if s["initial"] is None else s["initial"].float()
    x, a = x.clone(), a.clone()
    x[at] = x[at] + a[at] * h[some]
    a[at] = 0
    y = _scan(a, x, s["rows"])
    last = y[(end - 1).clamp(min=0)]
    final = torch.where(some[:, None], last, h)
    return y.to(s["x"].dtype).view(s["x"].shape), final


def _recurrence_backward(s):
    a, y, dy = _decays(s, _flat(s, s["gate"])), _flat(s, s["y"]), _flat(s, s["dy"])
    first, end, some = _ends(s, y.shape[0])
    at, last = first[some], end[some] - 1
    zeros = torch.zeros(s["batch"], s["channels"], device=DEVICE)
    h = zeros if s["initial"] is None else s["initial"].float()
    p = zeros if s["dfinal"] is None else s["dfinal"].float()
    g = dy.clone()
    g[last] = g[last] + p[some]
    after = torch.cat([a[1:], a[:1]])  # the gate of the row behind
    after[last] = 0
    g = _scan(after.flip(0), g.flip(0), s["rows"]).flip(0)
    before = torch.cat([y[:1], y[:-1]])
    before[at] = h[some]
    da = g * before
    if s["log"]:
        da = da * a
    da = da.view(-1, s["heads"], s["channels"] // s["heads"]).sum(2)
    dh = p.clone()
    dh[some] = a[at] * g[at]
    return g.to(s["dy"].dtype).view(s["dy"].shape), da.to(s["gate"].dtype).view(s["gate"].shape), dh


def _step(s):
    a = _decays(s, s["gate"])
    at = s["slots"].long()
    h = a * s["state"][at] + s["x"].float()
    s["state"][at] = h
    return h.to(s["x"].dtype), s["state"]


def _counts(s, which, batch):
    """How often every expert is chosen in every sequence; `which` names each row's sequence."""
    e = s["experts"]
    keys = which[:, None] * e + s["ids"].long()
    if s["mask"] is not None:
        keys = keys[s["mask"]]
    keys = keys.reshape(-1)
    counts = torch.zeros(batch * e, dtype=torch.int64, device=DEVICE)
    return counts.index_add_(0, keys, torch.ones_like(keys)).view(batch, e)


def _which(s):
    """The sequence of every row."""
    rows = torch.arange(s["rows"], device=DEVICE)
    if s.get("offsets") is None:
        return torch.zeros_like(rows)
    return (rows[:, None] >= s["offsets"][None, 1:]).sum(1)


def _softmax(z):
    z = z.float()
    p = torch.exp(z - z.amax(1, keepdim=True))
    return p / p.sum(1, keepdim=True)


def _balance(s):
    which, batch = _which(s), s["batch"]
    counts = _counts(s, which, batch)
    p = _softmax(s["logits"])
    kept = torch.ones(s["rows"], device=DEVICE) if s["mask"] is None else s["mask"].float()
    sums = torch.zeros(batch, s["experts"], dtype=torch.float64, device=DEVICE).index_add_(0, which, (p * kept[:, None]).double())
    n = torch.zeros(batch, dtype=torch.float64, device=DEVICE).index_add_(0, which, kept.double())
    w = torch.where(n[:, None] > 0, counts.double() * (s["experts"] / s["k"]) / (n * n).clamp(min=1)[:, None], 0.0)
    return (w * sums).sum(1).float(), counts, w.float()


def _balance_backward(s):
    which = _which(s)
    p = _softmax(s["logits"])
    w = s["weights"][which]
    d = p * (w - (p * w).sum(1, keepdim=True)) * s["dloss"][which][:, None]
    if s["mask"] is not None:
        d = torch.where(s["mask"][:, None], d, 0.0)
    return d.to(s["logits"].dtype)


def _expert_counts(s):
    counts = _counts(s, _which(s), 1)[0]
    return counts, torch.cat([torch.zeros_like(counts[:1]), torch.cumsum(counts, 0)])


def run(s):
    op = s["op"]
    if own:
        import thrust_b200 as tb
        if op == "recurrence":
            return tb.linear_recurrence(s["x"], s["gate"], initial=s["initial"], offsets=s["offsets"], log_gate=s["log"],
                                        sync=False)
        if op == "recurrence_backward":
            return tb.linear_recurrence_backward(s["gate"], s["y"], s["dy"], initial=s["initial"], dfinal=s["dfinal"],
                                                 offsets=s["offsets"], log_gate=s["log"], sync=False)
        if op == "step":
            return tb.linear_recurrence_step(s["state"], s["x"], s["gate"], slots=s["slots"], log_gate=s["log"]), s["state"]
        if op == "counts":
            return tb.expert_counts(s["ids"], s["experts"], mask=s["mask"], sync=False)
        if op == "balance":
            return tb.balance_loss(s["logits"], s["ids"], mask=s["mask"], offsets=s["offsets"], sync=False)
        return tb.balance_loss_backward(s["logits"], s["weights"], s["dloss"], mask=s["mask"], offsets=s["offsets"])
    if op == "recurrence":
        return _recurrence(s)
    if op == "recurrence_backward":
        return _recurrence_backward(s)
    if op == "step":
        return _step(s)
    if op == "counts":
        return _expert_counts(s)
    if op == "balance":
        return _balance(s)
    return _balance_backward(s)


# ---- the work of a pass -------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op in ("recurrence", "recurrence_backward", "step"):
        rows = case["rows"] * (case["batch"] if not case.get("packed") and op != "step" else 1)
        many, gates = rows * case["channels"], rows * case["heads"] * _BYTES[case["gates"]]
        if op == "step":
            return {"bytes": many * (8 + 2 * _BYTES[case["dtype"]]) + gates + 4 * rows, "flops": 2 * many}
        states = 4 * case["batch"] * case["channels"]
        if op == "recurrence":
            return {"bytes": many * 2 * _BYTES[case["dtype"]] + gates + states * (2 if case["initial"] else 1),
                    "flops": 2 * many}
        return {"bytes": many * 3 * _BYTES[case["dtype"]] + 2 * gates + states * (3 if case["initial"] else 1),
                "flops": 4 * many}
    rows, e = case["rows"], case["experts"]
    ids = rows * case["k"] * _BYTES[case["ids"]] + (rows if case["masked"] else 0)
    if op == "counts":
        return {"bytes": ids + 16 * e, "flops": rows * case["k"]}
    logits = rows * e * _BYTES[case["dtype"]]
    if op == "balance":
        return {"bytes": logits + ids + 12 * e * case["batch"], "flops": 5 * rows * e}
    return {"bytes": 2 * logits + 4 * e * case["batch"], "flops": 8 * rows * e}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def _spans(s, rows):
    """(sequence, first row, end) of every sequence, on the host."""
    if s.get("offsets") is not None:
        cut = s["offsets"].tolist()
    else:
        cut = [i * rows // s["batch"] for i in range(s["batch"] + 1)]
    return [(i, cut[i], cut[i + 1]) for i in range(s["batch"])]


def _exact_gates(s, lead):
    a = s["gate"].double()
    a = a.exp() if s["log"] else a
    return a[..., None].expand(*a.shape, s["channels"] // s["heads"]).reshape(*lead, s["channels"])


def _exact_recurrence(s):
    """Row by row, all sequences of a batch at once; packed ones one after the other."""
    x = s["x"].double()
    a = _exact_gates(s, x.shape[:-1])
    h = torch.zeros(s["batch"], s["channels"], dtype=torch.float64, device=DEVICE)
    if s["initial"] is not None:
        h += s["initial"].double()
    y = torch.empty_like(x)
    if not s["packed"]:
        for t in range(s["rows"]):
            h = torch.addcmul(x[:, t], a[:, t], h)
            y[:, t] = h
        return y, h
    for i, begin, end in _spans(s, x.shape[0]):
        state = h[i]
        for t in range(begin, end):
            state = torch.addcmul(x[t], a[t], state)
            y[t] = state
        h[i] = state
    return y, h


def _exact_recurrence_backward(s):
    y, dy = s["y"].double(), s["dy"].double()
    a = _exact_gates(s, y.shape[:-1])
    carry = torch.zeros(s["batch"], s["channels"], dtype=torch.float64, device=DEVICE)
    start = carry.clone() if s["initial"] is None else s["initial"].double()
    if s["dfinal"] is not None:
        carry += s["dfinal"].double()
    dx, da = torch.empty_like(y), torch.empty_like(y)
    if not s["packed"]:
        for t in reversed(range(s["rows"])):
            g = dy[:, t] + carry
            dx[:, t] = g
            da[:, t] = g * (y[:, t - 1] if t else start)
            carry = a[:, t] * g
    else:
        for i, begin, end in _spans(s, y.shape[0]):
            p = carry[i]
            for t in reversed(range(begin, end)):
                g = dy[t] + p
                dx[t] = g
                da[t] = g * (y[t - 1] if t > begin else start[i])
                p = a[t] * g
            carry[i] = p
    if s["log"]:
        da *= a
    return dx, da.unflatten(-1, (s["heads"], -1)).sum(-1), carry


def _exact_step(s):
    a = _exact_gates(s, s["x"].shape[:-1])
    state = s["state"].double()
    at = s["slots"].long()
    y = torch.addcmul(s["x"].double(), a, state[at])
    state[at] = y
    return y, state


def _exact_balance(s):
    p = torch.softmax(s["logits"].double(), 1)
    loss, weights = [], []
    for i, begin, end in _spans(s, s["rows"]):
        keep = torch.ones(end - begin, dtype=torch.bool, device=DEVICE) if s["mask"] is None else s["mask"][begin:end]
        n = int(keep.sum())
        c = torch.bincount(s["ids"][begin:end][keep].reshape(-1), minlength=s["experts"]).double()
        w = c * s["experts"] / (s["k"] * n * n) if n else c
        weights.append(w)
        loss.append((w * p[begin:end][keep].sum(0)).sum())
    return torch.stack(loss), None, torch.stack(weights)


def _exact_balance_backward(s):
    p = torch.softmax(s["logits"].double(), 1)
    d = torch.zeros_like(p)
    for i, begin, end in _spans(s, s["rows"]):
        q, w = p[begin:end], s["weights"][i].double()
        d[begin:end] = s["dloss"][i].double() * q * (w - (q @ w)[:, None])
    if s["mask"] is not None:
        d[~s["mask"]] = 0
    return d


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "recurrence":
        return _exact_recurrence(s)
    if op == "recurrence_backward":
        return _exact_recurrence_backward(s)
    if op == "step":
        return _exact_step(s)
    if op == "counts":
        return None
    if op == "balance":
        return _exact_balance(s)
    return _exact_balance_backward(s)
