"""The cases on which the row lookup and the gated recurrence of ``lightgbm_amd.ops`` are timed, with their plain forms.

A tree ensemble answers with a lookup (the value of the leaf a row falls into, tree by tree) followed by a linear
recurrence over the trees (a running sum for boosting, a running mean for a random forest), and its leaf values are
fitted with the gradients of both.  The same two operators carry the embedding and the recurrent layers of sequence
models, whose shapes are among the cases.

``own`` selects what :func:`run` calls: the framework's operators, or elementary torch operations.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}


def _lookup(name, tokens, rows, width, dtype, scale=1.0, pad=0.0):
    return {"name": name, "op": "embedding", "samples": tokens, "trees": 0, "rows": rows, "width": width, "dtype": dtype,
            "scale": scale, "pad": pad}


def _leaves(name, op, samples, trees, leaves, width, dtype, scale=1.0):
    return {"name": name, "op": op, "samples": samples, "trees": trees, "rows": trees * leaves, "width": width,
            "dtype": dtype, "scale": scale, "pad": 0.0}


def _scan(name, op, batch, steps, width, dtype, gate, groups, gate_batch=None, mix=False, ragged=False):
    return {"name": name, "op": op, "batch": batch, "steps": steps, "width": width, "dtype": dtype, "gate": gate,
            "groups": groups, "gate_batch": batch if gate_batch is None else gate_batch, "mix": mix, "ragged": ragged}


def listed():
    return [
        # one decoding step of a small batch: 16 tokens looked up, where the launch is all there is
        _lookup("lookup-step", 16, 32000, 2048, "bf16", scale=math.sqrt(2048.0)),
        # a training batch's tokens, with the usual scaling by the square root of the width and some padding
        _lookup("lookup-train", 32768, 65536, 4096, "bf16", scale=64.0, pad=0.02),
        # staged prediction: the leaf values of 45.8 k rows (the reference's training split) in 300 trees of 127 leaves,
        # leaf ids as pred_leaf gives them ([rows, trees]) and taken tree by tree
        _leaves("lookup-leaves", "embedding", 45800, 300, 127, 1, "f64"),
        # gradient of a short batch: most of the table gets zeros
        _lookup("lookup-grad-short", 256, 8192, 512, "f32") | {"op": "embedding_grad"},
        # gradient of a training batch of words (a few frequent ones, many rare, some padding)
        _lookup("lookup-grad-words", 65537, 50000, 1024, "bf16", scale=32.0, pad=0.02) | {"op": "embedding_grad"},
        # gradient of the leaf values of a whole ensemble: 45.8 k rows x 300 trees of 31 leaves
        _leaves("lookup-grad-leaves", "embedding_grad", 45800, 300, 31, 1, "f32", scale=0.1),
        # one step of 64 sequences that are being served
        _scan("scan-step", "gated_scan", 64, 1, 4096, "bf16", "f32", 4096),
        # one long sequence
        _scan("scan-long", "gated_scan", 1, 65537, 1024, "bf16", "bf16", 1024),
        # a training batch, gates kept in 32 bits
        _scan("scan-train", "gated_scan", 8, 4096, 2560, "bf16", "f32", 2560, mix=True),
        # staged scores of a random forest: the running mean over 500 trees for 45.8 k rows, one gate per tree
        _scan("scan-stages", "gated_scan", 1, 500, 45800, "f64", "f64", 1, gate_batch=1, mix=True),
        # the training batch backwards
        _scan("scan-grad-train", "gated_scan_grad", 8, 4096, 2560, "bf16", "f32", 2560, mix=True),
        # sequences of unequal lengths and odd width, a gate per head of 103 channels
        _scan("scan-grad-heads", "gated_scan_grad", 5, 2047, 515, "f32", "f32", 5, ragged=True),
    ]


def _between(rng, lo, hi):
    """A whole number, spread over the logarithm of the range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "embedding_grad", "gated_scan", "gated_scan_grad"])
    if op in ("embedding", "embedding_grad"):
        if rng.random() < 0.4:
            trees, leaves = _between(rng, 10, 500), _between(rng, 7, 255)
            width = rng.choice([1, 1, 1, 3, 7])
            samples = _between(rng, 100, max(101, 13000000 // (trees * width)))
            return {k: v for k, v in _leaves("", op, samples, trees, leaves, width, rng.choice(["f32", "f64"]),
                                             rng.choice([1.0, 0.1, 0.05])).items() if k != "name"}
        width = _between(rng, 32, 4096)
        tokens = _between(rng, 1, min(65536, 60000000 // width))
        rows = _between(rng, 1000, min(65536, 60000000 // width))
        case = _lookup("", tokens, rows, width, rng.choice(["bf16", "bf16", "f16", "f32"]),
                       rng.choice([1.0, math.sqrt(width)]), rng.choice([0.0, 0.02, 0.3]))
        return {k: v for k, v in case.items() if k != "name"} | {"op": op}
    most = 60000000 if op == "gated_scan" else 40000000
    if rng.random() < 0.25:
        steps = _between(rng, 10, 1000)
        width = _between(rng, 100, most // 3 // steps)
        case = _scan("", op, 1, steps, width, rng.choice(["f32", "f64"]), None, 1, 1, mix=rng.random() < 0.5)
        case["gate"] = case["dtype"] if case["mix"] else "none"
    else:
        groups, per = rng.choice([(1, 64), (1, 0), (1, 0), (1, 0), (5, 103), (8, 64), (16, 96), (32, 128)])
        width = groups * per if per else _between(rng, 16, 4096)
        groups = groups if per else width
        batch = _between(rng, 1, 64)
        steps = _between(rng, 1, max(2, min(65536, most // (batch * width))))
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        case = _scan("", op, batch, steps, width, dtype, rng.choice([dtype, "f32"]), groups,
                     rng.choice([batch, batch, batch, 1]), mix=rng.random() < 0.4, ragged=rng.random() < 0.3)
    return {k: v for k, v in case.items() if k != "name"}


def _normal(g, shape, dtype):
    wide = torch.float64 if dtype is torch.float64 else torch.float32
    return torch.randn(shape, generator=g, device="cuda", dtype=wide).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dtype = _TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] in ("embedding", "embedding_grad"):
        rows, samples, trees = case["rows"], case["samples"], case["trees"]
        if trees:
            # leaves are not equally full: the square of a uniform number prefers a tree's first ones
            leaves = rows // trees
            u = torch.rand((samples, trees), generator=g, device="cuda")
            ids = (u * u * leaves).to(torch.int32).clamp_(max=leaves - 1)
            ids = (ids + torch.arange(trees, device="cuda", dtype=torch.int32) * leaves).t()
        else:
            # word frequencies: uniform in the logarithm of the rank, ranks scattered over the table
            u = torch.rand((samples,), generator=g, device="cuda")
            rank = torch.exp(u * math.log(float(rows))).to(torch.int64).clamp_(1, rows) - 1
            ids = torch.randperm(rows, generator=g, device="cuda")[rank]
            ids[torch.rand((samples,), generator=g, device="cuda") < case["pad"]] = -1
        state["ids"] = ids
        if case["op"] == "embedding":
            state["table"] = _normal(g, (rows, case["width"]), dtype)
        else:
            state["grad"] = _normal(g, tuple(ids.shape) + (case["width"],), dtype)
        return state
    b, t, d = case["batch"], case["steps"], case["width"]
    wide = torch.float64 if dtype is torch.float64 else torch.float32
    state["x"] = _normal(g, (b, t, d), dtype)
    state["state"] = _normal(g, (b, d), wide)
    state["lengths"] = None
    if case["ragged"]:
        state["lengths"] = torch.randint(0, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        state["lengths"][b - 1] = t
    if case["gate"] == "none":
        state["gate"] = None
    else:
        gate = _TYPES[case["gate"]]
        if case["groups"] == 1 and case["gate_batch"] == 1 and b == 1:
            n = torch.arange(1, t + 1, device="cuda", dtype=torch.float64)      # the running mean over the trees
            state["gate"] = ((n - 1) / n).reshape(1, t, 1).to(gate)
        else:
            # most gates near one, some sequences within the sequence start anew (a gate of zero)
            a = torch.sigmoid(_normal(g, (case["gate_batch"], t, case["groups"]), torch.float32) + 2.0)
            anew = torch.rand((case["gate_batch"], t, 1), generator=g, device="cuda") < 1e-3
            state["gate"] = torch.where(anew, torch.zeros_like(a), a).to(gate)
    if case["op"] == "gated_scan_grad":
        a, x = _wide_gate(state, wide), state["x"].to(wide)
        a, w = _inside(state, a, x)
        state["states"] = torch.where(_valid(state), _recurrence(a, w, state["state"]), torch.zeros_like(w)).to(dtype)
        state["grad_states"] = _normal(g, (b, t, d), dtype)
        state["grad_last"] = _normal(g, (b, d), wide)
        if not case["mix"]:
            state["x"] = None       # the gradients need x for the mixed form alone
    return state


# -- plain forms ------------------------------------------------------------------------------------------------------

def _wide_gate(state, wide):
    """The gate of every value: [B, T, D]."""
    case = state["case"]
    shape = (case["batch"], case["steps"], case["width"])
    if state["gate"] is None:
        return torch.ones(shape, device="cuda", dtype=wide)
    a = state["gate"].to(wide)
    return a.repeat_interleave(case["width"] // case["groups"], dim=2).expand(shape)


def _valid(state):
    case = state["case"]
    at = torch.arange(case["steps"], device="cuda").reshape(1, -1, 1)
    if state["lengths"] is None:
        return at < case["steps"]
    return at < state["lengths"].reshape(-1, 1, 1)


def _inside(state, a, x):
    """Gates and inputs of the recurrence; behind a sequence's end the state is kept."""
    w = (1 - a) * x if state["case"]["mix"] else x
    if state["lengths"] is None:
        return a, w
    valid = _valid(state)
    return torch.where(valid, a, torch.ones_like(a)), torch.where(valid, w, torch.zeros_like(w))


def _recurrence(a, w, first):
    """h[t] = a[t] h[t-1] + w[t] along dim 1, in log2(T) passes: after the pass with distance s every position holds the
    composition of its 2 s last steps."""
    h = w.clone()
    h[:, 0] += a[:, 0] * first
    s = 1
    while s < h.shape[1]:
        head, tail = h[:, :s], h[:, s:] + a[:, s:] * h[:, :-s]
        h = torch.cat([head, tail], dim=1)
        a = torch.cat([a[:, :s], a[:, s:] * a[:, :-s]], dim=1)
        s *= 2
    return h


def _plain(state):
    case = state["case"]
    dtype = _TYPES[case["dtype"]]
    wide = torch.float64 if dtype is torch.float64 else torch.float32
    if case["op"] == "embedding":
        ids = state["ids"].long()
        valid = (ids >= 0) & (ids < case["rows"])
        got = state["table"][torch.where(valid, ids, torch.zeros_like(ids))].to(wide) * case["scale"]
        return torch.where(valid.unsqueeze(-1), got, torch.zeros_like(got)).to(dtype)
    if case["op"] == "embedding_grad":
        ids = state["ids"].reshape(-1).long()
        grad = state["grad"].reshape(-1, case["width"])
        valid = (ids >= 0) & (ids < case["rows"])
        sums = torch.zeros((case["rows"] + 1, case["width"]), device="cuda", dtype=wide)
        sums.index_add_(0, torch.where(valid, ids, torch.full_like(ids, case["rows"])), grad.to(wide))
        return (sums[:-1] * case["scale"]).to(dtype)
    a = _wide_gate(state, wide)
    x = None if state["x"] is None else state["x"].to(wide)
    if case["op"] == "gated_scan":
        a, w = _inside(state, a, x)
        h = _recurrence(a, w, state["state"])
        last = h[:, -1].clone()
        return torch.where(_valid(state), h, torch.zeros_like(h)).to(dtype), last
    valid = _valid(state)
    zero = torch.zeros((), device="cuda", dtype=wide)
    grad = torch.where(valid, state["grad_states"].to(wide), zero)
    keep = torch.where(valid, a, torch.ones_like(a))
    # backwards: c[t] = grad[t] + a[t+1] c[t+1], started by the last state's gradient
    gates = torch.cat([keep[:, 1:], torch.ones_like(keep[:, :1])], dim=1)
    c = _recurrence(gates.flip(1), grad.flip(1), state["grad_last"]).flip(1)
    grad_state = keep[:, 0] * c[:, 0]
    grad_x = torch.where(valid, (1 - a) * c if case["mix"] else c, zero).to(dtype)
    if state["gate"] is None:
        return grad_x, grad_state
    before = torch.cat([state["state"].unsqueeze(1), state["states"][:, :-1].to(wide)], dim=1)
    grad_gate = torch.where(valid, c * (before - x if case["mix"] else before), zero)
    b, t, d = grad_gate.shape
    grad_gate = grad_gate.reshape(b, t, case["groups"], d // case["groups"]).sum(3)
    if case["gate_batch"] < b:
        grad_gate = grad_gate.sum(0, keepdim=True)
    return grad_x, grad_state, grad_gate.to(state["gate"].dtype)


def run(state):
    if not own:
        return _plain(state)
    from lightgbm_amd import ops
    case = state["case"]
    if case["op"] == "embedding":
        return ops.embedding(state["table"], state["ids"], scale=case["scale"])
    if case["op"] == "embedding_grad":
        return ops.embedding_grad(state["grad"], state["ids"], case["rows"], scale=case["scale"])
    if case["op"] == "gated_scan":
        return ops.gated_scan(state["x"], state["gate"], state["state"], mix=case["mix"], lengths=state["lengths"])
    got = ops.gated_scan_grad(state["grad_states"], state["states"], state["gate"], state["state"], x=state["x"],
                              grad_last=state["grad_last"], mix=case["mix"], lengths=state["lengths"])
    return got if state["gate"] is not None else got[:2]


# -- 64-bit values from the definitions -------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "embedding":
        padded = torch.cat([state["table"].to(f64), torch.zeros((1, case["width"]), device="cuda", dtype=f64)])
        return torch.index_select(padded, 0, state["ids"].reshape(-1).long() % (case["rows"] + 1)).mul_(case["scale"]).reshape(
            tuple(state["ids"].shape) + (case["width"],))
    if case["op"] == "embedding_grad":
        # every row of the table is the difference of two partial sums of the gradients in the order of their ids
        ids, order = torch.sort(state["ids"].reshape(-1).long(), stable=True)
        bounds = torch.searchsorted(ids, torch.arange(case["rows"] + 1, device="cuda"))
        got = torch.empty((case["rows"], case["width"]), device="cuda", dtype=f64)
        flat = state["grad"].reshape(-1, case["width"])
        for at in range(0, case["width"], 128):
            part = flat[:, at:at + 128][order].to(f64).cumsum(0)
            part = torch.cat([torch.zeros_like(part[:1]), part])
            got[:, at:at + 128] = (part[bounds[1:]] - part[bounds[:-1]]) * case["scale"]
        return got
    b, t, d = case["batch"], case["steps"], case["width"]
    lengths = [t] * b if state["lengths"] is None else state["lengths"].tolist()
    per = d // case["groups"]

    def gates(at):
        """The gates of one step, [B, D], and where they apply, [B, 1]."""
        live = torch.tensor([at < n for n in lengths], device="cuda").reshape(b, 1) if state["lengths"] is not None else None
        if state["gate"] is None:
            return torch.ones((b, d), device="cuda", dtype=f64), live
        a = state["gate"][:, at].to(f64).unsqueeze(2).expand(-1, -1, per).reshape(-1, d).expand(b, d)
        return a, live

    def only(live, new, old):
        return new if live is None else torch.where(live, new, old)

    if case["op"] == "gated_scan":
        h = state["state"].to(f64)
        states = torch.zeros((b, t, d), device="cuda", dtype=f64)
        for at in range(t):
            a, live = gates(at)
            x = state["x"][:, at].to(f64)
            h = only(live, torch.addcmul((1 - a) * x if case["mix"] else x, a, h), h)
            states[:, at] = only(live, h, torch.zeros_like(h))
        return states, h
    c = state["grad_last"].to(f64)          # the gradient of the state behind the step
    grad_x = torch.zeros((b, t, d), device="cuda", dtype=f64)
    grad_gate = torch.zeros((b, t, case["groups"]), device="cuda", dtype=f64)
    for at in reversed(range(t)):
        a, live = gates(at)
        whole = c + state["grad_states"][:, at].to(f64)
        before = state["states"][:, at - 1].to(f64) if at else state["state"].to(f64)
        value = (1 - a) * whole if case["mix"] else whole
        slope = whole * (before - state["x"][:, at].to(f64)) if case["mix"] else whole * before
        nothing = torch.zeros_like(whole)
        grad_x[:, at] = only(live, value, nothing)
        grad_gate[:, at] = only(live, slope, nothing).reshape(b, case["groups"], per).sum(2)
        c = only(live, a * whole, c)
    if state["gate"] is None:
        return grad_x, c
    return grad_x, c, grad_gate.sum(0, keepdim=True) if case["gate_batch"] < b else grad_gate


# -- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    e = {"bf16": 2, "f16": 2, "f32": 4, "f64": 8, "none": 0}
    size, wide = e[case["dtype"]], 8 if case["dtype"] == "f64" else 4
    if case["op"] in ("embedding", "embedding_grad"):
        tokens = case["samples"] * max(1, case["trees"])
        ids = tokens * (4 if case["trees"] else 8)
        table = (min(tokens, case["rows"]) if case["op"] == "embedding" else case["rows"]) * case["width"] * size
        return {"bytes": ids + tokens * case["width"] * size + table, "flops": tokens * case["width"]}
    values = case["batch"] * case["steps"] * case["width"]
    gates = case["gate_batch"] * case["steps"] * case["groups"] * e[case["gate"]]
    ends = 2 * case["batch"] * case["width"] * wide
    if case["op"] == "gated_scan":
        return {"bytes": 2 * values * size + gates + ends, "flops": (4 if case["mix"] else 2) * values}
    return {"bytes": (4 if case["mix"] else 3) * values * size + 2 * gates + 1.5 * ends, "flops": (6 if case["mix"] else 4) * values}
