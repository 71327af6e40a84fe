"""Row lookup and gated recurrence (lightgbm_amd.ops): the formulas in 64 bits, the refusals, and their use together.

Tolerances count roundings.  u(T) = eps(T) / 2 is the relative error of one rounding to T; sums and states are held in
W (fp32, for fp64 fp64).  A sum of n terms, in any order, is off by at most (n - 1) u(W) times the sum of their absolute
values.  In the recurrence a term passes at most two roundings a step (one in the product of the gates, one in the sum,
whichever way the steps are grouped) and a handful at the ends, so a state is off by at most (2 t + 10) u(W) times the
same recurrence over absolute values.  1.01 covers the products of these errors, `_TINY` what underflows.
"""
import itertools

import numpy as np
import pytest
import torch

from lightgbm_amd import LightGBMError, ops

gpu = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}
_TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0**-25, torch.float32: 1e-38, torch.float64: 1e-300}


def u(dtype):
    return torch.finfo(dtype).eps / 2


def wide(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def rng(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, shape, dtype):
    return torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)


def within(got, want, bound, dtype):
    """|got - want| <= bound + the rounding to dtype, element by element."""
    got = got.detach().double().cpu()
    allowed = 1.01 * (bound + u(dtype) * want.abs()) + _TINY[dtype]
    off = (got - want).abs()
    assert got.shape == want.shape
    bad = ~(off <= allowed)
    assert not bad.any(), (int(bad.sum()), off[bad].max().item(), allowed[bad].min().item(), torch.nonzero(bad)[0].tolist())


# -- oracles, on the CPU in 64 bits -----------------------------------------------------------------------------------

def lookup_oracle(table, ids, scale):
    t = torch.cat([table.double().cpu(), torch.zeros((1, table.shape[1]), dtype=torch.float64)])
    i = ids.long().cpu()
    i = torch.where((i >= 0) & (i < table.shape[0]), i, torch.full_like(i, table.shape[0]))
    return t[i] * scale


def lookup_grad_oracle(grad, ids, rows, scale):
    """(sums, sums of absolute values, tokens of every row)."""
    i = ids.long().cpu().reshape(-1)
    g = grad.double().cpu().reshape(i.numel(), grad.shape[-1])
    ok = (i >= 0) & (i < rows)
    out, mag = torch.zeros((rows, g.shape[1]), dtype=torch.float64), torch.zeros((rows, g.shape[1]), dtype=torch.float64)
    out.index_add_(0, i[ok], g[ok])
    mag.index_add_(0, i[ok], g[ok].abs())
    n = torch.zeros(rows, dtype=torch.float64).index_add_(0, i[ok], torch.ones(int(ok.sum()), dtype=torch.float64))
    return out * scale, mag * abs(scale), n


def _gates(gate, b, t, d):
    if gate is None:
        return torch.ones((b, t, d), dtype=torch.float64)
    a = gate.double().cpu()
    return a.repeat_interleave(d // a.shape[2], dim=2).expand(b, t, d)


def scan_oracle(x, gate, state, mix, lengths):
    """(states, last, bound of the states, bound of the last)."""
    b, t, d = x.shape
    a, xs = _gates(gate, b, t, d), x.double().cpu()
    n = torch.full((b,), t) if lengths is None else lengths.cpu().long().clamp(0, t)
    h = torch.zeros((b, d), dtype=torch.float64) if state is None else state.double().cpu()
    s = h.abs()
    states, mags = torch.zeros((b, t, d), dtype=torch.float64), torch.zeros((b, t, d), dtype=torch.float64)
    for k in range(t):
        live = (k < n).reshape(b, 1)
        w = (1 - a[:, k]) * xs[:, k] if mix else xs[:, k]
        h = torch.where(live, a[:, k] * h + w, h)
        s = torch.where(live, a[:, k].abs() * s + w.abs(), s)
        states[:, k] = torch.where(live, h, torch.zeros_like(h))
        mags[:, k] = torch.where(live, s, torch.zeros_like(s))
    e = u(wide(x.dtype))
    steps = torch.arange(t, dtype=torch.float64).reshape(1, t, 1)
    return states, h, (2 * steps + 12) * e * mags, (2 * t + 12) * e * s


def scan_grad_oracle(dh, states, gate, state, x, dlast, mix, lengths):
    """(grad_x, grad_state, grad_gate) and their bounds."""
    b, t, d = states.shape
    a = _gates(gate, b, t, d)
    n = torch.full((b,), t) if lengths is None else lengths.cpu().long().clamp(0, t)
    zero = torch.zeros((b, d), dtype=torch.float64)
    e = zero if dlast is None else dlast.double().cpu()
    s = e.abs()
    first = zero if state is None else state.double().cpu()
    hs, g = states.double().cpu(), dh.double().cpu()
    gx, gx_b = torch.zeros((b, t, d), dtype=torch.float64), torch.zeros((b, t, d), dtype=torch.float64)
    da, da_b = gx.clone(), gx.clone()
    for k in reversed(range(t)):
        live = (k < n).reshape(b, 1)
        c, cs = e + g[:, k], s + g[:, k].abs()
        before = hs[:, k - 1] if k else first
        if mix:
            xv = x.double().cpu()[:, k]
            w, slope, mag = 1 - a[:, k], before - xv, before.abs() + xv.abs()
        else:
            w, slope, mag = torch.ones_like(c), before, before.abs()
        gx[:, k], gx_b[:, k] = torch.where(live, w * c, zero), torch.where(live, w.abs() * cs, zero)
        da[:, k], da_b[:, k] = torch.where(live, c * slope, zero), torch.where(live, cs * mag, zero)
        e, s = torch.where(live, a[:, k] * c, e), torch.where(live, a[:, k].abs() * cs, s)
    r = u(wide(states.dtype))
    back = (t - torch.arange(t, dtype=torch.float64)).reshape(1, t, 1)
    out = [(gx, (2 * back + 12) * r * gx_b), (e, (2 * t + 12) * r * s)]
    if gate is None:
        return out + [None]
    groups = gate.shape[2]
    terms = d // groups * (b if gate.shape[0] < b else 1)

    def shared(v):
        v = v.reshape(b, t, groups, d // groups).sum(3)
        return v.sum(0, keepdim=True) if gate.shape[0] < b else v
    return out + [(shared(da), (2 * back + 14 + terms) * r * shared(da_b))]


# -- row lookup -------------------------------------------------------------------------------------------------------

def make_ids(g, shape, rows, dtype=torch.int64, pad=0.1, kind="uniform"):
    if kind == "one":
        ids = torch.full(shape, max(0, rows - 1), dtype=dtype)
    elif kind == "few":
        ids = (torch.rand(shape, generator=g, dtype=torch.float64) ** 6 * rows).to(dtype)
    else:
        ids = torch.randint(0, max(rows, 1), shape, generator=g, dtype=dtype)
    out = torch.rand(shape, generator=g) < pad
    wrong = torch.tensor([-1, rows, -2**31, 2**31 - 1])[torch.randint(0, 4, shape, generator=g)]
    return torch.where(out, wrong.to(dtype), ids)


LOOKUPS = [((1,), 1, 1), ((0,), 5, 8), ((7,), 3, 5), ((64,), 100, 8), ((257,), 33, 64), ((3, 5), 10, 129), ((2, 3, 4), 50, 256),
           ((1000,), 7, 1), ((513,), 1000, 3), ((130,), 64, 1024), ((65,), 40, 2050), ((5,), 4, 4096), ((40, 300), 90, 1), ((33, 65), 90, 7)]


@gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape,rows,width", LOOKUPS)
def test_lookup_is_the_scaled_row(shape, rows, width, name):
    g = rng(rows * 7 + width)
    table = normal(g, (rows, width), TYPES[name])
    for dtype, scale in ((torch.int64, 1.0), (torch.int32, 0.3)):
        ids = make_ids(g, shape, rows, dtype)
        got = ops.embedding(table.cuda(), ids.cuda(), scale=scale)
        assert got.dtype == table.dtype and got.is_contiguous()
        want = lookup_oracle(table, ids, scale)
        within(got, want, 3 * u(wide(table.dtype)) * want.abs(), table.dtype)
        if scale == 1.0:
            assert torch.equal(got.double().cpu(), want)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f64"])
def test_lookup_reads_strided_tables_and_ids_in_place(name):
    g = rng(3)
    big = normal(g, (40, 6, 72), TYPES[name]).cuda()
    ids = make_ids(g, (70, 130), 40, torch.int32).cuda()
    for table in (big[:, 2, :64], big[:, 0, 1:62], big.transpose(1, 2)[:, :, 3], big[3:4, 0].expand(40, 72), big[::2, 1, 8:24]):
        for i in (ids.t(), ids[::2, ::3], ids[:, 5], ids.t()[4:, 1:], ids.reshape(10, 7, 130).permute(2, 0, 1), ids[:1].expand(9, 130)):
            got = ops.embedding(table, i, scale=0.7)
            want = lookup_oracle(table, i, 0.7)
            within(got, want, 3 * u(wide(table.dtype)) * want.abs(), table.dtype)


@gpu
def test_lookup_passes_on_infinities_and_nan_of_named_rows_only():
    table = torch.ones((4, 16))
    table[1], table[2], table[3] = float("inf"), float("nan"), -float("inf")
    got = ops.embedding(table.cuda(), torch.tensor([0, 1, 2, 3, -1, 4]).cuda(), scale=-2.0).cpu()
    assert torch.equal(got[:, 0].nan_to_num(7.0, 8.0, 9.0), torch.tensor([-2.0, 9.0, 7.0, 8.0, 0.0, 0.0]))


@gpu
def test_lookup_of_offsets_behind_32_bits():
    table = torch.zeros((70000, 32768), dtype=torch.bfloat16, device="cuda")        # 2.3e9 elements
    table[-1] = 3.0
    table[65536] = 5.0
    ids = torch.tensor([69999, 65536, 0, 69999], dtype=torch.int32, device="cuda")
    got = ops.embedding(table, ids)
    assert got.float().mean(1).tolist() == [3.0, 5.0, 0.0, 3.0]
    many = ids.repeat(17500)
    out = ops.embedding(table, many)                                                   # and as many out
    assert out[-4:].float().mean(1).tolist() == [3.0, 5.0, 0.0, 3.0] and out[65538].float().sum() == 0


GRADS = [((0,), 5, 8, "uniform"), ((1,), 1, 1, "uniform"), ((9,), 0, 4, "uniform"), ((40,), 1, 7, "one"), ((300,), 5000, 40, "uniform"),
         ((2000,), 300, 33, "few"), ((5000,), 60, 1, "uniform"), ((4097,), 70000, 3, "uniform"), ((20000,), 40, 64, "one"), ((30000,), 3000, 130, "few"),
         ((70, 300), 900, 1, "uniform"), ((33000,), 257, 2, "few"), ((12, 90, 11), 65537, 8, "uniform"), ((50001,), 70001, 16, "few"),
         ((100000,), 20, 1, "one"), ((70001,), 300, 1, "few")]


@gpu
@pytest.mark.parametrize("shape,rows,width,kind", GRADS)
@pytest.mark.parametrize("name,out", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "f32"), ("f64", "f64")])
def test_lookup_gradient_is_the_sum_over_the_tokens_of_a_row(shape, rows, width, kind, name, out):
    g = rng(rows + width)
    grad = normal(g, (*shape, width), TYPES[name])
    for dtype, pad, scale in ((torch.int64, 0.1, 1.0), (torch.int32, 0.0, -0.3)):
        ids = make_ids(g, shape, rows, dtype, pad, kind)
        got = ops.embedding_grad(grad.cuda(), ids.cuda(), rows, scale=scale, dtype=TYPES[out])
        again = ops.embedding_grad(grad.cuda(), ids.cuda(), rows, scale=scale, dtype=TYPES[out])
        assert got.dtype == TYPES[out] and got.shape == (rows, width) and torch.equal(got, again)
        want, mag, n = lookup_grad_oracle(grad, ids, rows, scale)
        within(got, want, (n + 4).reshape(-1, 1) * u(wide(TYPES[name])) * mag, TYPES[out])
        assert not got[(n == 0).to("cuda")].any()


@gpu
@pytest.mark.parametrize("tokens,rows,width,name", [((40, 20000), 32766, 1, "f32"), ((40, 20000), 32767, 1, "f32"), ((37, 9001), 18203, 1, "f64"), ((70001,), 4001, 3, "f32"),
                                                    ((300, 1700), 9300, 7, "f64"), ((100, 31), 150, 2, "bf16"), ((3100, 100), 400, 1, "f16")])
def test_lookup_gradient_of_few_rows(tokens, rows, width, name):
    """Sums of a column in LDS: tables up to a CU's LDS, lanes that share rows, lines shorter than a step."""
    g = rng(rows)
    grad = normal(g, (*tokens, width), TYPES[name])
    for kind, ids in (("uniform", make_ids(g, tokens, rows, torch.int32, 0.05)), ("few", make_ids(g, tokens, rows, torch.int64, 0.0, "few"))):
        for view, like in ((ids, grad), (ids.transpose(0, -1), grad.transpose(0, -2))):
            got = ops.embedding_grad(_on_gpu(like), _on_gpu(view), rows, scale=0.5, dtype=torch.float32 if name in ("bf16", "f16") else None)
            want, mag, n = lookup_grad_oracle(like, view, rows, 0.5)
            within(got, want, (n + 4).reshape(-1, 1) * u(wide(TYPES[name])) * mag, got.dtype)


@gpu
@pytest.mark.parametrize("tokens,rows,width", [(300, 3000001, 1), (3000, 2000003, 3), (20000, 700001, 40), (5, 400000, 17), (600, 20000000, 1)])
def test_lookup_gradient_of_large_tables(tokens, rows, width):
    g = rng(tokens)
    grad, ids = normal(g, (tokens, width), torch.float32), make_ids(g, (tokens,), rows, torch.int64)
    got = ops.embedding_grad(grad.cuda(), ids.cuda(), rows)
    named = torch.unique(ids[(ids >= 0) & (ids < rows)])
    at = torch.searchsorted(named, ids.clamp(0, rows - 1))
    inner = torch.where((ids >= 0) & (ids < rows), at, torch.full_like(at, -1))
    want, mag, n = lookup_grad_oracle(grad, inner, len(named), 1.0)
    within(got[named.cuda()], want, (n + 4).reshape(-1, 1) * u(torch.float32) * mag, torch.float32)
    got[named.cuda()] = 0
    assert not got.any()


@gpu
def test_lookup_gradient_reads_expanded_and_strided_gradients_in_place():
    g = rng(11)
    ids = make_ids(g, (500, 60), 400, torch.int32)
    per_row = normal(g, (500, 1, 3), torch.float32)
    wide_grad = normal(g, (60, 500, 8), torch.float32)
    for ids_view, grad in ((ids, per_row.expand(500, 60, 3)), (ids.t(), per_row.transpose(0, 1).expand(60, 500, 3)), (ids.t(), wide_grad[:, :, 2:7]),
                           (ids, wide_grad.transpose(0, 1)), (ids[::2, 3:7], wide_grad[3:7, ::2, 1].t().unsqueeze(2))):
        got = ops.embedding_grad(_on_gpu(grad), _on_gpu(ids_view), 400, scale=2.0)
        want, mag, n = lookup_grad_oracle(grad, ids_view, 400, 2.0)
        within(got, want, (n + 4).reshape(-1, 1) * u(torch.float32) * mag, torch.float32)


def _on_gpu(t):
    """A copy on the GPU with the same strides."""
    size = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    flat = torch.as_strided(t, (size,), (1,), t.storage_offset()).cuda()
    return torch.as_strided(flat, t.shape, t.stride())


@gpu
def test_lookup_gradient_equals_differences_of_the_lookup():
    g = rng(5)
    table, ids = normal(g, (30, 6), torch.float64).cuda(), make_ids(g, (200,), 30).cuda()
    weight = normal(g, (200, 6), torch.float64).cuda()
    grad = ops.embedding_grad(weight, ids, 30, scale=0.5)
    for v, k in itertools.product((0, 7, 29), (0, 5)):
        up, down = table.clone(), table.clone()
        up[v, k] += 0.5
        down[v, k] -= 0.5
        diff = (ops.embedding(up, ids, 0.5) * weight).sum() - (ops.embedding(down, ids, 0.5) * weight).sum()
        # linear in the table: the difference is the gradient, up to the roundings of two sums of 1200 terms of about 1
        assert abs(diff.item() - grad[v, k].item()) <= 1200 * 1200 * 8 * u(torch.float64)


# -- recurrence -------------------------------------------------------------------------------------------------------

def make_scan(g, b, t, d, name, gate_name, groups, gate_batch, state, lengths):
    x = normal(g, (b, t, d), TYPES[name])
    gate = None
    if groups:
        a = torch.sigmoid(normal(g, (gate_batch, t, groups), torch.float64) + 1.5)
        pick = torch.rand((gate_batch, t, groups), generator=g)
        a = torch.where(pick < 0.02, torch.zeros_like(a), torch.where(pick > 0.98, torch.ones_like(a), a))
        a = torch.where((pick > 0.5) & (pick < 0.55), -a, a)
        gate = a.to(TYPES[gate_name])
    w = wide(TYPES[name])
    first = normal(g, (b, d), w) if state else None
    n = None
    if lengths:
        n = torch.randint(0, t + 1, (b,), generator=g, dtype=torch.int32)
        n[0], n[-1] = (t, 0) if b > 1 else (max(0, t - 1), max(0, t - 1))
        if b > 3:
            n[1], n[2] = t + 5, -3        # clamped
    return x, gate, first, n


#        batch steps width  type  gate  groups gate_batch mix state lengths
SCANS = [(1, 1, 1, "f32", "f32", 1, 1, False, False, False),
         (3, 1, 64, "bf16", "f32", 64, 3, False, True, False),
         (2, 1, 130, "f16", "f16", 130, 1, True, True, True),
         (2, 2, 5, "f64", "f64", 5, 2, True, True, False),
         (4, 7, 33, "bf16", "bf16", 33, 4, True, True, True),
         (1, 16, 64, "f32", "f32", 0, 0, False, True, False),
         (5, 17, 128, "bf16", "f32", 8, 5, False, True, True),
         (2, 65, 1, "f32", "f32", 1, 1, False, True, True),
         (1, 128, 300, "f64", "f64", 1, 1, True, False, False),
         (3, 129, 96, "f16", "f32", 3, 1, True, True, True),
         (1, 500, 451, "f64", "f64", 0, 0, False, False, False),
         (2, 513, 16, "bf16", "bf16", 16, 2, False, True, False),
         (7, 1000, 3, "f32", "f32", 3, 7, False, True, True),
         (1, 2049, 515, "f32", "f32", 5, 1, False, True, False),
         (4, 300, 256, "bf16", "f32", 256, 4, True, True, True),
         (2, 4097, 66, "f16", "f16", 66, 2, False, False, True),
         (1, 20000, 40, "f32", "f32", 40, 1, True, True, False),
         (65, 40, 24, "bf16", "bf16", 24, 1, False, True, True),
         (3, 700, 128, "f64", "f64", 4, 3, True, True, True),
         # gates shared by whole teams of lanes, by all channels of an odd width, by the batch
         (3, 70, 512, "bf16", "f32", 8, 3, False, True, True),
         (2, 90, 192, "f32", "f32", 2, 1, True, True, False),
         (4, 33, 1536, "f16", "f16", 16, 4, True, False, True),
         (1, 40, 1021, "f32", "f32", 1, 1, True, True, True),
         (6, 300, 64, "f16", "f16", 1, 1, False, True, True),
         (5, 260, 33, "bf16", "bf16", 1, 1, True, False, False),
         (6, 140, 35, "f16", "f32", 35, 1, True, True, True),
         (2, 1, 256, "bf16", "f32", 4, 2, True, True, False),
         (7, 1, 1030, "f32", "f32", 1, 7, False, True, True)]


@gpu
@pytest.mark.parametrize("case", SCANS, ids=lambda c: "-".join(map(str, c)))
def test_recurrence_and_its_gradients_follow_the_formula(case):
    b, t, d, name, gate_name, groups, gate_batch, mix, with_state, with_lengths = case
    g = rng(t * 31 + d)
    x, gate, state, lengths = make_scan(g, b, t, d, name, gate_name, groups, gate_batch, with_state, with_lengths)
    to = lambda v: None if v is None else v.cuda()
    states, last = ops.gated_scan(to(x), to(gate), to(state), mix=mix, lengths=to(lengths))
    again = ops.gated_scan(to(x), to(gate), to(state), mix=mix, lengths=to(lengths))
    assert torch.equal(states, again[0]) and torch.equal(last, again[1])
    assert states.dtype == x.dtype and last.dtype == wide(x.dtype) and states.is_contiguous()
    want, want_last, bound, bound_last = scan_oracle(x, gate, state, mix, lengths)
    within(states, want, bound, x.dtype)
    within(last, want_last, bound_last, last.dtype)

    dh, dlast = normal(g, (b, t, d), x.dtype), normal(g, (b, d), wide(x.dtype)) if with_state else None
    got = ops.gated_scan_grad(to(dh), states, to(gate), to(state), x=to(x), grad_last=to(dlast), mix=mix, lengths=to(lengths))
    again = ops.gated_scan_grad(to(dh), states, to(gate), to(state), x=to(x), grad_last=to(dlast), mix=mix, lengths=to(lengths))
    expect = scan_grad_oracle(dh, states.cpu(), gate, state, x, dlast, mix, lengths)
    for value, same, oracle, dtype in zip(got, again, expect, (x.dtype, wide(x.dtype), None if gate is None else gate.dtype)):
        if oracle is None:
            assert value is None
            continue
        assert value.dtype == dtype and torch.equal(value, same)
        within(value, *oracle, dtype)


@gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_recurrence_reads_strided_tensors_in_place(name):
    g = rng(9)
    big = normal(g, (6, 50, 3, 72), TYPES[name])
    gates = torch.sigmoid(normal(g, (6, 50, 3, 72), TYPES[name]))
    to = _on_gpu
    for x, gate in ((big[:, :, 1, :64], gates[:, :, 2, 4:68]), (big[:, :, 0, 1:62], gates[:1, :, 0, 3:4]), (big[::2, 10:, 2], gates[::2, 10:, 1]),
                    (big.transpose(0, 1)[:, :, 1], gates.transpose(0, 1)[:, :, 0, :8]), (big[:1, :, 0].expand(4, 50, 72), gates[:1, :, 0].expand(4, 50, 72)),
                    (big[:, :, :, 5], gates[:, :, :, 6]), (big.permute(0, 3, 1, 2)[:, :, :, 1], gates.permute(0, 3, 1, 2)[:, :, :, 1])):
        x_g, gate_g = to(x), to(gate)
        states, last = ops.gated_scan(x_g, gate_g, mix=True)
        want, want_last, bound, bound_last = scan_oracle(x, gate, None, True, None)
        within(states, want, bound, x.dtype)
        within(last, want_last, bound_last, last.dtype)
        dh = normal(g, x.shape, x.dtype)
        got = ops.gated_scan_grad(dh.cuda().transpose(0, 1).contiguous().transpose(0, 1), states, gate_g, x=x_g, mix=True)
        for value, oracle, dtype in zip(got, scan_grad_oracle(dh, states.cpu(), gate, None, x, None, True, None), (x.dtype, wide(x.dtype), gate.dtype)):
            within(value, *oracle, dtype)


@gpu
@pytest.mark.parametrize("t,d", [(40, 64), (300, 128), (1500, 37)])
def test_what_stands_behind_a_length_reaches_nothing(t, d):
    g = rng(t)
    x, gate, state, _ = make_scan(g, 4, t, d, "f32", "f32", d, 4, True, False)
    n = torch.tensor([0, 1, t // 2, t], dtype=torch.int32)
    dh, dlast = normal(g, (4, t, d), torch.float32), normal(g, (4, d), torch.float32)
    behind = (torch.arange(t).reshape(1, t, 1) >= n.reshape(4, 1, 1)).expand(4, t, d)
    results = []
    for junk in (0.0, float("nan"), float("inf"), -3e38):
        fill = lambda v: torch.where(behind, torch.full_like(v, junk), v).cuda()
        states, last = ops.gated_scan(fill(x), fill(gate), state.cuda(), lengths=n.cuda(), mix=True)
        assert not states[behind.cuda()].any()
        got = ops.gated_scan_grad(fill(dh), fill(states.cpu()), fill(gate), state.cuda(), x=fill(x), grad_last=dlast.cuda(), mix=True, lengths=n.cuda())
        assert not got[0][behind.cuda()].any() and not got[2][behind.cuda()].any()
        assert torch.equal(last[0].cpu(), state[0]) and torch.equal(got[1][0].cpu(), dlast[0])
        results.append((states, last, *got))
    for other in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(results[0], other))


@gpu
def test_a_gate_of_zero_starts_anew_and_infinities_stay_where_they_are():
    x = torch.ones((2, 600, 64))
    gate = torch.full((2, 600, 64), 0.5)
    x[0, 100] = float("inf")
    x[1, 70, 3] = float("nan")
    states, last = ops.gated_scan(x.cuda(), gate.cuda())
    states = states.cpu()
    assert torch.isfinite(states[0, :100]).all() and torch.isinf(states[0, 100:]).all()
    nan = torch.isnan(states[1])
    assert nan[70:, 3].all() and int(nan.sum()) == 530
    long = ops.gated_scan(torch.ones((1, 3000, 8)).cuda(), torch.zeros((1, 3000, 1)).cuda(), torch.full((1, 8), 1e30).cuda())[0]
    assert torch.equal(long.cpu(), torch.ones((1, 3000, 8)))


@gpu
@pytest.mark.parametrize("mix", [False, True])
def test_pieces_and_single_steps_continue_a_sequence(mix):
    g = rng(21)
    x, gate, state, _ = make_scan(g, 3, 400, 96, "bf16", "f32", 96, 3, True, False)
    x, gate, state = x.cuda(), gate.cuda(), state.cuda()
    whole, last = ops.gated_scan(x, gate, state, mix=mix)
    want, want_last, bound, bound_last = scan_oracle(x, gate, state, mix, None)
    h, pieces = state, []
    for at in [0, 1, 2, 3, 50, 51, 180, 399]:
        end = {0: 1, 1: 2, 2: 3, 3: 50, 50: 51, 51: 180, 180: 399, 399: 400}[at]
        part, h = ops.gated_scan(x[:, at:end], gate[:, at:end], h, mix=mix)
        pieces.append(part)
    within(torch.cat(pieces, 1), want, bound, torch.bfloat16)
    within(h, want_last, bound_last, torch.float32)
    within(whole, want, bound, torch.bfloat16)


@gpu
def test_gradients_of_the_recurrence_equal_differences():
    g = rng(2)
    b, t, d = 2, 70, 6
    x, gate, state, _ = make_scan(g, b, t, d, "f64", "f64", 3, 1, True, False)
    n = torch.tensor([70, 41], dtype=torch.int32).cuda()
    x, gate, state = x.cuda(), gate.cuda(), state.cuda()
    weight, weight_last = normal(g, (b, t, d), torch.float64).cuda(), normal(g, (b, d), torch.float64).cuda()

    def loss(x, gate, state):
        states, last = ops.gated_scan(x, gate, state, mix=True, lengths=n)
        return ((states * weight).sum() + (last * weight_last).sum()).item()
    states, _ = ops.gated_scan(x, gate, state, mix=True, lengths=n)
    grads = ops.gated_scan_grad(weight, states, gate, state, x=x, grad_last=weight_last, mix=True, lengths=n)
    step = 1e-4
    for which, (value, grad) in enumerate(zip((x, state, gate), grads)):
        for at in range(0, value.numel(), max(1, value.numel() // 17)):
            moved = []
            for sign in (1, -1):
                copy = value.clone()
                copy.view(-1)[at] += sign * step
                args = [x, gate, state]
                args[(0, 2, 1)[which]] = copy
                moved.append(loss(*args))
            # values about 10, summed over 840 terms: 1e-9 from roundings over 2e-4, 1e-8 (cubic term) from the step
            assert abs((moved[0] - moved[1]) / (2 * step) - grad.view(-1)[at].item()) <= 1e-4


@gpu
def test_recurrence_of_offsets_behind_32_bits():
    t, d = 66000, 32768                                             # 2.16e9 values, 4.3 GB
    x = torch.zeros((1, t, d), dtype=torch.bfloat16, device="cuda")
    x[0, 3], x[0, -2] = 1.0, 2.0
    gate = torch.ones((1, t, 1), dtype=torch.bfloat16, device="cuda")
    states, last = ops.gated_scan(x, gate)
    assert torch.equal(last, torch.full_like(last, 3.0))
    for at, want in ((2, 0.0), (3, 1.0), (t - 3, 1.0), (t - 2, 3.0), (t - 1, 3.0)):
        assert states[0, at].eq(want).all()
    grad_x, grad_state, grad_gate = ops.gated_scan_grad(x, states, gate)
    assert grad_state.eq(3.0).all() and grad_x[0, t - 1].eq(0).all() and grad_x[0, t - 2].eq(2).all() and grad_x[0, 0].eq(3).all()
    # da[t] = sum over the channels of c[t] h[t-1]: 32768 of 2 * 1 at t - 2, none where either is zero
    assert grad_gate[0, t - 2, 0].item() == 65536.0 and grad_gate[0, 3, 0].item() == 0.0 and grad_gate[0, t - 1, 0].item() == 0.0


# -- streams, graphs, empties -----------------------------------------------------------------------------------------

def _everything(seed, t=300, d=96):
    g = rng(seed)
    ids = make_ids(g, (2, t), 700, torch.int64, kind="few").cuda()
    table = normal(g, (700, d), torch.bfloat16).cuda()
    gate = torch.sigmoid(normal(g, (2, t, d), torch.float32)).cuda()
    dh = normal(g, (2, t, d), torch.bfloat16).cuda()
    return ids, table, gate, dh


def _chain(ids, table, gate, dh):
    """Lookup, recurrence and both gradients, as a training step runs them, and the gradient of a forest's leaves."""
    leaves = (ids.reshape(-1, 1) * 31 + torch.arange(200, device="cuda")) % 20001
    grad_leaves = ops.embedding_grad(gate.reshape(-1)[:len(leaves)].reshape(-1, 1, 1).expand(-1, 200, 1), leaves, 20001)
    return (*_step(ids, table, gate, dh), grad_leaves)


def _step(ids, table, gate, dh):
    x = ops.embedding(table, ids, scale=2.0)
    states, last = ops.gated_scan(x, gate, mix=True)
    grad_x, grad_state, grad_gate = ops.gated_scan_grad(dh, states, gate, x=x, mix=True)
    grad_table = ops.embedding_grad(grad_x, ids, table.shape[0], scale=2.0, dtype=torch.float32)
    return x, states, last, grad_x, grad_state, grad_gate, grad_table


@gpu
@pytest.mark.parametrize("t,d", [(1, 64), (60, 96), (300, 96), (2500, 130)])
def test_a_training_step_of_all_four_follows_the_formulas(t, d):
    ids, table, gate, dh = _everything(t, t, d)
    x, states, last, grad_x, grad_state, grad_gate, grad_table = _step(ids, table, gate, dh)
    want = lookup_oracle(table, ids, 2.0)
    assert torch.equal(x.double().cpu(), want)
    want, want_last, bound, bound_last = scan_oracle(x, gate, None, True, None)
    within(states, want, bound, torch.bfloat16)
    for value, oracle, dtype in zip((grad_x, grad_state, grad_gate), scan_grad_oracle(dh, states.cpu(), gate.cpu(), None, x.cpu(), None, True, None),
                                    (torch.bfloat16, torch.float32, torch.float32)):
        within(value, *oracle, dtype)
    want, mag, n = lookup_grad_oracle(grad_x, ids, 700, 2.0)
    within(grad_table, want, (n + 4).reshape(-1, 1) * u(torch.float32) * mag, torch.float32)


@gpu
def test_captured_graphs_replay_and_share_nothing():
    steps = [_everything(1), _everything(2, 2500, 130)]
    want = [[v.clone() for v in _chain(*s)] for s in steps]
    graphs, outs, inputs = [], [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in steps:
            _chain(*s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for s in steps:
        still = [torch.zeros_like(v) for v in s]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _chain(*still)
        graphs.append(graph)
        outs.append(out)
        inputs.append(still)
    streams = [torch.cuda.Stream() for _ in steps]
    for replay in range(4):
        for k, s in enumerate(steps):
            for dst, src in zip(inputs[k], s):
                dst.copy_(src)
        torch.cuda.synchronize()
        for k in range(len(steps)):             # both at once
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        eager = _chain(*steps[replay % 2])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, want[replay % 2]))
        for k in range(len(steps)):
            assert all(torch.equal(p, q) for p, q in zip(outs[k], want[k])), (replay, k)
            for v in outs[k]:
                v.zero_()


@gpu
def test_two_streams_and_threads_at_once():
    import threading
    steps = [_everything(k, 400 + 37 * k, 64 + 32 * k) for k in range(4)]
    want = [[v.clone() for v in _chain(*s)] for s in steps]
    torch.cuda.synchronize()
    got = [None] * len(steps)

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(5):
                got[k] = _chain(*steps[k])
        stream.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(steps))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@gpu
def test_empty_tensors():
    dev = "cuda"
    assert ops.embedding(torch.ones((0, 4), device=dev), torch.tensor([0, 1], device=dev)).eq(0).all()
    assert ops.embedding(torch.ones((3, 0), device=dev), torch.tensor([0, 1], device=dev)).shape == (2, 0)
    assert ops.embedding_grad(torch.ones((0, 4), device=dev), torch.zeros(0, dtype=torch.int32, device=dev), 3).eq(0).all()
    state = torch.full((2, 5), 3.0, device=dev)
    states, last = ops.gated_scan(torch.ones((2, 0, 5), device=dev), torch.ones((2, 0, 5), device=dev), state)
    assert states.shape == (2, 0, 5) and torch.equal(last, state)
    for shape in ((2, 0, 3, 0), (0, 2, 3), (2, 3, 0), (0,)):
        none = torch.zeros(shape, dtype=torch.int32, device=dev)
        assert ops.embedding(torch.ones((3, 2), device=dev), none).shape == (*shape, 2)
        assert not ops.embedding_grad(torch.ones((*shape, 2), device=dev), none, 4).any()
    gx, gs, gg = ops.gated_scan_grad(states, states, torch.ones((2, 0, 5), device=dev), state, grad_last=2 * state)
    assert gx.shape == (2, 0, 5) and torch.equal(gs, 2 * state) and gg.shape == (2, 0, 5)
    for shape in ((0, 7, 5), (2, 7, 0)):
        x = torch.ones(shape, device=dev)
        states, last = ops.gated_scan(x, torch.ones((1, 7, 1), device=dev), mix=True)
        gx, gs, gg = ops.gated_scan_grad(x, states, torch.ones((1, 7, 1), device=dev), x=x, mix=True)
        assert states.shape == gx.shape == shape and gg.shape == (1, 7, 1) and not gg.any()


# -- refusals (no GPU needed: arguments are looked at first) ---------------------------------------------------------

_X, _I = torch.ones((2, 3, 4)), torch.zeros(3, dtype=torch.int64)
REFUSED = {
    "table is no tensor": lambda: ops.embedding(np.ones((2, 3)), _I),
    "table of whole numbers": lambda: ops.embedding(torch.ones((2, 3), dtype=torch.int32), _I),
    "table of one dimension": lambda: ops.embedding(torch.ones(3), _I),
    "ids of floats": lambda: ops.embedding(torch.ones((2, 3)), torch.zeros(3)),
    "ids of bytes": lambda: ops.embedding(torch.ones((2, 3)), torch.zeros(3, dtype=torch.uint8)),
    "table on the CPU": lambda: ops.embedding(torch.ones((2, 3)), _I),
    "table with autograd": lambda: ops.embedding(torch.ones((2, 3), requires_grad=True), _I),
    "gradient of another shape": lambda: ops.embedding_grad(torch.ones((4, 3)), _I, 5),
    "gradient without a width": lambda: ops.embedding_grad(torch.ones(3), _I, 5),
    "negative rows": lambda: ops.embedding_grad(torch.ones((3, 2)), _I, -1),
    "too many rows": lambda: ops.embedding_grad(torch.ones((3, 2)), _I, 2**31),
    "half a row": lambda: ops.embedding_grad(torch.ones((3, 2)), _I, 1.5),
    "narrower result": lambda: ops.embedding_grad(torch.ones((3, 2)), _I, 5, dtype=torch.bfloat16),
    "wider result": lambda: ops.embedding_grad(torch.ones((3, 2)), _I, 5, dtype=torch.float64),
    "gradient on the CPU": lambda: ops.embedding_grad(torch.ones((3, 2)), _I, 5),
    "x of two dimensions": lambda: ops.gated_scan(torch.ones((2, 3))),
    "x of whole numbers": lambda: ops.gated_scan(_X.long()),
    "gate of another batch": lambda: ops.gated_scan(_X, torch.ones((3, 3, 4))),
    "gate of other steps": lambda: ops.gated_scan(_X, torch.ones((2, 2, 4))),
    "gate of three groups": lambda: ops.gated_scan(_X, torch.ones((2, 3, 3))),
    "gate without groups": lambda: ops.gated_scan(_X, torch.ones((2, 3, 0))),
    "gate of two dimensions": lambda: ops.gated_scan(_X, torch.ones((2, 3))),
    "gate of 64 bits": lambda: ops.gated_scan(_X, torch.ones((2, 3, 4), dtype=torch.float64)),
    "gate of 16 bits": lambda: ops.gated_scan(_X, torch.ones((2, 3, 4), dtype=torch.bfloat16)),
    "state of 16 bits": lambda: ops.gated_scan(_X.bfloat16(), None, torch.ones((2, 4), dtype=torch.bfloat16)),
    "state of another shape": lambda: ops.gated_scan(_X, None, torch.ones((2, 3))),
    "lengths of 64 bits": lambda: ops.gated_scan(_X, lengths=torch.ones(2, dtype=torch.int64)),
    "lengths of another batch": lambda: ops.gated_scan(_X, lengths=torch.ones(3, dtype=torch.int32)),
    "mixed form without a gate": lambda: ops.gated_scan(_X, mix=True),
    "x on the CPU": lambda: ops.gated_scan(_X),
    "x with autograd": lambda: ops.gated_scan(_X.clone().requires_grad_()),
    "gradient of another type": lambda: ops.gated_scan_grad(_X.bfloat16(), _X),
    "gradient of other steps": lambda: ops.gated_scan_grad(_X[:, :2], _X),
    "x of another shape": lambda: ops.gated_scan_grad(_X, _X, torch.ones((2, 3, 4)), x=_X[:1], mix=True),
    "mixed gradient without x": lambda: ops.gated_scan_grad(_X, _X, torch.ones((2, 3, 4)), mix=True),
    "last gradient of another shape": lambda: ops.gated_scan_grad(_X, _X, grad_last=torch.ones((2, 3))),
    "states on the CPU": lambda: ops.gated_scan_grad(_X, _X),
}


@pytest.mark.parametrize("what", REFUSED)
def test_refused(what):
    with pytest.raises(LightGBMError):
        REFUSED[what]()


@gpu
def test_tensors_of_different_devices_are_refused():
    with pytest.raises(LightGBMError, match="tensors on"):
        ops.embedding(torch.ones((2, 3)).cuda(), _I)
    with pytest.raises(LightGBMError, match="tensors on"):
        ops.gated_scan(_X.cuda(), torch.ones((2, 3, 4)))


# -- views whose memory is not what they say --------------------------------------------------------------------------

def _negated(t):
    """Equal to ``t``, with -t in memory and torch's negative bit set."""
    view = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert view.is_neg() and torch.equal(view, t)
    return view


def test_arguments_are_taken_as_their_memory_has_to_be_read():
    from lightgbm_amd.ops import _args
    v = torch.arange(1.0, 4.0).reshape(3, 1)
    got = _args.need_tensor("op", "x", _negated(v))
    assert not got.is_neg() and torch.equal(got, v)
    assert _args.need_tensor("op", "x", v) is v


@gpu
@pytest.mark.parametrize("width", [1, 6])
@pytest.mark.parametrize("name", ["f32", "f64"])
def test_negated_views_are_read_with_their_sign(name, width):
    g = rng(width)
    ids = make_ids(g, (3, 20), 30).cuda()
    table, grad, x, dh, state, dlast = (normal(g, shape, TYPES[name]).cuda()
                                        for shape in ((30, width), (3, 20, width), (3, 20, width), (3, 20, width), (3, width), (3, width)))
    gate = torch.sigmoid(normal(g, (3, 20, 1), TYPES[name])).cuda()
    assert torch.equal(ops.embedding(_negated(table), ids), ops.embedding(table, ids))
    assert torch.equal(ops.embedding_grad(_negated(grad), ids, 30), ops.embedding_grad(grad, ids, 30))
    want = ops.gated_scan(x, gate, state, mix=True)
    got = ops.gated_scan(_negated(x), _negated(gate), _negated(state), mix=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    states = want[0]
    want = ops.gated_scan_grad(dh, states, gate, state, x=x, grad_last=dlast, mix=True)
    got = ops.gated_scan_grad(_negated(dh), _negated(states), _negated(gate), _negated(state), x=_negated(x), grad_last=_negated(dlast), mix=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


DUALS = {
    "table": lambda d: ops.embedding(d(30, 4), _I),
    "grad": lambda d: ops.embedding_grad(d(3, 4), _I, 5),
    "x": lambda d: ops.gated_scan(d(2, 3, 4)),
    "gate": lambda d: ops.gated_scan(_X, d(2, 3, 4)),
    "state": lambda d: ops.gated_scan(_X, None, d(2, 4)),
    "grad_states": lambda d: ops.gated_scan_grad(d(2, 3, 4), _X),
    "states": lambda d: ops.gated_scan_grad(_X, d(2, 3, 4)),
    "x of the gradient": lambda d: ops.gated_scan_grad(_X, _X, torch.ones((2, 3, 4)), x=d(2, 3, 4), mix=True),
    "grad_last": lambda d: ops.gated_scan_grad(_X, _X, grad_last=d(2, 4)),
}


@pytest.mark.parametrize("what", DUALS)
def test_dual_tensors_are_refused(what):
    """Their tangents would be dropped without a word; under no_grad() too, which leaves forward mode on."""
    from torch.autograd import forward_ad
    for grad_mode in (torch.enable_grad, torch.no_grad):
        with forward_ad.dual_level(), grad_mode():
            with pytest.raises(LightGBMError, match="dual"):
                DUALS[what](lambda *shape: forward_ad.make_dual(torch.ones(shape), torch.ones(shape)))
            with pytest.raises(LightGBMError, match="GPU"):          # others are taken inside a level too
                DUALS[what](lambda *shape: torch.ones(shape))


# -- products of gates beyond the type's range --------------------------------------------------------------------------

#         type  steps state     gate
FADING = [("f32", 300, 1e30, 0.5), ("f32", 3000, 1e30, -0.5), ("f32", 1000, 1.2e30, 0.9), ("f32", 700, 3e38, 0.8), ("f32", 40, 1e30, 2.0**-20),
          ("f32", 2100, 1e30, 2.0**-140), ("bf16", 700, 1e30, 0.5), ("f64", 3000, 1e300, 0.5), ("f64", 5000, 1e300, -0.81), ("f64", 300, 1e300, 2.0**-60),
          # products above the range too, of states that stay within it
          ("f32", 200, 2.0**-120, 2.0), ("f32", 600, 0.0, 4.0), ("f64", 1200, 2.0**-1000, 2.0), ("f64", 700, 0.0, 2.0**9)]


@gpu
@pytest.mark.parametrize("groups", [1, 24])
@pytest.mark.parametrize("name,t,start,factor", FADING)
def test_products_of_gates_leave_the_range_and_states_do_not(name, t, start, factor, groups):
    """What is left of a state is the product of many gates times a large (small, no) number, whatever the product alone is."""
    g = rng(t)
    b, d = 2, 24
    x, w = torch.zeros((b, t, d), dtype=TYPES[name]), wide(TYPES[name])
    x[:, -1] = 1.0
    gate = torch.full((b, t, groups), factor, dtype=w)
    gate[1, t // 2:] = gate[1, t // 2:].abs().clamp(max=1.0)
    state = start * (1 + 0.1 * torch.rand((b, d), generator=g, dtype=w))
    states, last = ops.gated_scan(x.cuda(), gate.cuda(), state.cuda())
    want, want_last, bound, bound_last = scan_oracle(x, gate, state, False, None)
    within(states, want, bound, x.dtype)
    within(last, want_last, bound_last, w)

    x, gate = x.flip(1), gate.flip(1)                       # backwards the gradient of the last state fades
    before = torch.zeros_like(x)
    got = ops.gated_scan_grad(x.cuda(), before.cuda(), gate.cuda(), grad_last=state.cuda())
    for value, oracle, dtype in zip(got, scan_grad_oracle(x, before, gate, None, None, state, False, None), (x.dtype, w, w)):
        within(value, *oracle, dtype)


@gpu
@pytest.mark.parametrize("name,factor", [("f32", 2.0**-30), ("f32", -0.5), ("f64", 2.0**-300), ("f64", -0.5)])
def test_infinite_states_stay_infinite_under_gates_that_are_not_zero(name, factor):
    t = 2501
    w = TYPES[name]
    state = torch.tensor([[float("inf"), -float("inf"), 1.0, 0.0]], dtype=w)
    zero = torch.zeros((1, t, 4), dtype=w)
    gate = torch.full((1, t, 1), factor, dtype=w)
    sign = torch.sign(torch.tensor(factor, dtype=w)) ** torch.arange(1, t + 1, dtype=w)
    _, last = ops.gated_scan(zero.cuda(), gate.cuda(), state.cuda())
    assert last.cpu().tolist() == [[sign[-1].item() * float("inf"), -sign[-1].item() * float("inf"), 0.0, 0.0]]
    gate[0, 1700] = 0.0                                      # 0 * inf, as step by step
    states, last = ops.gated_scan(zero.cuda(), gate.cuda(), state.cuda())
    states = states.cpu()
    assert torch.equal(states[0, :1700, 0], sign[:1700] * float("inf")) and states[0, 1700:, :2].isnan().all() and states[0, 1700:, 2:].eq(0).all()
    _, grad_state, _ = ops.gated_scan_grad(zero.cuda(), zero.cuda(), gate.abs().clamp(min=0.25).cuda(), grad_last=state.cuda())
    assert grad_state.cpu().tolist() == [[float("inf"), -float("inf"), 0.0, 0.0]]


@gpu
@pytest.mark.parametrize("name,power", [("f32", 9), ("f64", 80)])
def test_a_gate_of_zero_between_large_gates_leaves_nothing(name, power):
    """The product of a run is zero, and so is what it leaves of a state, however large the gates around the zero are."""
    t, w = 700, TYPES[name]
    gate = torch.full((1, t, 1), 2.0**power, dtype=w)
    zeros = [5, 300, 301]
    gate[0, zeros] = 0.0
    x = torch.zeros((1, t, 8), dtype=w)
    state = torch.linspace(-1.0, 1.0, 8, dtype=w).reshape(1, 8)
    states, last = ops.gated_scan(x.cuda(), gate.cuda(), state.cuda())
    assert not states[0, 5:].any() and not last.any()
    want = torch.ldexp(state.double(), power * torch.arange(1, 6).reshape(1, 5, 1))
    assert torch.equal(states[:, :5].cpu().double(), want)               # powers of two: exact
    _, grad_state, grad_gate = ops.gated_scan_grad(x.cuda(), states, gate.flip(1).cuda(), grad_last=state.cuda())
    assert not grad_state.any()
    assert torch.isfinite(grad_gate).all()


# -- token grids with a short axis ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("n0,n1", [(1000000, 2), (1000000, 3), (90001, 33), (50001, 65), (3000, 1001), (65, 50001), (33, 90001), (3, 1000000),
                                   (2**30 - 1, 2), (715827882, 3), (65075262, 33), (33038209, 65), (16519104, 130), (46340, 46341), (65, 33038209),
                                   (33, 65075262), (2, 2**30 - 1), (1, 2**31 - 1)])
def test_sorted_token_grids_are_filled_up_to_less_than_twice_their_size(n0, n1):
    """The core sizes its workspace on the host: 16 bytes of ids and token numbers a slot, up to 2 of counts, a few thousandths of
    partial sums, 1 a table row; a slot belongs to a token or fills up a tile of at most 4096, and there are less than two a
    token and some tiles at the edges (at most one row of tiles of 64 and one column, or 2 MB)."""
    import ctypes
    from lightgbm_amd import _lib, build
    from lightgbm_amd.ops import lookup
    lib, hip = _lib.load()
    if not hip:
        path = build.PKG / "_lga_hip.so"
        if not path.exists():
            pytest.skip("the HIP core is not built")
        lib = ctypes.CDLL(str(path))
        lib.lga_hip_embedding_grad.argtypes = [ctypes.c_char_p, ctypes.POINTER(ctypes.c_int64)]
        lib.lga_last_error.restype = ctypes.c_char_p
    rows, tokens = 200000, n0 * n1
    for ids_stride in ((n1 + 1, 1), (1, n0 + 1)):
        for grad_stride in ((n1 + 1, 1), (1, n0 + 1)):
            need = ctypes.c_int64()
            words = lookup._LOOKUP_GRAD.pack(1, 1, 1, 0, 0, 0, rows, 1, n0, n1, *ids_stride, *grad_stride, 2, 2, 0, 1.0)      # no workspace: only its size
            assert lib.lga_hip_embedding_grad(words, need) == 0, lib.lga_last_error()
            assert tokens * 16 <= need.value <= 2 * 18.1 * tokens + rows + 2**21


SHORT_AXIS = [((300001, 2), 70001, 1, "f32"), ((2, 300001), 70001, 1, "f64"), ((40001, 3), 70001, 2, "bf16"), ((30007, 3), 300, 1, "f64"),
              ((9001, 5), 20000, 40, "f32"), ((2049, 33), 60000, 3, "f16"), ((2049, 65), 60000, 1, "f64"), ((300, 129), 60000, 7, "f32"), ((5000001, 2), 500, 1, "bf16")]


@gpu
@pytest.mark.parametrize("shape,rows,width,name", SHORT_AXIS)
def test_token_grids_with_a_short_axis(shape, rows, width, name):
    """Ids that cannot merge to one axis, either one's neighbours next to each other: lookup and gradient."""
    g = rng(rows + shape[0])
    whole = make_ids(g, (shape[0], shape[1] + 1), rows, torch.int32, 0.05)
    table, grad = normal(g, (rows, width), TYPES[name]), normal(g, (*shape, width), TYPES[name])
    table_g, grad_g = table.cuda(), grad.cuda()
    ids = whole[:, 1:]
    looked = lookup_oracle(table, ids, 0.3)
    want, mag, n = lookup_grad_oracle(grad, ids, rows, 0.3)
    # all of 1e7 tokens to 500 rows in 16 bits: the count of a row's tokens times u(fp32) stays far below one
    for view in (whole.cuda()[:, 1:], whole.t().contiguous().cuda().t()[:, 1:]):
        assert torch.equal(view.cpu(), ids) and not view.is_contiguous()
        within(ops.embedding(table_g, view, 0.3), looked, 3 * u(wide(TYPES[name])) * looked.abs(), TYPES[name])
        got = ops.embedding_grad(grad_g, view, rows, scale=0.3, dtype=torch.float32 if name in ("bf16", "f16") else None)
        within(got, want, (n + 4).reshape(-1, 1) * u(wide(TYPES[name])) * mag, got.dtype)
        got = ops.embedding_grad(grad_g.transpose(0, 1), view.t(), rows, scale=0.3, dtype=got.dtype)
        within(got, want, (n + 4).reshape(-1, 1) * u(wide(TYPES[name])) * mag, got.dtype)


@gpu
def test_threads_with_tables_of_different_lds_sizes():
    """Sums of few rows take 66 to 160 KB of LDS a wave here; the launch limit is one of the process, set by every thread."""
    import threading
    g = rng(77)
    steps = []
    for rows in (18000, 7400, 12000, 9000):
        grad = normal(g, (20 * rows, 1), torch.float64).cuda()
        steps.append((grad, make_ids(g, (20 * rows,), rows, torch.int32).cuda(), rows))
    want = [ops.embedding_grad(*s) for s in steps]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        stream = torch.cuda.Stream()
        try:
            with torch.cuda.stream(stream):
                got = [ops.embedding_grad(*steps[k]) for _ in range(40)]
            stream.synchronize()
            wrong.extend(k for v in got if not torch.equal(v, want[k]))
        except Exception as e:                     # noqa: BLE001 - of any kind, for the assertion below
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(steps))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong
    for (grad, ids, rows), got in zip(steps, want):
        expect, mag, n = lookup_grad_oracle(grad, ids, rows, 1.0)
        within(got, expect, (n + 4).reshape(-1, 1) * u(torch.float64) * mag, torch.float64)


RELEASED = {
    "table": lambda d, x: ops.embedding(d(30, 4), _I.to(x.device)),
    "strided table": lambda d, x: ops.embedding(d(4, 30, columns=True), _I.to(x.device)),
    "ids": lambda d, x: ops.embedding(x[0], d(3).view(torch.int32)),
    "grad": lambda d, x: ops.embedding_grad(d(3, 4), _I.to(x.device), 5),
    "x": lambda d, x: ops.gated_scan(d(2, 3, 4)),
    "gate": lambda d, x: ops.gated_scan(x, d(2, 3, 4)),
    "state": lambda d, x: ops.gated_scan(x, None, d(2, 4)),
    "lengths": lambda d, x: ops.gated_scan(x, lengths=d(2).view(torch.int32)),
    "grad_states": lambda d, x: ops.gated_scan_grad(d(2, 3, 4), x),
    "states": lambda d, x: ops.gated_scan_grad(x, d(2, 3, 4)),
    "x of the gradient": lambda d, x: ops.gated_scan_grad(x, x, torch.ones_like(x), x=d(2, 3, 4), mix=True),
    "grad_last": lambda d, x: ops.gated_scan_grad(x, x, grad_last=d(2, 4)),
}


def _released(what, device):
    """Parameters whose storage a sharding wrapper has taken back keep their shape and have the address 0."""
    def make(*shape, columns=False):
        t = torch.ones(shape, device=device)
        t = t.t() if columns else t
        t.untyped_storage().resize_(0)
        return t
    with pytest.raises(LightGBMError, match="no memory"):
        RELEASED[what](make, _X.to(device))


@pytest.mark.parametrize("what", RELEASED)
def test_tensors_without_memory_are_refused(what):
    _released(what, "cpu")


@gpu
@pytest.mark.parametrize("what", RELEASED)
def test_gpu_tensors_without_memory_are_refused(what):
    _released(what, "cuda")


# -- every variant of the lookup's gradient ------------------------------------------------------------------------------

#         tokens shape    rows  width type  transposed
PATHS = [((3000,), 3000, 1, "f64", False),             # sorted by one workgroup, 8 bytes carried
         ((60000,), 70000, 1, "f64", False),           # few small tiles, 8 bytes
         ((190000,), 60000, 1, "f64", False),          # offsets by a kernel of their own, 8 bytes
         ((210007,), 90000, 1, "f32", False), ((71, 3001), 60000, 2, "bf16", True),
         ((300, 16411), 400000, 1, "f64", True),       # tiles of 4096, 8 bytes; ids the other way round, ragged edges
         ((16411, 300), 400000, 1, "f32", True),       # 4 bytes, values carried
         ((67, 70003), 300000, 3, "f32", False), ((4400000,), 280000, 1, "f16", False),      # 4 bytes, token numbers carried
         ((1300000,), 82000, 17, "bf16", False),       # strips of 64 tokens and more
         ((2200, 1000), 140000, 24, "f32", True), ((1400001,), 90000, 40, "f16", False),
         ((8400001,), 530000, 17, "bf16", False)]


@gpu
@pytest.mark.parametrize("shape,rows,width,name,transposed", PATHS)
def test_lookup_gradient_of_many_tokens(shape, rows, width, name, transposed):
    """Sizes that reach the sorts of 4 and 8 bytes by one workgroup, by small and by large tiles, with and without a kernel of its
    own for the offsets, and the longer strips.  The oracle sums on the GPU in 64 bits, with torch."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    ids = (torch.rand(shape, generator=g, device="cuda", dtype=torch.float64) ** 2 * (rows + 3)).to(torch.int32) - 1
    grad = torch.randn((*shape, width), generator=g, device="cuda", dtype=wide(TYPES[name])).to(TYPES[name])
    if transposed:
        ids = ids.t().contiguous().t()
    got = ops.embedding_grad(grad, ids, rows, scale=0.5, dtype=torch.float32 if name in ("bf16", "f16") else None)
    assert torch.equal(got, ops.embedding_grad(grad, ids, rows, scale=0.5, dtype=got.dtype))
    i = ids.reshape(-1).long()
    i = torch.where((i >= 0) & (i < rows), i, torch.full_like(i, rows))
    want, mag = torch.zeros((2, rows + 1, width), dtype=torch.float64, device="cuda")
    g64 = grad.reshape(-1, width).double()
    # atomic additions in 64 bits: their order costs n u(fp64), which for fp64 the bound counts twice
    want.index_add_(0, i, g64)
    mag.index_add_(0, i, g64.abs())
    n = torch.bincount(i, minlength=rows + 1).double()
    want, mag, n = (0.5 * want[:rows]).cpu(), (0.5 * mag[:rows]).cpu(), n[:rows].cpu()
    within(got, want, (2 * n + 4).reshape(-1, 1) * u(wide(TYPES[name])) * mag, got.dtype)


@gpu
@pytest.mark.parametrize("name", ["f64", "f32", "bf16"])
@pytest.mark.parametrize("width", [1, 2])
def test_lookup_of_many_narrow_rows(name, width):
    """More tokens than small tiles are taken for, ids the other way round, edges that fill no tile."""
    g = torch.Generator(device="cuda").manual_seed(width)
    ids = torch.randint(-1, 38102, (15013, 301), generator=g, device="cuda", dtype=torch.int32)
    table = torch.randn((38101, width), generator=g, device="cuda", dtype=torch.float64).to(TYPES[name])
    padded = torch.cat([table, torch.zeros((1, width), dtype=table.dtype, device="cuda")])
    for view in (ids, ids.t(), ids[1:, 3:], ids.t()[2:, 5:], ids.long().t()):
        want = padded[torch.where((view >= 0) & (view < 38101), view, torch.full_like(view, 38101)).long()]
        assert torch.equal(ops.embedding(table, view), want)


#        tokens rows width type: sums in one workgroup's list, sums in LDS, sorted by one workgroup, by tiles, wide rows
ODD = [(300, 50, 3, "f32"), (40000, 500, 1, "f32"), (40000, 500, 2, "bf16"), (3000, 3000, 1, "f64"), (3000, 3000, 2, "f16"), (90000, 40000, 1, "f64"),
       (90000, 40000, 5, "f32"), (3000, 2000, 40, "bf16"), (50000, 20000, 24, "f64")]


@gpu
@pytest.mark.parametrize("tokens,rows,width,name", ODD)
def test_infinite_and_nan_gradients_reach_their_own_rows_only(tokens, rows, width, name):
    g = rng(tokens + width)
    ids = make_ids(g, (tokens,), rows, torch.int32, 0.1)
    grad = normal(g, (tokens, width), TYPES[name])
    clean = ops.embedding_grad(grad.cuda(), ids.cuda(), rows).cpu()
    inside = (ids >= 0) & (ids < rows)
    used = torch.nonzero(inside).reshape(-1)
    named = torch.unique(ids[inside])
    for tok in torch.nonzero(~inside).reshape(-1)[:20].tolist():          # padding: whatever it holds
        grad[tok] = float("nan")
    plus, nan, both = named[1].item(), named[len(named) // 2].item(), named[-1].item()
    first = {r: used[ids[used] == r][0].item() for r in (plus, nan, both)}
    grad[first[plus], 0], grad[first[nan], width - 1], grad[first[both], 0] = float("inf"), float("nan"), -float("inf")
    if int((ids == both).sum()) > 1:
        grad[used[ids[used] == both][-1], 0] = float("inf")               # inf - inf
    got = ops.embedding_grad(grad.cuda(), ids.cuda(), rows).cpu()
    want, _, _ = lookup_grad_oracle(torch.where(torch.isfinite(grad), torch.zeros_like(grad), grad), ids, rows, 1.0)
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    assert torch.equal(got[odd & torch.isinf(want)].double(), want[odd & torch.isinf(want)])
    assert torch.equal(got[~odd], clean[~odd])                            # and no other value changes by a bit


@gpu
@pytest.mark.parametrize("tokens,rows,width", [(300, 50, 3), (40000, 500, 1), (3000, 3000, 2), (50000, 20000, 24)])
def test_scales_that_are_not_finite_are_refused_by_every_variant(tokens, rows, width):
    """Times infinity a row that no id names would be NaN, not zero."""
    grad, ids = torch.ones((tokens, width), device="cuda"), torch.zeros(tokens, dtype=torch.int32, device="cuda")
    for scale in (float("inf"), -float("inf"), float("nan"), 1e39):          # the last one in fp32
        with pytest.raises(LightGBMError, match="finite"):
            ops.embedding_grad(grad, ids, rows, scale=scale)
    got = ops.embedding_grad(grad.double(), ids, rows, scale=1e39)
    assert got[0].eq(tokens * 1e39).all() or (got[0] / (tokens * 1e39) - 1).abs().max() < 1e-12
    assert not got[1:].any()


#            ids' shape   rows  width type: one list, LDS sums of up to 64 KB and above, sorted by one workgroup, by small and large tiles
CAPTURED = [((300,), 50, 3, "f32"), ((70, 300), 900, 1, "f32"), ((40, 8000), 15000, 1, "f64"), ((3000,), 3000, 2, "f16"), ((60000,), 70000, 1, "f64"),
            ((300, 16411), 400000, 1, "f32"), ((50000,), 20000, 24, "bf16")]


@gpu
@pytest.mark.parametrize("shape,rows,width,name", CAPTURED)
def test_every_variant_of_the_gradient_can_be_captured(shape, rows, width, name):
    g = rng(rows)
    sets = [(make_ids(g, shape, rows, torch.int32, 0.05).cuda(), normal(g, (*shape, width), TYPES[name]).cuda()) for _ in range(2)]
    want = [ops.embedding_grad(grad, ids, rows) for ids, grad in sets]
    ids, grad = (torch.zeros_like(v) for v in sets[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.embedding_grad(grad, ids, rows)
    for replay in range(4):
        ids.copy_(sets[replay % 2][0])
        grad.copy_(sets[replay % 2][1])
        graph.replay()
        eager = ops.embedding_grad(*sets[1 - replay % 2][::-1], rows)
        torch.cuda.synchronize()
        assert torch.equal(out, want[replay % 2]) and torch.equal(eager, want[1 - replay % 2])
        out.zero_()


@gpu
@pytest.mark.parametrize("case", [(2, 1, 64, "bf16", "f32", 64), (1, 3000, 40, "f64", "f64", 1), (3, 700, 515, "f32", "f32", 5), (2, 900, 96, "f16", "f16", 0),
                                  (1, 9000, 70, "bf16", "bf16", 70)], ids=lambda c: "-".join(map(str, c)))
def test_recurrences_of_every_kind_of_gate_can_be_captured(case):
    b, t, d, name, gate_name, groups = case
    g = rng(t)
    sets = []
    for _ in range(2):
        x, gate, state, _ = make_scan(g, b, t, d, name, gate_name, groups, b, True, False)
        sets.append([v if v is None else v.cuda() for v in (x, gate, state, normal(g, (b, t, d), TYPES[name]))])

    def run(x, gate, state, dh):
        states, last = ops.gated_scan(x, gate, state)
        return [v for v in (states, last, *ops.gated_scan_grad(dh, states, gate, state)) if v is not None]
    want = [run(*s) for s in sets]
    still = [v if v is None else torch.zeros_like(v) for v in sets[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*still)
    for replay in range(4):
        for dst, src in zip(still, sets[replay % 2]):
            if dst is not None:
                dst.copy_(src)
        graph.replay()
        eager = run(*sets[1 - replay % 2])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[replay % 2]))
        assert all(torch.equal(p, q) for p, q in zip(eager, want[1 - replay % 2]))
        for v in out:
            v.zero_()


@gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("width", [8, 9, 11, 15, 16, 17])
def test_widths_around_a_pack(width, name):
    """Rows of a pack or two: tiles of tokens up to eight values, groups of lanes whose last pack starts earlier above."""
    g = rng(width)
    for shape, rows in (((700,), 900), ((20011,), 30000), ((9, 1300), 9000), ((3000, 7), 20000)):
        table, ids = normal(g, (rows, width), TYPES[name]), make_ids(g, shape, rows, torch.int32)
        got = ops.embedding(table.cuda(), ids.cuda(), 0.3)
        want = lookup_oracle(table, ids, 0.3)
        within(got, want, 3 * u(wide(TYPES[name])) * want.abs(), TYPES[name])
        grad = normal(g, (*shape, width), TYPES[name])
        for to, ids_to in ((grad.cuda(), ids.cuda()), (_on_gpu(grad.transpose(0, -2)), _on_gpu(ids.transpose(0, -1)))):
            got = ops.embedding_grad(to, ids_to, rows, scale=2.0, dtype=torch.float32 if name in ("bf16", "f16") else None)
            want, mag, n = lookup_grad_oracle(grad, ids, rows, 2.0)
            within(got, want, (n + 4).reshape(-1, 1) * u(wide(TYPES[name])) * mag, got.dtype)


@gpu
@pytest.mark.parametrize("name,power", [("f32", 9), ("f64", 90)])
@pytest.mark.parametrize("fade,grow", [(512, 512), (700, 400), (100, 100), (2000, 2000), (513, 1500)])
def test_a_state_that_faded_for_good_is_not_brought_back_as_another(name, power, fade, grow):
    """Gates below one, then their inverses: single steps lose the state on the way, the product of all gates may keep it.  What is
    left is nothing or the exact power of two times the state, never anything between - and nothing infinite for a state of zero."""
    w, t = TYPES[name], 4200
    gate = torch.ones((1, t, 1), dtype=w)
    gate[:, :fade], gate[:, fade:fade + grow] = 2.0**-power, 2.0**power
    gate = torch.cat([gate, gate.roll(7, 1)])
    state = torch.tensor([[1.0, -1.5, 0.0, 3.0]], dtype=w).expand(2, 4).contiguous()
    x = torch.zeros((2, t, 4), dtype=w)
    exact = torch.ldexp(state.double(), torch.tensor(power * (grow - fade)))
    _, last = ops.gated_scan(x.cuda(), gate.cuda(), state.cuda())
    _, grad_state, _ = ops.gated_scan_grad(x.cuda(), x.cuda(), gate.flip(1).cuda(), grad_last=state.cuda())
    for got in (last.cpu().double(), grad_state.cpu().double()):
        assert (got.eq(0) | got.eq(exact) | (exact.abs() > torch.finfo(w).max) & (got.abs() >= torch.finfo(w).max)).all(), got
        assert got[:, 2].eq(0).all()
