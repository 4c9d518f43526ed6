"""Edges of the step attention that its other tests leave out."""
import ctypes

import pytest
import torch

import hcp_ring_amd as H
from test_step_attn import AT, DESC, POOL, Step, check


# ---------------------------------------------------------------------------------
# a step without tokens
# ---------------------------------------------------------------------------------
@pytest.mark.parametrize("prefixes", [0, 3])
def test_an_empty_step_has_sizes_and_needs_no_workspace(hcp, prefixes):
    """0 is the answer for a bad shape, and a step of no tokens is none: its sizes are positive, and
    the call takes any workspace, or none."""
    L, d = H.lib(), H.DecodeDesc(**DESC)
    assert L.hcp_step_attn_plan_size(ctypes.byref(d), 0, prefixes) > 0
    assert L.hcp_step_attn_workspace_size(ctypes.byref(d), 0, prefixes) > 0
    shard = ctypes.byref(H.DecodeShard(AT, 3, 3, AT, 0))
    for ws, size in ((None, 0), (AT, 0), (AT, 1 << 20)):
        assert L.hcp_step_attn(ctypes.byref(d), ctypes.byref(H.PagedPool(*POOL)), 0, 1, H.View(0, 0, 0), AT, prefixes, shard, AT, 1 << 30,
                               2, H.View(0, 0, 0), None, ws, size, None) == 0, H.last_error()
    x = Step([0, 0], [3, 4], 4, 2, 64, ids=[0, -1], plens=[5]).device("cpu")
    assert H.step_attn_plan_size(x["q"], x["pool"], x["tables"], x["ptables"]) > 0
    assert H.step_attn_workspace_size(x["q"], x["pool"], x["tables"], x["ptables"]) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [False, True])
def test_an_empty_step_runs(gpu, prefix):
    """No sequence has a new token: the plan and the call of every layer still go through."""
    step = Step([0, 0, 0], [3, 40, 0], 8, 2, 64, ids=[0, -1, 0] if prefix else None, plens=[37] if prefix else ())
    out, lse = step.run()
    assert out.shape == (8, 0, 64) and lse.shape == (8, 0)
    assert H.fetch_device_errors() == 0


# ---------------------------------------------------------------------------------
# the range of scores
# ---------------------------------------------------------------------------------
RANGE = {"narrow": dict(new=[1, 1, 5], lens=[300, 33, 2000]), "cut": dict(new=[1], lens=[20000]),
         "prefix": dict(new=[1] * 40, lens=[200 + b for b in range(40)], ids=[0] * 40, plens=[3000]),
         "wide": dict(new=[1500, 700], lens=[3500, 2700])}


@pytest.mark.gpu
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("kind", RANGE)
def test_scores_of_the_largest_size(gpu, kind, sign, dtype, f32):
    """Scores of one sign, 2^19.5 in size, that rise by 5 (2^7.2 of a weight) every 128 keys, eight
    times over, and one key of each sequence 29 above all others.  Dim 0 gives the size and dim 1
    the steps: every product and sum is exact in fp32 (multiples of 4 below 2^23).

    The other keys weigh up to 20000 e^-29 < 2^-27 of a row together, and what their own weights are
    off by (parts are joined by LSEs that are rounded to 2^-5) leaves them below 2^-25.  The winner's
    weight is within 2^-19 of 1 (exponential, sums, reciprocal) and enters the product within
    eps / 2 of it (one term); the output rounds once more.  The LSE is a product of the score's fp32
    image with ln 2, joined and rounded: 8 roundings of its size."""
    kw = RANGE[kind]
    step = Step(hq=8, hkv=2, d=64, dtype=dtype, seed=31, **kw)
    step.q.zero_()
    step.q[..., 0], step.q[..., 1] = sign * 1024.0, 32.0
    k = step.pool[0]
    k[~torch.isnan(k)] = 0.0

    def keys(table, n, best):
        j = torch.arange(n)
        at = torch.from_numpy(table)[j // step.bs].long(), j % step.bs
        k1 = 1.25 * (j // 128 % 8)
        if best is not None:
            k1[best] = 16.0
        k[at[0], at[1], :, 0] = 5632.0
        k[at[0], at[1], :, 1] = k1.to(k.dtype)[:, None]
        return at

    won = torch.zeros(step.tokens, 2, 64, dtype=torch.float64)
    for b, n in enumerate(step.new):
        best = int(step.lens[b] - n)  # the last key that all new tokens see
        at = keys(step.tables[b], int(step.lens[b]), best)
        won[int(step.starts[b]): int(step.starts[b]) + int(n)] = step.pool[1, at[0][best], at[1][best]].double()
    for p, n in enumerate(step.plens):
        keys(step.ptables[p], int(n), None)
    won = won.repeat_interleave(4, 1).permute(1, 0, 2)
    out = torch.empty(8, step.tokens, 64, dtype=torch.float32, device="cuda") if f32 else None
    out, lse = step.run(out=out)
    assert H.fetch_device_errors() == 0
    got, eps = out.double().cpu(), torch.finfo(out.dtype).eps
    bound = (torch.finfo(step.q.dtype).eps / 2 + 2.0 ** -19 + eps / 2) * won.abs() + 2.0 ** -25 * 6.0
    assert bool(((got - won).abs() <= bound).all()), float(((got - won).abs() / bound).nan_to_num(1e30).max())
    want = (sign * 1024.0 * 5632.0 + 32.0 * 16.0) / 8.0  # ln of 1 + 2^-27 behind it
    assert bool(((lse.double().cpu() - want).abs() <= 8 * 2.0 ** -24 * abs(want)).all())


# ---------------------------------------------------------------------------------
# which sequences share a prefix's read
# ---------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("new,heads,shared", [
    ([32, 1, 32], (8, 2), 65),      # 128 rows at most: all three
    ([33, 1, 32], (8, 2), 33),      # 132 rows: reads the prefix for itself
    ([33, 1, 40], (8, 2), 0),       # one sequence is left, and reads it alone
    ([1, 0, 33], (8, 2), 0),
    ([1, 1, 1], (128, 1), 3), ([2, 1, 1], (128, 1), 2), ([1, 1, 1], (130, 1), 0), ([3, 1, 2], (256, 1), 0)])
def test_what_shares_a_prefix(gpu, new, heads, shared):
    """The plan's own count of the tokens behind shared prefixes (word 14 of its head), and the outputs."""
    step = Step(new, [70, 9, 90], *heads, 64, ids=[0, 0, 0], plens=[300], seed=32)
    x = step.device()
    plan = H.step_attn_plan(x["q"], x["pool"], x["tables"], x["starts"], x["lens"], x["ptables"], x["ids"], x["plens"])
    assert int(plan[:64].view(torch.int32)[14]) == shared
    check(step, *H.step_attn(x["q"], x["pool"], x["tables"], plan, x["ptables"]))


# ---------------------------------------------------------------------------------
# the bits of a softmax weight
# ---------------------------------------------------------------------------------
# Two keys a row, and scores that are one product each, exact in fp32 and in [-2, 2] (dim 0 alone, a scale
# of 1/8).  Units of 2^-24, an error of a weight relative to it: log2 e in fp32 times the distance of two
# scores, 4; the exponent's rounding (at most 8 + 7 in size: 2^-21 of a factor, times ln 2), 6; the
# exponential, 2^-22: 4.  Normalised, twice that: 28.  The sum of two weights, its reciprocal and the
# product with it, 4; two keys of up to three terms added up, 6.  38 in all, below 2^-18 of A = sum w |v|,
# beside what a weight of `terms` 16-bit terms is off by, (eps / 2)^terms, and the output's own half step.
# Nothing is joined: a unit of two keys has one step.
def _two_keys(new, dtype, out):
    """A step over two keys a sequence, V of the second the negative of the first's, so that an output of
    close weights is small beside A and its own rounding hides nothing."""
    step = Step(new, [2] * len(new), 8, 2, 64, dtype=dtype, causal=False, seed=33)
    g = torch.Generator().manual_seed(34)
    step.q.zero_()
    step.q[..., 0] = (1 + torch.rand(step.tokens, 8, generator=g)).to(step.q.dtype)
    for b in range(len(new)):
        k, v = (step.pool[p, int(step.tables[b, 0])] for p in (0, 1))
        k[:2] = 0.0
        k[:2, :, 0] = ((torch.rand(2, 2, generator=g) - 0.5) * (16 if out == "f32" else 1)).to(k.dtype)
        v[1] = -v[0]
    return step


def _weights_and_values(step):
    """(w [Hq, T, 2], v [Hq, T, 2, D]) in fp64."""
    seq = torch.repeat_interleave(torch.arange(len(step.new)), torch.from_numpy(step.new))
    k, v = (step.pool[p, torch.from_numpy(step.tables[:, 0]).long(), :2].double()[seq].repeat_interleave(4, 2).permute(2, 0, 1, 3)
            for p in (0, 1))
    return torch.softmax((step.q.double().permute(1, 0, 2)[:, :, None] * k).sum(-1) / 8, -1), v


def _bound(step, w, v, terms, out):
    half = torch.finfo(step.q.dtype).eps / 2
    o, mag = (w[..., None] * v).sum(2), (w[..., None] * v.abs()).sum(2)
    b = (2.0 ** -18 + half ** terms) * mag + torch.finfo(out).eps / 2 * o.abs()
    return o, b + (2.0 ** -25 if out == torch.float16 else 0.0)


# kind: (new tokens, terms of a weight by type of the rows and of the output)
KINDS = {"narrow": ([1, 1, 3, 5, 7, 1, 2, 32], {("bf16", "f32"): 3, ("f16", "f32"): 2, ("bf16", "same"): 2, ("f16", "same"): 2}),
         "wide": ([6000, 1, 3], {("bf16", "f32"): 3, ("f16", "f32"): 2})}
WEIGHTS = [(kind, dtype, out, terms) for kind, (_, t) in KINDS.items() for (dtype, out), terms in t.items()]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype,out,terms", WEIGHTS)
def test_bits_of_a_weight(gpu, kind, dtype, out, terms):
    step = _two_keys(KINDS[kind][0], dtype, out)
    x = step.device()
    otype = torch.float32 if out == "f32" else step.q.dtype
    plan = H.step_attn_plan(x["q"], x["pool"], x["tables"], x["starts"], x["lens"], causal=False)
    assert (int(plan[:64].view(torch.int32)[12]) > 0) == (kind == "wide")  # word 12 of a plan's head: wide tiles
    got, _ = H.step_attn(x["q"], x["pool"], x["tables"], plan, causal=False,
                         out=torch.empty(8, step.tokens, 64, dtype=otype, device="cuda"))
    o, bound = _bound(step, *_weights_and_values(step), terms, otype)
    worst = ((got.double().cpu() - o).abs() / bound).max()
    assert float(worst) <= 1.0, float(worst)
    assert H.fetch_device_errors() == 0


@pytest.mark.parametrize("kind,dtype,out,terms", WEIGHTS)
def test_a_term_less_would_be_seen(kind, dtype, out, terms):
    """The oracle with weights of one term less is outside the bound, with all of them within."""
    step = _two_keys(KINDS[kind][0], dtype, out)
    otype = torch.float32 if out == "f32" else step.q.dtype
    w, v = _weights_and_values(step)
    o, bound = _bound(step, w, v, terms, otype)
    for n, seen in ((terms, False), (terms - 1, True)):
        kept, rest = torch.zeros_like(w), (w * 100).float().double()  # as beside a maximum taken elsewhere
        for _ in range(n):
            t = rest.to(step.q.dtype).double()
            kept, rest = kept + t, rest - t
        got = ((kept / 100)[..., None] * v).sum(2).to(otype).double()
        assert bool(((got - o).abs() > bound).any()) == seen, n


# ---------------------------------------------------------------------------------
# the same step, the same bits
# ---------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kw", [
    dict(new=[1], lens=[30000]), dict(new=[1] * 50 + [5] * 9, lens=[300 + 17 * b for b in range(59)], ids=[0] * 40 + [1] * 19, plens=[4000, 333]),
    dict(new=[1] * 9 + [2000, 1100], lens=[900 + 300 * b for b in range(9)] + [3000, 1100], ids=[0] * 5 + [-1] * 5 + [0], plens=[700])])
def test_the_same_step_gives_the_same_bits(gpu, kw, dtype, f32):
    """Cut units and shared prefixes, by the same plan and by others of the same lengths, whatever the
    workspace, the plan's memory and the outputs held before."""
    step = Step(hq=8, hkv=2, d=128, dtype=dtype, seed=35, **kw)
    x = step.device()
    out = torch.empty(8, step.tokens, 128, dtype=torch.float32 if f32 else step.q.dtype, device="cuda")
    lse = torch.empty(8, step.tokens, device="cuda")
    ws = torch.empty(H.step_attn_workspace_size(x["q"], x["pool"], x["tables"], x["ptables"]), dtype=torch.uint8, device="cuda")
    plan = torch.empty(H.step_attn_plan_size(x["q"], x["pool"], x["tables"], x["ptables"]), dtype=torch.uint8, device="cuda")
    first = None
    for i, fill in enumerate((0, 255, 0x3f, 255)):
        for t in (ws, out.view(torch.uint8), lse.view(torch.uint8)):
            t.fill_(fill)
        if i % 2 == 0:
            plan.fill_(fill)
            H.step_attn_plan(x["q"], x["pool"], x["tables"], x["starts"], x["lens"], x["ptables"], x["ids"], x["plens"], plan=plan)
        H.step_attn(x["q"], x["pool"], x["tables"], plan, x["ptables"], out=out, lse=lse, workspace=ws)
        got = out.clone(), lse.clone()
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first)), i
    check(step, *first, terms=2 if f32 else 1)
