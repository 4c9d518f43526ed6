"""Norms of q and k heads over enough rows that a wave takes several runs of them, and more tokens
than one grid of waves takes.

The launcher gives a wave floor(tokens * runs / 8192) runs of rows of a token, a run being the rows
that 64 lanes hold at once: `runs_of` and `groups` restate it, so that every case says what it is
there for.  Each is compared with the formula in 64 bits (the bound of test_qk_norm) and bit by bit
with calls on few tokens at a time, whose waves take one run each."""
import pytest
import torch

import hcp_ring_amd as H
from test_qk_norm import DTYPES, check, inputs, reference

RESIDENT = 256 * 32  # waves that the GPU holds


def runs_of(rows, d, rot, dtype):
    """Passes of a wave over a token's rows."""
    c = 8 if dtype.itemsize == 2 and d % 16 == 0 and rot % 16 == 0 else 4
    lanes = 1
    while lanes * 2 * c < d:
        lanes *= 2
    return -(-rows // (64 // lanes))


def groups(rows, d, rot, dtype, tokens):
    runs = runs_of(rows, d, rot, dtype)
    return max(1, min(runs, tokens * runs // RESIDENT))


def device_inputs(seed, hq, hkv, t, d, dtype, rot):
    x, w, pos, tab = inputs(seed, hq, hkv, t, d, dtype, rot)
    return x.cuda(), w[0].cuda(), w[1].cuda(), pos.cuda(), None if tab is None else tab.cuda()


def parts(x, hq, hkv):
    return (x[:, a:b].permute(1, 0, 2) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))


# hq, hkv, d, rot, type, tokens, runs of a wave in the dense form, runs of a token
CASES = [
    (32, 8, 128, 128, "bf16", 3500, 2, 5),   # the last of three waves of a token has one run
    (32, 8, 128, 64, "f16", 5000, 3, 5),     # and here of two, two
    (32, 8, 128, 128, "bf16", 8300, 5, 5),   # one wave a token
    (7, 2, 128, 128, "f32", 6000, 2, 3),     # a run of one row behind whole ones
    (6, 3, 256, 32, "f32", 3500, 2, 5),
    (9, 4, 72, 40, "bf16", 6500, 3, 4),      # chunks of four, 9 of 16 lanes in use, a last run of one row
    (14, 5, 64, 0, "f16", 9000, 2, 2),       # no rotation
]


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_waves_of_several_runs(gpu, case, pairs):
    """Dense, out of place, in place, and on rows that no wide load fits."""
    hq, hkv, d, rot, dt, t, per_wave, runs = case
    dtype = DTYPES[dt]
    assert runs_of(hq + hkv, d, rot, dtype) == runs and groups(hq + hkv, d, rot, dtype, t) == per_wave > 1
    x, wq, wk, pos, tab = device_inputs(41, hq, hkv, t, d, dtype, rot)
    q, k, _ = parts(x, hq, hkv)
    qo, ko = H.qk_norm_rope(q, k, wq, wk, pos, tab, pairs=pairs)
    for a in range(0, t, 500):  # one run a wave
        b = min(a + 500, t)
        assert groups(hq + hkv, d, rot, dtype, b - a) == 1
        some = H.qk_norm_rope(q[:, a:b], k[:, a:b], wq, wk, pos[a:b], tab, pairs=pairs)
        assert torch.equal(some[0], qo[:, a:b]) and torch.equal(some[1], ko[:, a:b]), a
    cos, sin = (tab[0][pos].double(), tab[1][pos].double()) if rot else (None, None)
    for got, src, w in ((qo, q, wq), (ko, k, wk)):
        ref, mag = reference(src, w, cos, sin, rot, pairs, 1e-6)
        check(got, ref.cpu(), mag.cpu(), dtype)
    odd = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(x).copy_(x)
    oq, ok, _ = parts(odd, hq, hkv)
    for u, v in ((oq, ok), (q, k)):  # in place: the next run's rows are read before this one's are written
        rest = (odd if u is oq else x)[:, hq + hkv:].clone()
        H.qk_norm_rope(u, v, wq, wk, pos, tab, pairs=pairs, q_out=u, k_out=v)
        assert torch.equal(u, qo) and torch.equal(v, ko)
        assert torch.equal((odd if u is oq else x)[:, hq + hkv:], rest)
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("case", [(32, 8, 128, 128, "bf16", 3500, 2, 6), (32, 8, 128, 128, "bf16", 7000, 5, 6),
                                  (32, 8, 128, 64, "f16", 12000, 6, 6), (14, 2, 64, 64, "bf16", 9000, 2, 2),
                                  (5, 3, 128, 128, "f32", 6000, 2, 3), (3, 2, 256, 256, "f32", 5000, 2, 4)])
def test_appends_of_several_runs(gpu, case, pairs):
    """q, k and v rows change from run to run of a wave, and within one; some tokens have no slot."""
    hq, hkv, d, rot, dt, t, per_wave, runs = case
    dtype, bs = DTYPES[dt], 16
    assert runs_of(hq + 2 * hkv, d, rot, dtype) == runs and groups(hq + 2 * hkv, d, rot, dtype, t) == per_wave > 1
    x, wq, wk, pos, tab = device_inputs(42, hq, hkv, t, d, dtype, rot)
    q, k, v = parts(x, hq, hkv)
    nb = t // bs + 3
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(43))[:t].cuda()
    slots[::17] = -1
    pool = torch.randn(2, nb, bs, hkv, d, generator=torch.Generator().manual_seed(44)).to(dtype).cuda()
    want = pool.clone().view(2, nb * bs, hkv, d)
    dense, ko = H.qk_norm_rope(q, k, wq, wk, pos, tab, pairs=pairs)
    held = slots >= 0
    want[0, slots[held]], want[1, slots[held]] = ko.permute(1, 0, 2)[held], v.permute(1, 0, 2)[held]
    qo = H.qk_norm_rope_append(q, k, v, wq, wk, pool, slots, pos, tab, pairs=pairs)
    assert torch.equal(qo, dense) and torch.equal(pool.view_as(want), want)
    cos, sin = tab[0][pos].double(), tab[1][pos].double()
    for got, src, w in ((qo, q, wq), (ko, k, wk)):
        ref, mag = reference(src, w, cos, sin, rot, pairs, 1e-6)
        check(got, ref.cpu(), mag.cpu(), dtype)
    H.qk_norm_rope_append(q, k, v, wq, wk, pool, slots, pos, tab, pairs=pairs, q_out=q)
    assert torch.equal(q, dense) and torch.equal(pool.view_as(want), want)
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
def test_more_tokens_than_one_grid_takes(gpu):
    """2^20 workgroups of four waves take 4 194 304 tokens of one run: the waves of the first go on to the rest."""
    t, d = (4 << 20) + 70001, 8
    assert runs_of(2, d, d, torch.bfloat16) == 1 and t > 4 << 20
    g = torch.Generator(device="cuda").manual_seed(45)
    x = torch.randn(t, 3, d, generator=g, device="cuda").bfloat16()
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g, device="cuda")).bfloat16()
    pos = torch.randint(0, 99, (t,), generator=g, device="cuda")
    tab = H.rope_table(d, 99)
    q, k, v = parts(x, 1, 1)
    slots = torch.randperm(t, generator=g, device="cuda")
    pool = torch.zeros(2, -(-t // 16), 16, 1, d, dtype=torch.bfloat16, device="cuda")
    qo, ko = H.qk_norm_rope(q, k, wq, wk, pos, tab)
    qa = H.qk_norm_rope_append(q, k, v, wq, wk, pool, slots, pos, tab)
    rows = pool.view(2, -1, 1, d)
    assert torch.equal(qa, qo) and torch.equal(rows[0, slots], ko.permute(1, 0, 2)) and torch.equal(rows[1, slots], v.permute(1, 0, 2))
    cos, sin = tab[0][pos].double(), tab[1][pos].double()
    for got, src, w in ((qo, q, wq), (ko, k, wk)):
        ref, mag = reference(src, w, cos, sin, d, False, 1e-6)
        check(got, ref.cpu(), mag.cpu(), torch.bfloat16)
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
def test_no_tokens(gpu):
    """Steps without tokens come through the bindings too."""
    x, wq, wk, pos, tab = device_inputs(46, 4, 2, 0, 64, torch.bfloat16, 64)
    q, k, v = parts(x, 4, 2)
    pool = torch.ones(2, 2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    qo, ko = H.qk_norm_rope(q, k, wq, wk, pos, tab)
    qa = H.qk_norm_rope_append(q, k, v, wq, wk, pool, pos, pos, tab)
    assert qo.shape == qa.shape == (4, 0, 64) and ko.shape == (2, 0, 64)
    assert bool((pool == 1).all()) and H.fetch_device_errors() == 0
