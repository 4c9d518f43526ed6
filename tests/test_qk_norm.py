"""Norms of q and k heads with the position rotation, dense and into the paged cache, against
the formulas in 64 bits.

Bound of an element: the sum of squares adds up to 2 * 8 + 6 terms in a chain (22 roundings of
2^-24, half of them after the root), the reciprocal root is within 2 ulp (4 * 2^-24), scaling
the mean, eps and the two products round 5 times: 20 * 2^-24 in all, below 2^-19 of the normed
value; turning a plane adds 2 * 2^-24 of |y_i| + |y_j|.  With the store's half step:
eps(t) / 2 * |ref| + 2^-19 (|y_i| + |y_j|), and half the smallest step of fp16."""
import ctypes

import pytest
import torch

import hcp_ring_amd as H

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def reference(x, w, cos, sin, rot, pairs, eps):
    """(rows in fp64, |y_i| + |y_j| of every element) of x [H, T, D]."""
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double()
    z, mag = y.clone(), y.abs()
    if rot:
        p = torch.arange(rot // 2)
        i, j = (2 * p, 2 * p + 1) if pairs else (p, p + rot // 2)
        z[..., i] = y[..., i] * cos - y[..., j] * sin
        z[..., j] = y[..., j] * cos + y[..., i] * sin
        mag[..., i] = mag[..., j] = y[..., i].abs() + y[..., j].abs()
    return z, mag


def check(got, ref, mag, dtype):
    bound = torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -19 * mag + (2.0 ** -25 if dtype == torch.float16 else 0)
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-300)).max())


def angles(rot, rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(rows, rot // 2, generator=g, dtype=torch.float64) * 6.28
    return torch.stack([torch.cos(a), torch.sin(a)]).float()


def inputs(seed, hq, hkv, t, d, dtype, rot, rows=77):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, hq + 2 * hkv, d, generator=g) * 3
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)]
    pos = torch.randint(0, rows, (t,), generator=g)
    return x.to(dtype), w, pos, (angles(rot, rows, seed) if rot else None)


SHAPES = [  # hq, hkv, tokens, d, rot
    (32, 8, 1, 128, 128), (16, 2, 67, 128, 128), (14, 2, 33, 64, 64), (8, 1, 19, 96, 48), (3, 3, 5, 256, 256),
    (5, 1, 7, 72, 40), (1, 1, 3, 8, 8), (7, 7, 2, 40, 0), (9, 3, 11, 128, 32), (2, 1, 4, 24, 8), (40, 8, 130, 80, 80),
]


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_dense_matches_the_formula(gpu, shape, dt, pairs):
    hq, hkv, t, d, rot = shape
    dtype = DTYPES[dt]
    x, w, pos, tab = inputs(1, hq, hkv, t, d, dtype, rot)
    dev = x.cuda()
    q, k = dev[:, :hq].permute(1, 0, 2), dev[:, hq: hq + hkv].permute(1, 0, 2)
    qo, ko = H.qk_norm_rope(q, k, w[0].cuda(), w[1].cuda(), pos.cuda(), None if tab is None else tab.cuda(), eps=1e-5, pairs=pairs)
    cos, sin = (tab[0][pos].double(), tab[1][pos].double()) if rot else (None, None)
    for got, src, wt in ((qo, x[:, :hq], w[0]), (ko, x[:, hq: hq + hkv], w[1])):
        check(got, *reference(src.permute(1, 0, 2), wt, cos, sin, rot, pairs, 1e-5), dtype)
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("off", [1, 2, 4])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_views_of_any_alignment_and_outputs_that_are_inputs(gpu, dt, off):
    """Rows that start `off` elements behind a 16-byte boundary, head-major and token-major
    views, and q / k normed in place: the same bits as aligned copies give."""
    hq, hkv, t, d = 6, 2, 13, 128
    dtype = DTYPES[dt]
    x, w, pos, tab = inputs(2, hq, hkv, t, d, dtype, d)
    wq, wk, pos, tab = w[0].cuda(), w[1].cuda(), pos.cuda(), tab.cuda()
    q, k = x[:, :hq].permute(1, 0, 2).contiguous().cuda(), x[:, hq: hq + hkv].permute(1, 0, 2).contiguous().cuda()
    want = H.qk_norm_rope(q, k, wq, wk, pos, tab)

    def shifted(a):  # [H, T, D] with rows D + 3 apart, `off` elements into an allocation
        h = a.shape[0]
        flat = torch.full((off + h * t * (d + 3),), 7.0, dtype=dtype, device="cuda")
        v = flat[off:].view(h, t, d + 3)[..., :d]
        v.copy_(a)
        return flat, v
    fq, vq = shifted(q)
    fk, vk = shifted(k)
    got = H.qk_norm_rope(vq, vk, wq, wk, pos, tab)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    H.qk_norm_rope(vq, vk, wq, wk, pos, tab, q_out=vq, k_out=vk)
    assert torch.equal(vq, want[0]) and torch.equal(vk, want[1])
    for f, v in ((fq, vq), (fk, vk)):  # what lies between the rows stays
        v.fill_(7.0)
        assert bool((f == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(32, 8, 128, 128, 16), (14, 2, 64, 64, 32), (8, 1, 96, 48, 7), (3, 1, 256, 256, 16)])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_append_writes_its_slots_alone(gpu, shape, dt):
    hq, hkv, d, rot, bs = shape
    t, nb, dtype = 29, 11, DTYPES[dt]
    x, w, pos, tab = inputs(3, hq, hkv, t, d, dtype, rot)
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(4))[:t]
    slots[[0, 5]] = -1
    pool = torch.randn(2, nb, bs, hkv, d, generator=torch.Generator().manual_seed(5)).to(dtype)
    dev, dpool = x.cuda(), pool.cuda()
    q, k, v = (dev[:, a:b].permute(1, 0, 2) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    qo = H.qk_norm_rope_append(q, k, v, w[0].cuda(), w[1].cuda(), dpool, slots.cuda(), pos.cuda(), tab.cuda())
    dense, ko = H.qk_norm_rope(q, k, w[0].cuda(), w[1].cuda(), pos.cuda(), tab.cuda())
    assert torch.equal(qo, dense)
    want = pool.view(2, nb * bs, hkv, d).clone()
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            want[0, s], want[1, s] = ko[:, i].cpu(), x[i, hq + hkv:]
    assert torch.equal(dpool.cpu().view_as(want), want)  # V rows and all other slots bit for bit
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
def test_no_weights_and_no_rotation(gpu):
    x, _, _, _ = inputs(6, 4, 2, 9, 64, torch.float32, 0)
    q, k = x[:, :4].permute(1, 0, 2), x[:, 4:6].permute(1, 0, 2)
    qo, ko = H.qk_norm_rope(q.cuda(), k.cuda())
    check(qo, *reference(q, None, None, None, 0, False, 1e-6), torch.float32)
    check(ko, *reference(k, None, None, None, 0, False, 1e-6), torch.float32)


@pytest.mark.gpu
def test_rows_that_are_not_finite_or_zero_keep_to_themselves(gpu):
    x, w, pos, tab = inputs(7, 4, 2, 9, 128, torch.bfloat16, 128)
    q, k = x[:, :4].permute(1, 0, 2).contiguous().cuda(), x[:, 4:6].permute(1, 0, 2).contiguous().cuda()
    args = (w[0].cuda(), w[1].cuda(), pos.cuda(), tab.cuda())
    want = H.qk_norm_rope(q, k, *args)[0]
    q2 = q.clone()
    q2[1, 3, 5], q2[2, 4, 100], q2[0, 0] = float("nan"), float("inf"), 0.0
    got = H.qk_norm_rope(q2, k, *args)[0]
    assert bool(got[1, 3].isnan().all()) and bool((got[0, 0] == 0).all()) and bool(got[2, 4, 100].isnan())
    same = torch.ones(4, 9, dtype=torch.bool)
    same[1, 3] = same[2, 4] = same[0, 0] = False
    assert torch.equal(got[same.cuda()], want[same.cuda()])


@pytest.mark.gpu
def test_bad_positions_and_slots_set_their_flags(gpu):
    x, w, pos, tab = inputs(8, 4, 2, 6, 64, torch.bfloat16, 64)
    pos[1], pos[4] = -1, tab.shape[1]
    pool = torch.zeros(2, 2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.tensor([0, 1, 32, 3, 2 ** 40, -5]).cuda()
    dev = x.cuda()
    q, k, v = (dev[:, a:b].permute(1, 0, 2) for a, b in ((0, 4), (4, 6), (6, 8)))
    qo = H.qk_norm_rope_append(q, k, v, w[0].cuda(), w[1].cuda(), pool, slots, pos.cuda(), tab.cuda())
    assert H.fetch_device_errors() == 5
    ref, mag = reference(x[:, :4].permute(1, 0, 2), w[0], None, None, 0, False, 1e-6)
    check(qo[:, [1, 4]], ref[:, [1, 4]], mag[:, [1, 4]], torch.bfloat16)  # normed, not turned
    written = pool.view(2, 32, -1).abs().amax((0, 2)) > 0
    assert written.nonzero().flatten().tolist() == [0, 1, 3]


@pytest.mark.gpu
def test_another_stream_and_many_tokens(gpu):
    """On a stream of its own, and with more tokens than one grid of workgroups takes."""
    t = 70000
    x, w, pos, tab = inputs(9, 1, 1, t, 64, torch.float16, 64, rows=1000)
    s = torch.cuda.Stream()
    q, k = x[:, :1].permute(1, 0, 2), x[:, 1:2].permute(1, 0, 2)
    with torch.cuda.stream(s):
        args = [a.cuda() for a in (q, k, w[0], w[1], pos, tab)]
        qo, ko = H.qk_norm_rope(*args)
    s.synchronize()
    cos, sin = tab[0][pos].double(), tab[1][pos].double()
    check(qo, *reference(q, w[0], cos, sin, 64, False, 1e-6), torch.float16)
    check(ko, *reference(k, w[1], cos, sin, 64, False, 1e-6), torch.float16)


BASE = dict(dtype=2, num_q_heads=4, num_kv_heads=2, head_dim=64, rope=1, tokens=3, rope_rows=10)


def _raw(pool=None, null=False, rope_dims=64, eps=1e-6, q=1 << 20, table=1 << 20, w=1 << 20, slots=1 << 20, q_out=1 << 20, **kw):
    """Both entries with addresses that are never read: a call that is not refused would need a GPU."""
    v = lambda p: H.View(p, 64, 256)  # noqa: E731
    d = None if null else ctypes.byref(H.QkvDesc(**dict(BASE, **kw)))
    L, at = H.lib(), 1 << 20
    if pool is None:
        return L.hcp_qk_norm_rope(d, rope_dims, eps, v(q), v(at), w, w, at, table, v(q_out), v(at), None)
    return L.hcp_qk_norm_rope_append(d, rope_dims, eps, v(q), v(at), v(at), w, w, at, table, v(q_out),
                                     ctypes.byref(H.PagedPool(*pool)), slots, None)


POOL = (1 << 20, 4, 16, 2, 64, 2)


@pytest.mark.parametrize("kw", [dict(dtype=4), dict(num_q_heads=0), dict(num_kv_heads=-1), dict(head_dim=60), dict(head_dim=264),
                                dict(rope_dims=72), dict(rope_dims=-8), dict(rope_dims=12), dict(rope_dims=0), dict(rope=3),
                                dict(rope=-1), dict(tokens=-1), dict(tokens=1 << 31), dict(rope_rows=0), dict(eps=0.0),
                                dict(eps=float("nan")), dict(eps=float("inf")), dict(num_q_heads=1 << 21)])
def test_bad_descriptors_are_refused(hcp, kw):
    assert _raw(**kw) == -6
    assert _raw(POOL, **kw) == -6


def test_bad_pointers_and_pools_are_refused(hcp):
    assert _raw(null=True) == -6 and _raw(POOL, null=True) == -6
    assert _raw(q=0) == -6 and _raw(q=(1 << 20) + 1) == -6 and _raw(q_out=0) == -6
    assert _raw(table=None) == -6 and _raw(table=(1 << 20) + 2) == -6 and _raw(w=(1 << 20) + 1) == -6
    for i, bad in ((0, 0), (0, (1 << 20) + 1), (1, 0), (2, 0), (3, 1), (4, 128), (5, 4), (5, 1)):
        pool = list(POOL)
        pool[i] = bad
        assert _raw(pool) == -6, (i, bad)
    assert _raw(POOL, slots=None) == -6
    assert _raw(tokens=0) == 0 and _raw(POOL, tokens=0) == 0  # nothing to do


def test_bindings_refuse_what_does_not_fit(hcp):
    q, k, w = torch.zeros(4, 3, 64), torch.zeros(2, 3, 64), torch.ones(64)
    pos, tab = torch.zeros(3, dtype=torch.int64), torch.zeros(2, 5, 32)
    for args in ((q, k[:, :2], w, w, pos, tab), (q, k.half(), w, w, pos, tab), (q, k, w[:32], w, pos, tab),
                 (q, k, w.half(), w, pos, tab), (q, k, w, w, None, tab), (q, k, w, w, pos.int(), tab),
                 (q, k, w, w, pos, tab[0]), (q, k, w, w, pos, tab.double()), (q, k, w, w, pos, tab)):
        with pytest.raises(ValueError):  # the last: tensors on the CPU
            H.qk_norm_rope(*args)
    pool, slots = torch.zeros(2, 1, 16, 2, 64), torch.zeros(3, dtype=torch.int64)
    for p, s, v in ((pool.half(), slots, k), (pool, slots.int(), k), (pool, slots[:2], k), (pool, slots, k[:1]), (pool, slots, k)):
        with pytest.raises(ValueError):
            H.qk_norm_rope_append(q, k, v, w, w, p, s, pos, tab)
