"""Append to and gather from the 8-bit paged cache, and the prefill over it, against a plain
restatement in 64 bits (kv8_reference).  Codes and scales are whole numbers of a kind and
have to be equal; a gathered row is one rounding of scale * code."""
import ctypes
import math

import numpy as np
import pytest
import torch

import hcp_ring_amd as H
import kv8_reference as R

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def test_reference_formats_known_answers():
    # the e4m3 table against torch's own type, every code; rounding against torch's conversion
    c = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(c).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(R.E4M3, want, equal_nan=True)
    x = np.random.default_rng(0).normal(size=20000) * np.exp(np.random.default_rng(1).uniform(-8, 5, 20000))
    x = np.clip(np.float32(x), -448, 448).astype(np.float64)
    assert np.array_equal(R.encode(x, "e4m3"), torch.from_numpy(np.float32(x)).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    mid = (R.E4M3[:126] + R.E4M3[1:127]) / 2  # ties
    assert np.array_equal(R.encode(mid, "e4m3"), torch.from_numpy(np.float32(mid)).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert R.power_scale(448.0, "e4m3") == 1.0 and R.power_scale(448.1, "e4m3") == 2.0
    assert R.power_scale(127.0, "int8") == 1.0 and R.power_scale(0.0, "int8") == 2.0 ** -100


def _values(r, shape, dtype, size=1.0):
    """Values of the type, and the same in fp64."""
    t = torch.from_numpy(r.normal(size=shape) * size).to(DT[dtype])
    return t, t.double().numpy()


APPEND = [
    # seed, block size, kv heads, head dim, dtype, format, runs: (place, tokens) per block, in order
    (1, 16, 8, 128, "bf16", "e4m3", [(0, 16), (0, 5), (7, 1), (3, 13)]),
    (2, 16, 2, 64, "f16", "int8", [(15, 1), (0, 1), (1, 15), (0, 16)]),
    (3, 32, 1, 96, "f32", "e4m3", [(31, 1), (5, 20)]),
    (4, 128, 3, 128, "bf16", "int8", [(0, 128), (100, 28), (1, 127)]),
    (5, 48, 2, 8, "f16", "e4m3", [(0, 48), (47, 1)]),
    (6, 1, 2, 128, "bf16", "e4m3", [(0, 1), (0, 1), (0, 1)]),
    (7, 16, 4, 256, "f32", "int8", [(2, 3), (0, 16)]),
    (8, 200, 2, 72, "bf16", "int8", [(0, 200), (199, 1), (60, 100)]),
    (9, 16, 5, 120, "f16", "int8", [(0, 16)] * 40 + [(9, 3)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["token_major", "head_major", "odd_strides"])
@pytest.mark.parametrize("case", APPEND, ids=[str(c[0]) for c in APPEND])
def test_append_matches_the_host(gpu, case, layout):
    seed, bs, heads, d, dtype, fmt, runs = case
    r = np.random.default_rng(seed)
    nb = len(runs) + 2
    codes, scales = R.random_cache(r, nb, bs, heads, d, fmt)
    blocks = r.permutation(nb)[: len(runs)]
    slots = np.concatenate([b * bs + a + np.arange(n) for b, (a, n) in zip(blocks, runs)])
    t = len(slots)
    size = np.repeat(np.exp(r.uniform(-6, 6, len(runs))), [n for _, n in runs])  # scales that grow, and that do not
    kt, k = _values(r, (heads, t, d), dtype, size[None, :, None])
    vt, v = _values(r, (heads, t, d), dtype, size[None, :, None])
    if layout == "token_major":
        dev = [x.permute(1, 0, 2).contiguous().cuda().permute(1, 0, 2) for x in (kt, vt)]
    elif layout == "head_major":
        dev = [x.cuda() for x in (kt, vt)]
    else:  # rows that start on odd elements
        dev = [torch.nn.functional.pad(x, (1, 2)).cuda()[:, :, 1: d + 1] for x in (kt, vt)]
    pool, sc = R.to_device(codes, scales, fmt)
    H.fetch_device_errors()
    H.kv8_append(pool, sc, *dev, torch.from_numpy(slots).cuda())
    R.append(codes, scales, k, v, slots, fmt)
    got_codes, got_scales = R.to_host(pool, sc)
    assert np.array_equal(got_scales, scales)
    assert np.array_equal(got_codes, codes)
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_token_by_token(gpu, fmt):
    # a block filled one token at a time, magnitudes growing: every step equals the host's
    r = np.random.default_rng(11)
    bs, heads, d = 16, 3, 64
    codes, scales = R.random_cache(r, 4, bs, heads, d, fmt)
    pool, sc = R.to_device(codes, scales, fmt)
    for t in range(2 * bs):
        kt, k = _values(r, (heads, 1, d), "bf16", 1.3 ** t)
        vt, v = _values(r, (heads, 1, d), "bf16", 1.3 ** -t)
        slots = np.array([bs * (1 + t // bs) + t % bs])
        H.kv8_append(pool, sc, kt.cuda(), vt.cuda(), torch.from_numpy(slots).cuda())
        R.append(codes, scales, k, v, slots, fmt)
        got_codes, got_scales = R.to_host(pool, sc)
        assert np.array_equal(got_scales, scales) and np.array_equal(got_codes, codes), t


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_extreme_values(gpu, fmt):
    # zeros, the type's largest and smallest values, values at the format's limit, ties
    top = R.LARGEST[fmt]
    rows = [np.zeros(64), np.full(64, 3.0e38), np.full(64, 1e-44), np.linspace(-top, top, 64),
            np.concatenate([[top * 1.001], np.linspace(-1, 1, 63)]), np.concatenate([[top], np.arange(63) + 0.5]),
            np.concatenate([[top], 2.0 ** -np.arange(63.0)]), np.full(64, 2.0 ** -110), np.full(64, -0.0)]
    k = torch.tensor(np.array(rows), dtype=torch.float32)[None]  # one token a row, a block each
    slots = np.arange(len(rows)) * 16
    codes, scales = np.full((2, len(rows), 16, 1, 64), 9, np.uint8), np.full((2, len(rows), 1), 5.0, np.float32)
    pool, sc = R.to_device(codes, scales, fmt)
    H.kv8_append(pool, sc, k.cuda(), -k.cuda(), torch.from_numpy(slots).cuda())
    R.append(codes, scales, k.double().numpy(), -k.double().numpy(), slots, fmt)
    got_codes, got_scales = R.to_host(pool, sc)
    assert np.array_equal(got_scales, scales)
    assert np.array_equal(R.values(got_codes, fmt), R.values(codes, fmt))  # -0 is 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_append_value_that_is_not_finite(gpu, fmt, bad):
    # the scale of that block, plane and head is NaN and stays so until a run from place 0
    r = np.random.default_rng(12)
    codes, scales = R.random_cache(r, 3, 16, 2, 64, fmt)
    pool, sc = R.to_device(codes, scales, fmt)
    kt, k = _values(r, (2, 2, 64), "bf16")
    vt, v = _values(r, (2, 2, 64), "bf16")
    kt[1, 1, 5] = bad
    k[1, 1, 5] = bad
    for slots, kk, kr in (([20, 21], kt, k), ([22, 23], vt, v), ([16, 17], vt, v)):
        H.kv8_append(pool, sc, kk.cuda(), vt.cuda(), torch.tensor(slots).cuda())
        R.append(codes, scales, kr, v, slots, fmt)
        got_codes, got_scales = R.to_host(pool, sc)
        assert np.array_equal(got_scales, scales, equal_nan=True) and np.array_equal(got_codes, codes)
    assert not np.isnan(scales).any()


@pytest.mark.gpu
def test_append_skips_padding_and_flags_bad_slots(gpu):
    r = np.random.default_rng(13)
    codes, scales = R.random_cache(r, 3, 16, 2, 64, "e4m3")
    pool, sc = R.to_device(codes, scales, "e4m3")
    kt, k = _values(r, (2, 9, 64), "bf16")
    slots = np.array([-1, 33, 34, -1, -1, 48, 1 << 40, -7, 3])  # 48 is the first place past the pool
    H.fetch_device_errors()
    H.kv8_append(pool, sc, kt.cuda(), kt.cuda(), torch.from_numpy(slots).cuda())
    got_codes, got_scales = R.to_host(pool, sc)
    assert H.fetch_device_errors() == 1
    assert np.array_equal(got_codes[:, 1], codes[:, 1]) and np.array_equal(got_scales[:, 1], scales[:, 1])
    R.append(codes, scales, k, k, slots, "e4m3")
    assert np.array_equal(got_codes, codes) and np.array_equal(got_scales, scales)
    H.kv8_append(pool, sc, kt[:, :0].cuda(), kt[:, :0].cuda(), torch.zeros(0, dtype=torch.int64, device="cuda"))


GATHER = [
    # seed, block size, kv heads, head dim, out dtype, format, table offset, t0, t1
    (1, 16, 8, 128, "bf16", "e4m3", 0, 0, 77),
    (2, 16, 2, 64, "f16", "int8", 5, 9, 10),
    (3, 32, 1, 96, "f32", "e4m3", 3, 40, 300),
    (4, 128, 3, 128, "bf16", "int8", 0, 127, 129),
    (5, 48, 2, 8, "f16", "e4m3", 0, 0, 48),
    (6, 1, 2, 256, "f32", "int8", 0, 2, 9),
    (7, 16, 5, 72, "bf16", "e4m3", 0, 16, 1000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["head_major", "token_major", "odd_strides"])
@pytest.mark.parametrize("case", GATHER, ids=[str(c[0]) for c in GATHER])
def test_gather_matches_the_host(gpu, case, layout):
    seed, bs, heads, d, dtype, fmt, off, t0, t1 = case
    r = np.random.default_rng(seed)
    nb = -(-(t1 - off) // bs) + 2
    codes, scales = R.random_cache(r, nb, bs, heads, d, fmt)
    scales *= r.uniform(0.5, 1.0, scales.shape).astype(np.float32)  # any scale, not only powers of two
    table = r.permutation(nb).astype(np.int32)
    pool, sc = R.to_device(codes, scales, fmt)
    n = t1 - t0
    if layout == "head_major":
        out = [torch.empty(heads, n, d, dtype=DT[dtype], device="cuda") for _ in range(2)]
    elif layout == "token_major":
        out = [torch.empty(n, heads, d, dtype=DT[dtype], device="cuda").permute(1, 0, 2) for _ in range(2)]
    else:
        out = [torch.empty(heads, n, d + 3, dtype=DT[dtype], device="cuda")[:, :, 1: d + 1] for _ in range(2)]
    H.kv8_gather(pool, sc, torch.from_numpy(table).cuda(), off, t0, t1, k_out=out[0], v_out=out[1])
    for plane in range(2):
        # the product of an 8-bit code and an fp32 scale, rounded to fp32 and then to the type: half a step each
        want = R.rows(codes, scales, table, fmt, plane, t0, t1, off)
        got = out[plane].double().cpu().numpy()
        step = 2.0 ** -24 + (0 if dtype == "f32" else torch.finfo(DT[dtype]).eps / 2)
        floor = {"bf16": 0.0, "f16": 2.0 ** -25, "f32": 0.0}[dtype]  # half of fp16's smallest step
        assert (np.abs(got - want) <= np.abs(want) * step * (1 + 2.0 ** -20) + floor).all()
        assert dtype != "f32" or np.array_equal(got, np.float32(want).astype(np.float64))


@pytest.mark.gpu
def test_gather_exact_for_powers_of_two_and_default_outputs(gpu):
    r = np.random.default_rng(20)
    for fmt in ("e4m3", "int8"):
        codes, scales = R.random_cache(r, 5, 16, 2, 64, fmt)
        pool, sc = R.to_device(codes, scales, fmt)
        table = np.array([3, 0, 4], np.int32)
        k, v = H.kv8_gather(pool, sc, torch.from_numpy(table).cuda(), 0, 3, 40)
        assert k.dtype == torch.bfloat16
        for plane, got in enumerate((k, v)):
            assert np.array_equal(got.double().cpu().numpy(), R.rows(codes, scales, table, fmt, plane, 3, 40))


@pytest.mark.gpu
def test_gather_skips_bad_blocks(gpu):
    r = np.random.default_rng(21)
    codes, scales = R.random_cache(r, 3, 16, 2, 64, "int8")
    pool, sc = R.to_device(codes, scales, "int8")
    k = torch.full((2, 40, 64), 7.0, dtype=torch.float16, device="cuda")
    v = k.clone()
    H.fetch_device_errors()
    H.kv8_gather(pool, sc, torch.tensor([2, 3, -1], dtype=torch.int32).cuda(), 0, 0, 40, k_out=k, v_out=v)
    assert H.fetch_device_errors() == 1
    assert (k[:, 16:] == 7).all() and (v[:, 16:] == 7).all()
    assert np.array_equal(k[:, :16].double().cpu().numpy(), R.rows(codes, scales, [2], "int8", 0, 0, 16))


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    # chunks, Hq, Hkv, D, block size, format, dtype, strategy, schedule
    ([300, 117], 8, 2, 128, 16, "e4m3", "bf16", "vanilla", "auto"),
    ([100, 80, 33], 4, 2, 64, 32, "int8", "f16", "vanilla", "per_step"),
    ([129, 64], 6, 3, 96, 16, "e4m3", "bf16", "zigzag", "auto"),
    ([70], 4, 4, 64, 48, "int8", "f32", "vanilla", "auto"),
], ids=["fused", "per_step", "zigzag", "f32"])
def test_prefill_over_the_cache_equals_prefill_over_its_rows(gpu, case):
    # the cached prompt staged and folded: bit for bit the ring over the same rows as views
    chunks, hq, hkv, d, bs, fmt, dtype, strategy, schedule = case
    r = np.random.default_rng(30)
    s = sum(chunks)
    nb = -(-s // bs) + 1
    codes, scales = R.random_cache(r, nb, bs, hkv, d, fmt)
    table = r.permutation(nb).astype(np.int32)
    pool, sc = R.to_device(codes, scales, fmt)
    q = torch.from_numpy(r.normal(size=(hq, s, d))).to(DT[dtype]).cuda()
    k, v = (torch.from_numpy(R.rows(codes, scales, table, fmt, p, 0, s).copy()).to(DT[dtype]).cuda() for p in range(2))
    out, lse = H.kv8_ring_attention_replay_paged(q, pool, sc, torch.from_numpy(table).cuda(), chunks, strategy=strategy,
                                                 schedule=schedule)
    want, want_lse = H.ring_attention_replay(q, k, v, chunks, strategy=strategy, schedule=schedule)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


# ---- refusals (no GPU) ----
P = 256  # a pointer that is never followed: every call below is refused on the host


def _pool(**kw):
    f = dict(data=P, num_blocks=8, block_size=16, num_kv_heads=2, head_dim=64, elem_bytes=1)
    f.update(kw)
    return H.PagedPool(*[f[n] for n, _ in H.PagedPool._fields_])


BAD_POOLS = [dict(data=None), dict(num_blocks=0), dict(num_blocks=1 << 31), dict(block_size=0), dict(num_kv_heads=0),
             dict(head_dim=0), dict(head_dim=60), dict(head_dim=264), dict(elem_bytes=2), dict(data=264)]


def test_append_refusals():
    lib, view = H.lib(), H.View(P, 64, 128)

    def go(pool=None, scales=P, fmt=1, dtype=2, k=view, v=view, tokens=3, slots=P):
        return lib.hcp_kv8_append(ctypes.byref(pool or _pool()), scales, fmt, dtype, k, v, tokens, slots, None)

    for bad in BAD_POOLS:
        assert go(pool=_pool(**bad)) == -6, bad
    for bad in (dict(scales=None), dict(scales=P + 2), dict(fmt=0), dict(fmt=3), dict(dtype=4), dict(dtype=0),
                dict(tokens=-1), dict(tokens=1 << 31), dict(slots=None), dict(k=H.View(None, 64, 128)),
                dict(v=H.View(None, 64, 128)), dict(k=H.View(P + 1, 64, 128)), dict(v=H.View(P, -1, 128)),
                dict(k=H.View(P, 64, 0))):
        assert go(**bad) == -6, bad
        assert H.last_error().startswith("hcp_kv8_append:")
    assert go(tokens=0, k=H.View(None, 0, 1), v=H.View(None, 0, 1), slots=None) == 0
    assert lib.hcp_kv8_append(None, P, 1, 2, view, view, 3, P, None) == -6


def test_gather_and_prefill_refusals():
    lib, view = H.lib(), H.View(P, 64, 128)

    def go(pool=None, scales=P, fmt=1, dtype=2, table=P, n=4, off=0, t0=0, t1=64, k=view, v=view):
        return lib.hcp_kv8_gather(ctypes.byref(pool or _pool()), scales, fmt, dtype, table, n, off, t0, t1, k, v, None)

    for bad in BAD_POOLS:
        assert go(pool=_pool(**bad)) == -6, bad
    for bad in (dict(scales=None), dict(fmt=0), dict(dtype=5), dict(table=None), dict(t1=65), dict(off=1), dict(t0=9, t1=8),
                dict(k=H.View(None, 64, 128)), dict(v=H.View(P, 64, 64)), dict(k=H.View(P + 1, 64, 128))):
        assert go(**bad) == -6, bad
        assert H.last_error().startswith("hcp_kv8_gather:")
    desc, keep = H.replay_desc(torch.bfloat16, 4, 2, 64, [40, 24])

    def replay(pool=None, scales=P, fmt=1, table=P, n=4, ws=P, ws_bytes=1 << 30, q=view, out=view):
        return lib.hcp_kv8_prefill_replay_paged(ctypes.byref(desc), q, ctypes.byref(pool or _pool()), scales, fmt, table, n,
                                                out, None, ws, ws_bytes, None)

    for bad in [dict(pool=_pool(**b)) for b in BAD_POOLS] + [
            dict(scales=None), dict(fmt=7), dict(table=None), dict(n=3), dict(ws_bytes=0), dict(ws=None),
            dict(pool=_pool(num_kv_heads=4)), dict(pool=_pool(head_dim=128)), dict(q=H.View(None, 64, 128))]:
        rc = replay(**bad)
        assert rc in (-6, -5) and (rc == -6 or not torch.cuda.is_available()), bad
    assert lib.hcp_kv8_prefill_replay_paged(None, view, ctypes.byref(_pool()), P, 1, P, 4, view, None, P, 1, None) == -6
    assert lib.hcp_kv8_gather(None, P, 1, 2, P, 4, 0, 0, 64, view, view, None) == -6
    # a 16-bit entry point takes no 8-bit pool
    assert lib.hcp_paged_kv_gather(ctypes.byref(_pool()), P, 4, 0, 0, 64, view, view, None) == -6


def test_python_refusals():
    pool, sc = H.kv8_pool(4, 16, 2, 64, device="cpu")
    assert pool.dtype == torch.float8_e4m3fn and sc.shape == (2, 4, 2)
    k, slots = torch.zeros(2, 3, 64), torch.zeros(3, dtype=torch.int64)
    for args in ((pool.view(torch.uint8), sc, k, k, slots), (pool, sc[:, :3], k, k, slots), (pool, sc.double(), k, k, slots),
                 (pool, sc, k[:, :2], k, slots), (pool, sc, k, k.bfloat16(), slots), (pool, sc, k, k, slots.int()),
                 (pool[:, ::2], sc, k, k, slots), (pool, sc, k.transpose(1, 2), k, slots)):
        with pytest.raises(ValueError):
            H.kv8_append(*args)
    with pytest.raises(ValueError, match="GPU"):
        H.kv8_append(pool, sc, k, k, slots)
    with pytest.raises(ValueError):
        H.kv8_gather(pool, sc, torch.zeros(2, dtype=torch.int64), 0, 0, 20)
    with pytest.raises(ValueError):
        H.kv8_gather(pool, sc, torch.zeros(2, dtype=torch.int32), 0, 0, 20, k_out=torch.zeros(2, 19, 64))
    with pytest.raises(ValueError):
        H.kv8_ring_attention_replay_paged(torch.zeros(4, 20, 64), pool, sc, torch.zeros(2, dtype=torch.int32), [10, 9])


def _ties(fmt):
    """Values halfway between two codes, and the codes' own values (positive, above the smallest)."""
    v = R.E4M3[8:127] if fmt == "e4m3" else np.arange(1.0, 128.0)
    return (v[:-1] + v[1:]) / 2, v


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_to_blocks_of_any_scale(gpu, dtype, fmt):
    # held rows under scales that are no powers of two (quantised elsewhere): one token and three.
    # Values on and next to a tie of x / scale, where the scale stays; held codes next to a tie of
    # code * old / new, where it grows.  A code is the nearest to an fp32 product that two roundings
    # (1 / scale and the product) leave within 2 * 2^-24 (1 + 2^-24) of x / scale: where that lies
    # next to a tie the code may be the one across it, else it is equal
    r = np.random.default_rng(14)
    bs, heads, d, nb = 16, 64, 64, 4
    ties, own = _ties(fmt)
    slots = np.array([9, bs + 5, bs + 6, bs + 7, 2 * bs + 1, 3 * bs + 3, 3 * bs + 4])
    for case in ("some grow", "grow", "stay"):
        grow = case == "grow"
        if case == "stay":  # at most half of the format's range: the least power of two is not past the scale
            ties = ties[ties < R.LARGEST[fmt] / 2]
        codes, scales = R.random_cache(r, nb, bs, heads, d, fmt)
        scales[:] = np.float32(r.uniform(0.5, 1.0, scales.shape) * 2.0 ** r.integers(-6, 3, scales.shape))
        if grow:  # scale = tie / code: the code times it is a tie, but for the scale's own rounding
            c = r.integers(0, len(own), scales.shape)
            t = r.integers(0, len(ties), scales.shape)
            down = 2.0 ** np.ceil(np.log2(ties[t] / own[c]))
            scales[:] = np.float32(ties[t] / down / own[c])  # in (1/2, 1]
            one = R.encode(own[c].ravel(), fmt).reshape(c.shape)
            codes[..., ::3] = one[:, :, None, :, None]
        rows = []
        for plane in range(2):
            x = np.empty((heads, len(slots), d), np.float32)
            for i, s in enumerate(slots):
                size = scales[plane, s // bs][:, None].astype(np.float64)
                near = np.float32(r.choice(ties, (heads, d)) * size) * r.choice([-1, 1], (heads, d))
                x[:, i] = near * np.float32(0.9) if r.random() < 0.2 else near
                if grow:
                    x[:, i, 0] = R.LARGEST[fmt]  # the scale becomes 1 where it was not more
                    x[:, i, 1:] = np.clip(x[:, i, 1:], -R.LARGEST[fmt], R.LARGEST[fmt])
            rows.append(torch.from_numpy(x).to(DT[dtype]))
        pool, sc = R.to_device(codes, scales, fmt)
        held, old = R.values(codes, fmt), scales.astype(np.float64)
        H.kv8_append(pool, sc, rows[0].cuda(), rows[1].cuda(), torch.from_numpy(slots).cuda())
        before = scales.copy()
        R.append(codes, scales, rows[0].double().numpy(), rows[1].double().numpy(), slots, fmt)
        assert case != "stay" or np.array_equal(scales, before)
        got_codes, got_scales = R.to_host(pool, sc)
        assert np.array_equal(got_scales, scales)
        got, want = R.values(got_codes, fmt), R.values(codes, fmt)
        exact = held * (old / scales)[:, :, None, :, None]
        for plane in range(2):
            at = exact[plane].reshape(nb * bs, heads, d)
            at[slots] = rows[plane].double().numpy().transpose(1, 0, 2) / scales[plane].astype(np.float64)[slots // bs][:, :, None]
        # y within e of the value v, `got` the nearest code to y: |got - v| <= |got - y| + e <= |want - y| + e <= |want - v| + 2 e
        off = np.abs(got - exact) - np.abs(want - exact)
        assert (off <= 2 * np.abs(exact) * 2.0 ** -23 * (1 + 2.0 ** -20)).all(), off.max()
        whole = (np.log2(scales) % 1 == 0) & (np.log2(old) % 1 == 0)
        assert np.array_equal(got[whole[:, :, None, :].repeat(bs, 2)], want[whole[:, :, None, :].repeat(bs, 2)])
