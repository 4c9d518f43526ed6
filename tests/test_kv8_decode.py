"""Decode attention over the 8-bit paged cache against a plain restatement in 64 bits
(kv8_reference), and the whole step -- plan, projection, append, decode -- eager and captured."""
import ctypes
import math

import numpy as np
import pytest
import torch

import hcp_ring_amd as H
import kv8_reference as R

DT = {"bf16": torch.bfloat16, "f16": torch.float16}

# The kernel's products q * code are exact (16-bit q, codes of at most 8 significant bits) and
# summed in fp32; so are the softmax statistics.  A score is a sum of D <= 128 products in at
# most 128 + 8 roundings of 2^-24 of the partial sums, |S| <= sum |q c| s / sqrt(D): with the
# inputs below sum |q c| s / sqrt(D) <= 2^6, so |dS| <= 2^6 * 136 * 2^-24 < 2^-10.9 at the very worst and
# about sqrt(136) instead of 136 as a rule: 2^-14.  exp turns that into a relative error of a
# weight; weights carry 22 bits beside it.  o is an average of V, |V| <= vmax: |do| <= 2 |dS| vmax.
SCORE = 2.0 ** -14


def tolerance(vmax, out_dtype):
    """Largest |o - exact|: the scores' error, sums of up to 16k weights in 32 bits, one output rounding."""
    step = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[out_dtype]
    return vmax * (2 * SCORE + 2.0 ** -18 + step)


def reference(q, codes, scales, fmt, shards, lens, t0=0, scale=None):
    """fp64 rows over the shards' tokens: (o [B, Hq, D], lse [B, Hq])."""
    b, hq, d = q.shape
    hkv = codes.shape[3]
    rep = hq // hkv
    o, lse = np.zeros((b, hq, d)), np.zeros((b, hq))
    for i in range(b):
        kv = [np.concatenate([R.rows(codes, scales, t[i], fmt, p, min(t0, n[i]), n[i]) for t, n in zip(shards, lens)], 1)
              for p in range(2)]
        for h in range(hkv):
            at = slice(h * rep, (h + 1) * rep)
            o[i, at], lse[i, at] = R.attend(q[i, at], kv[0][h], kv[1][h], scale or 1 / math.sqrt(d))
    return o, lse


def inputs(seed, b, hq, hkv, d, bs, dtype, fmt, tokens, domains=1, q_layout="plain", spread=3):
    r = np.random.default_rng(seed)
    lens = [r.integers(0, tokens + 1, b) for _ in range(domains)]
    lens[0][0] = tokens
    blocks = [max(1, -(-int(n.max()) // bs)) for n in lens]
    nb = b * sum(blocks) + 1
    codes, scales = R.random_cache(r, nb, bs, hkv, d, fmt, spread)
    ids = r.permutation(nb).astype(np.int32)
    tables, cur = [], 0
    for n in blocks:
        tables.append(ids[cur: cur + b * n].reshape(b, n))
        cur += b * n
    qt = torch.from_numpy(r.normal(size=(b, hq, d)) * 0.5).to(DT[dtype])
    q = qt.double().numpy()
    if q_layout == "strided":  # rows of a wider projection output
        wide = torch.zeros(b, hq + 2, d + 8, dtype=DT[dtype])
        wide[:, 1: hq + 1, :d] = qt
        qt = wide.cuda()[:, 1: hq + 1, :d]
    return r, lens, codes, scales, tables, qt.cuda(), q


def compare(got, lse, want, want_lse, vmax):
    o = got.double().cpu().numpy()
    assert np.isfinite(o).all()
    err = np.abs(o - want).max() if o.size else 0.0
    assert err <= tolerance(vmax, got.dtype), err
    l = lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(l), np.isneginf(want_lse))
    fin = np.isfinite(want_lse)
    # ln of a sum whose terms are off by dS, rounded at |lse| < 2^7
    assert np.abs(l[fin] - want_lse[fin]).max(initial=0) <= 2 * SCORE + 2.0 ** -16


PARTIAL = [
    # seed, batch, Hq, Hkv, D, block size, dtype, format, tokens, t0
    (1, 1, 32, 8, 128, 16, "bf16", "e4m3", 1, 0),
    (2, 3, 16, 2, 128, 16, "f16", "int8", 37, 0),
    (3, 2, 14, 2, 64, 32, "bf16", "e4m3", 515, 3),
    (4, 5, 8, 1, 96, 48, "f16", "e4m3", 300, 0),
    (5, 2, 16, 1, 128, 16, "bf16", "int8", 1000, 100),
    (6, 40, 4, 4, 64, 16, "bf16", "int8", 70, 0),
    (7, 1, 4, 4, 8, 16, "f16", "e4m3", 130, 129),
    (8, 2, 10, 5, 120, 128, "bf16", "e4m3", 400, 17),
    (9, 1, 32, 8, 128, 16, "bf16", "e4m3", 9000, 0),
    (10, 3, 9, 3, 40, 16, "f16", "int8", 33, 32),
    (11, 1, 5, 1, 72, 80, "bf16", "int8", 2000, 0),
    (12, 70, 24, 12, 128, 64, "f16", "e4m3", 200, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("q_layout", ["plain", "strided"])
@pytest.mark.parametrize("case", PARTIAL, ids=[str(c[0]) for c in PARTIAL])
def test_decode_partial(gpu, case, q_layout):
    seed, b, hq, hkv, d, bs, dtype, fmt, tokens, t0 = case
    _, lens, codes, scales, tables, qt, q = inputs(seed, b, hq, hkv, d, bs, dtype, fmt, tokens, q_layout=q_layout)
    pool, sc = R.to_device(codes, scales, fmt)
    n = torch.from_numpy(lens[0].astype(np.int32)).cuda()
    H.fetch_device_errors()
    o, lse = H.kv8_decode_partial(qt, pool, sc, torch.from_numpy(tables[0]).cuda(), t0, tokens, seq_lens=n)
    want, want_lse = reference(q, codes, scales, fmt, tables, lens, t0)
    compare(o, lse, want, want_lse, R.LARGEST[fmt] * scales.max())
    assert H.fetch_device_errors() == 0


SPLIT = [
    # seed, batch, Hq, Hkv, D, block size, format, longest, sequences that hold more than a block
    (31, 1, 16, 1, 128, 16, "e4m3", 30000, 1),  # 16 waves of a head meet in LDS: 133 KB of it
    (32, 1, 16, 1, 64, 16, "int8", 30000, 1),
    (33, 1, 16, 1, 96, 16, "e4m3", 30000, 1),   # 8 waves
    (34, 2, 8, 8, 128, 64, "e4m3", 9000, 2),
    (35, 70, 8, 2, 64, 16, "int8", 4000, 5),    # more than 64 sequences in one row
    (36, 65, 16, 8, 128, 16, "e4m3", 3000, 65),
    (37, 200, 10, 5, 40, 32, "e4m3", 2500, 9),
    (38, 1024, 4, 4, 8, 16, "int8", 4000, 12),
    (39, 1025, 4, 4, 8, 16, "e4m3", 4000, 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", SPLIT, ids=[str(c[0]) for c in SPLIT])
def test_decode_of_few_long_and_many_short_sequences(gpu, case):
    """Lengths from none to the longest in one call, the empty ones also first, last and in a row;
    sequences share blocks, and a table names a block twice.  A wave sums at most a few thousand
    weights here and the waves' sums are joined in 32 bits, so `tolerance` holds as it stands."""
    seed, b, hq, hkv, d, bs, fmt, longest, long_ones = case
    r = np.random.default_rng(seed)
    lens = r.integers(0, bs + 1, b)
    lens[r.permutation(b)[:long_ones]] = r.integers(1, longest + 1, long_ones)
    if b > 8:
        lens[[0, b // 2, b // 2 + 1, b - 1]] = 0
    lens[b // 3] = longest
    codes, scales = R.random_cache(r, 60, bs, hkv, d, fmt, 3)
    table = r.integers(0, 60, (b, -(-longest // bs))).astype(np.int32)
    qt = torch.from_numpy(r.normal(size=(b, hq, d)) * 0.5).to(torch.bfloat16)
    pool, sc = R.to_device(codes, scales, fmt)
    H.fetch_device_errors()
    o, lse = H.kv8_decode_partial(qt.cuda(), pool, sc, torch.from_numpy(table).cuda(), 0, longest,
                                  seq_lens=torch.from_numpy(lens.astype(np.int32)).cuda())
    want, want_lse = reference(qt.double().numpy(), codes, scales, fmt, [table], [lens])
    compare(o, lse, want, want_lse, R.LARGEST[fmt] * scales.max())
    assert H.fetch_device_errors() == 0


RING = [
    # seed, batch, Hq, Hkv, D, block size, dtype, format, tokens, domains, seed domain
    (21, 2, 32, 8, 128, 16, "bf16", "e4m3", 200, 3, 1),
    (22, 4, 16, 2, 128, 32, "f16", "int8", 65, 2, 0),
    (23, 1, 14, 2, 64, 16, "bf16", "e4m3", 1500, 4, 3),
    (24, 3, 6, 3, 96, 16, "f16", "int8", 40, 7, 2),
    (25, 30, 8, 8, 64, 16, "bf16", "int8", 20, 64, 5),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", RING, ids=[str(c[0]) for c in RING])
def test_decode_ring(gpu, case):
    seed, b, hq, hkv, d, bs, dtype, fmt, tokens, domains, start = case
    _, lens, codes, scales, tables, qt, q = inputs(seed, b, hq, hkv, d, bs, dtype, fmt, tokens, domains)
    pool, sc = R.to_device(codes, scales, fmt)
    shards = [(torch.from_numpy(t).cuda(), torch.from_numpy(n.astype(np.int32)).cuda(), int(n.max()))
              for t, n in zip(tables, lens)]
    out, lse = H.kv8_decode_ring_replay(qt, pool, sc, shards, start)
    want, want_lse = reference(q, codes, scales, fmt, tables, lens)
    assert out.dtype == DT[dtype]
    compare(out, lse, want, want_lse, R.LARGEST[fmt] * scales.max())
    # without lengths every sequence has max_len tokens; a strided out
    if len({n.max() for n in lens}) and all(n.max() > 0 for n in lens):
        wide = torch.empty(b, hq, d + 4, dtype=DT[dtype], device="cuda")
        full = [np.full(b, n.max()) for n in lens]
        out, lse = H.kv8_decode_ring_replay(qt, pool, sc, [(t, None, m) for t, _, m in shards], start, out=wide[:, :, :d])
        want, want_lse = reference(q, codes, scales, fmt, tables, full)
        compare(out, lse, want, want_lse, R.LARGEST[fmt] * scales.max())


@pytest.mark.gpu
def test_decode_empty_ranges_and_tables(gpu):
    # no tokens at all: zeros and -inf; an empty shard without a table beside a full one
    _, lens, codes, scales, tables, qt, q = inputs(31, 3, 8, 2, 64, 16, "bf16", "e4m3", 50)
    pool, sc = R.to_device(codes, scales, "e4m3")
    table = torch.from_numpy(tables[0]).cuda()
    for t0, t1, n in ((0, 0, None), (7, 7, None), (0, 50, torch.zeros(3, dtype=torch.int32).cuda()),
                      (20, 50, torch.full((3,), 20, dtype=torch.int32).cuda()), (0, 50, torch.full((3,), -4, dtype=torch.int32).cuda())):
        o = torch.full((3, 8, 64), 9.0, device="cuda")
        o, lse = H.kv8_decode_partial(qt, pool, sc, table, t0, t1, seq_lens=n, o=o)
        assert (o == 0).all() and (lse == -math.inf).all()
    n = torch.from_numpy(lens[0].astype(np.int32)).cuda()
    one, l1 = H.kv8_decode_ring_replay(qt, pool, sc, [(table, n, 50)], 0)
    two, l2 = H.kv8_decode_ring_replay(qt, pool, sc, [(None, None, 0), (table, n, 50)], 1)
    assert torch.equal(one, two) and torch.equal(l1, l2)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_decode_does_not_read_past_the_tokens(gpu, fmt):
    # NaN codes and NaN scales behind the last token, in later blocks and table entries past
    # a sequence's own change no bit
    b, tokens, bs = 3, 90, 16
    _, lens, codes, scales, tables, qt, q = inputs(32, b, 8, 2, 128, bs, "bf16", fmt, tokens)
    n = torch.from_numpy(lens[0].astype(np.int32)).cuda()
    pool, sc = R.to_device(codes, scales, fmt)
    want = H.kv8_decode_partial(qt, pool, sc, torch.from_numpy(tables[0]).cuda(), 5, tokens, seq_lens=n)
    dirty, dirty_s, dirty_t = codes.copy(), scales.copy(), tables[0].copy()
    used = set()
    for i in range(b):
        for e in range(tables[0].shape[1]):
            lo = min(max(lens[0][i] - e * bs, 0), bs)
            dirty[:, tables[0][i, e], lo:] = 0x7f
            if e == 0:
                dirty[:, tables[0][i, e], :5] = 0x7f  # before t0
            if lo == 0:
                dirty_t[i, e] = 1 << 30
                dirty_s[:, tables[0][i, e]] = math.nan
            else:
                used.add(int(tables[0][i, e]))
    pool, sc = R.to_device(dirty, dirty_s, fmt)
    H.fetch_device_errors()
    got = H.kv8_decode_partial(qt, pool, sc, torch.from_numpy(dirty_t).cuda(), 5, tokens, seq_lens=n)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
def test_decode_values_that_are_not_finite(gpu):
    # a NaN scale (K or V) or a NaN e4m3 code that is visible reaches the rows of its head and
    # no other; a NaN or infinite q its own row
    b, tokens, bs = 2, 300, 16
    _, lens, codes, scales, tables, qt, q = inputs(33, b, 8, 2, 128, bs, "bf16", "e4m3", tokens)
    lens[0][:] = tokens
    table = torch.from_numpy(tables[0]).cuda()
    run = lambda c, s, qq: H.kv8_decode_partial(qq, *R.to_device(c, s, "e4m3"), table, 0, tokens)  # noqa: E731
    o, lse = run(codes, scales, qt)
    for plane, code in ((0, False), (1, False), (0, True), (1, True)):
        c, s = codes.copy(), scales.copy()
        if code:
            c[plane, tables[0][1, 9], 3, 1, 17] = 0x7f
        else:
            s[plane, tables[0][1, 9], 1] = math.nan
        go, gl = run(c, s, qt)
        if plane == 0:
            assert torch.isnan(go[1, 4:]).all() and torch.isnan(gl[1, 4:]).all()
        else:
            assert torch.isnan(go[1, 4:, 17]).all() and torch.equal(gl, lse)
            assert code is False or not torch.isnan(go[1, 4:, 18]).any()
        assert torch.equal(go[0], o[0]) and torch.equal(go[1, :4], o[1, :4]) and torch.equal(gl[1, :4], lse[1, :4])
    for bad in (math.nan, math.inf):
        qq = qt.clone()
        qq[1, 3, 8] = bad
        go, gl = run(codes, scales, qq)
        assert torch.isnan(go[1, 3]).all()
        keep = torch.ones(b, 8, dtype=torch.bool, device="cuda")
        keep[1, 3] = False
        assert torch.equal(go[keep], o[keep]) and torch.equal(gl[keep], lse[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_decode_scales_far_apart(gpu, fmt):
    # blocks whose V scales differ by up to 2^40, the largest on tokens that weigh next to
    # nothing and on tokens that weigh all; zero scales; tiny and huge q
    b, tokens, bs, d = 4, 160, 16, 128
    r, lens, codes, scales, tables, qt, q = inputs(34, b, 4, 1, d, bs, "bf16", fmt, tokens)
    lens[0][:] = tokens
    scales[1] *= (2.0 ** r.integers(-20, 21, scales[1].shape)).astype(np.float32)
    scales[1, tables[0][0, 2]] = 0
    scales[0, tables[0][0, 4]] = 0
    pool, sc = R.to_device(codes, scales, fmt)
    for size in (1.0, 2.0 ** -60, 30.0):
        qs = (qt.float() * size).to(qt.dtype)
        o, lse = H.kv8_decode_partial(qs, pool, sc, torch.from_numpy(tables[0]).cuda(), 0, tokens)
        want, want_lse = reference(qs.double().cpu().numpy(), codes, scales, fmt, tables, lens)
        top = np.abs(want).max(axis=(1, 2))  # a row's own size: V's largest value may weigh nothing
        err = np.abs(o.double().cpu().numpy() - want).max(axis=(1, 2))
        assert (err <= top * (2 * SCORE * 32 + 2.0 ** -18)).all(), (size, err / top)  # |S| up to 30 times larger
        assert np.abs(lse.double().cpu().numpy() - want_lse).max() <= 2 * SCORE * 32


@pytest.mark.gpu
def test_decode_bad_block_ids(gpu):
    # ids outside the pool are skipped, and flagged, as the 16-bit decode does
    _, lens, codes, scales, tables, qt, q = inputs(35, 1, 8, 2, 64, 16, "bf16", "int8", 100)
    pool, sc = R.to_device(codes, scales, "int8")
    t = tables[0].copy()
    t[0, 2], t[0, 4] = -1, codes.shape[1]
    H.fetch_device_errors()
    o, lse = H.kv8_decode_partial(qt, pool, sc, torch.from_numpy(t).cuda(), 0, 100)
    assert H.fetch_device_errors() == 1
    keep = [i for i in range(100) if i // 16 not in (2, 4)]
    k, v = (R.rows(codes, scales, tables[0][0], "int8", p, 0, 100)[:, keep] for p in range(2))
    for h in range(2):
        want, wl = R.attend(q[0, 4 * h: 4 * h + 4], k[h], v[h], 1 / 8)
        compare(o[0, 4 * h: 4 * h + 4], lse[0, 4 * h: 4 * h + 4], want, wl, 127 * scales.max())


@pytest.mark.gpu
def test_decode_workspace_sizes_serve_shorter_contexts(gpu):
    # a workspace sized for the longest context serves every shorter one, bit for bit
    _, lens, codes, scales, tables, qt, q = inputs(36, 2, 8, 2, 128, 16, "bf16", "e4m3", 3000)
    pool, sc = R.to_device(codes, scales, "e4m3")
    table = torch.from_numpy(tables[0]).cuda()
    ws = torch.empty(max(1, H.kv8_decode_workspace_size(qt, pool, table, 0, 3000)), dtype=torch.uint8, device="cuda")
    for t1 in (1, 16, 17, 100, 800, 2999, 3000):
        a = H.kv8_decode_partial(qt, pool, sc, table, 0, t1)
        ws.fill_(0xff)
        b = H.kv8_decode_partial(qt, pool, sc, table, 0, t1, workspace=ws)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def _step(case, st):
    """One decode step of a layer: plan, projection, append, decode."""
    hq, hkv, d, bs = case
    H.kv_plan_step(st["lens"], st["new"], st["tables"], st["free"], st["count"], bs, slots=st["slots"],
                   positions=st["pos"], token_starts=st["starts"], seq_lens_out=st["lens"], free_count_out=st["count"],
                   workspace=st["plan_ws"])
    H.qkv_rope_project(st["x"], *st["w"], hq, hkv, d, positions=st["pos"], table=st["rope"], q_out=st["q"],
                       k_out=st["k"], v_out=st["v"])
    H.kv8_append(st["pool"], st["scales"], st["k"], st["v"], st["slots"])
    return H.kv8_decode_ring_replay(st["q"].permute(1, 0, 2), st["pool"], st["scales"], [(st["tables"], st["lens"], st["max"])],
                                    0, out=st["out"], lse_out=st["lse"], workspace=st["ws"])


def _step_state(seed, case, batch, fmt, width=10):
    hq, hkv, d, bs = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    e = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
    i32 = torch.int32
    nb = batch * width
    st = dict(lens=torch.zeros(batch, dtype=i32, device="cuda"), new=torch.ones(batch, dtype=i32, device="cuda"),
              tables=torch.full((batch, width), -1, dtype=i32, device="cuda"),
              free=torch.randperm(nb, generator=g, device="cuda").to(i32), count=torch.tensor([nb], dtype=i32, device="cuda"),
              slots=e(batch, dt=torch.int64), pos=e(batch, dt=torch.int64), starts=e(batch + 1, dt=i32),
              plan_ws=e(H.kv_plan_workspace_size(batch), dt=torch.uint8), x=rnd(batch, 256),
              w=[rnd(n * d, 256) / 16 for n in (hq, hkv, hkv)], rope=H.rope_table(d, width * bs, 10000.0),
              q=e(hq, batch, d), k=e(hkv, batch, d), v=e(hkv, batch, d), out=e(batch, hq, d), lse=e(batch, hq, dt=torch.float32),
              max=width * bs, g=g)
    st["pool"], st["scales"] = H.kv8_pool(nb, bs, hkv, d, R.TORCH[fmt])
    q = st["q"].permute(1, 0, 2)
    st["ws"] = e(max(1, H.kv8_decode_ring_workspace_size(q, st["pool"], [(st["tables"], st["lens"], st["max"])])), dt=torch.uint8)
    return st


@pytest.mark.gpu
@pytest.mark.parametrize("case,batch,fmt", [((8, 2, 128, 16), 3, "e4m3"), ((4, 2, 64, 32), 5, "int8")])
def test_step_of_all_operators(gpu, case, batch, fmt):
    # prompts of different lengths come first by one ragged append, then decode steps; every
    # step's rows against attention in 64 bits over the rows that the cache should hold
    hq, hkv, d, bs = case
    st = _step_state(40, case, batch, fmt)
    prompt = [37 - 9 * i for i in range(batch)]
    prompt[-1] = 0
    total = sum(prompt)
    new = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    slots, pos, starts, _, _ = H.kv_plan_step(st["lens"], new, st["tables"], st["free"], st["count"], bs, total + 4,
                                              seq_lens_out=st["lens"], free_count_out=st["count"])
    x = torch.randn(total + 4, 256, generator=st["g"], device="cuda", dtype=torch.bfloat16)  # a padded batch
    _, k, v = H.qkv_rope_project(x, *st["w"], hq, hkv, d, positions=pos, table=st["rope"])
    H.kv8_append(st["pool"], st["scales"], k, v, slots)
    codes, scales = (a.copy() for a in R.to_host(*H.kv8_pool(st["pool"].shape[1], bs, hkv, d, R.TORCH[fmt])))
    host = lambda t: t.double().cpu().numpy()  # noqa: E731
    R.append(codes, scales, host(k), host(v), slots.cpu().numpy(), fmt)
    H.fetch_device_errors()
    for step in range(2 * bs):
        st["x"].copy_(torch.randn(batch, 256, generator=st["g"], device="cuda", dtype=torch.bfloat16))
        out, lse = _step(case, st)
        R.append(codes, scales, host(st["k"]), host(st["v"]), st["slots"].cpu().numpy(), fmt)
        got_codes, got_scales = R.to_host(st["pool"], st["scales"])
        assert np.array_equal(got_codes, codes) and np.array_equal(got_scales, scales), step
        lens = st["lens"].cpu().numpy()
        assert lens.tolist() == [p + step + 1 for p in prompt]
        want, want_lse = reference(host(st["q"].permute(1, 0, 2)), codes, scales, fmt, [st["tables"].cpu().numpy()], [lens])
        compare(out, lse, want, want_lse, R.LARGEST[fmt] * scales.max())
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
def test_step_replays_in_a_graph(gpu):
    # the whole step captured once and replayed as the sequences grow, end and start again, with
    # eager work between the replays; a second, eager state does the same steps
    case, batch = (8, 2, 128, 16), 4
    a, b = (_step_state(41, case, batch, "e4m3") for _ in range(2))
    for st in (a, b):
        _step(case, st)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _step(case, a)
    r = np.random.default_rng(5)
    for step in range(40):
        x = torch.randn(batch, 256, generator=a["g"], device="cuda", dtype=torch.bfloat16)
        new = np.ones(batch, np.int32)
        if step in (9, 20):
            new[r.integers(batch)] = -1
        for st in (a, b):
            st["x"].copy_(x)
            st["new"].copy_(torch.from_numpy(new).cuda())
        torch.cuda.synchronize()
        g.replay()
        _step(case, b)
        torch.cuda.synchronize()
        for name in ("lens", "tables", "free", "count", "slots", "pos", "out", "lse", "scales"):
            assert torch.equal(a[name], b[name]), (step, name)
        assert torch.equal(a["pool"].view(torch.uint8), b["pool"].view(torch.uint8)), step


@pytest.mark.gpu
def test_decode_on_another_stream(gpu):
    _, lens, codes, scales, tables, qt, q = inputs(37, 3, 8, 2, 64, 16, "f16", "int8", 200)
    pool, sc = R.to_device(codes, scales, "int8")
    table = torch.from_numpy(tables[0]).cuda()
    want = H.kv8_decode_partial(qt, pool, sc, table, 0, 200)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    ws = torch.empty(max(1, H.kv8_decode_workspace_size(qt, pool, table, 0, 200)), dtype=torch.uint8, device="cuda")
    o, l = torch.empty_like(want[0]), torch.empty_like(want[1])
    torch.cuda.synchronize()
    H.kv8_decode_partial(qt, pool, sc, table, 0, 200, workspace=ws, o=o, lse=l, stream=s)
    s.synchronize()
    assert torch.equal(o, want[0]) and torch.equal(l, want[1])


def _two_decodes():
    """Two calls that split sequences over workers: (q, pool, scales, table, tokens, lens) and what they give."""
    calls = []
    for seed, heads in ((38, (8, 2, 128)), (39, (8, 8, 64))):
        _, lens, codes, scales, tables, qt, _ = inputs(seed, 3, *heads, 16, "bf16", "e4m3", 4000)
        pool, sc = R.to_device(codes, scales, "e4m3")
        calls.append((qt, pool, sc, torch.from_numpy(tables[0]).cuda(), 4000, torch.from_numpy(lens[0].astype(np.int32)).cuda()))
    want = [H.kv8_decode_partial(q, p, sc, t, 0, n, seq_lens=l) for q, p, sc, t, n, l in calls]
    torch.cuda.synchronize()
    return calls, want


@pytest.mark.gpu
def test_two_calls_at_once(gpu):
    calls, want = _two_decodes()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        got = [H.kv8_decode_partial(q, p, sc, t, 0, n, seq_lens=l, stream=s) for s, (q, p, sc, t, n, l) in zip(streams, calls)]
        torch.cuda.synchronize()
        for (o, l), (wo, wl) in zip(got, want):
            assert torch.equal(o, wo) and torch.equal(l, wl)


@pytest.mark.gpu
def test_two_graphs_share_a_workspace(gpu):
    calls, want = _two_decodes()
    size = max(H.kv8_decode_workspace_size(q, p, t, 0, n) for q, p, _, t, n, _ in calls)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN
    graphs, outs = [], []
    for q, p, sc, t, n, l in calls:
        o, lse = torch.empty(q.shape, device="cuda"), torch.empty(q.shape[:2], device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            H.kv8_decode_partial(q, p, sc, t, 0, n, seq_lens=l, workspace=ws, o=o, lse=lse)
        graphs.append(g)
        outs.append((o, lse))
    for k in (0, 1, 1, 0, 1):
        outs[k][0].fill_(7)
        graphs[k].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[k][0], want[k][0]) and torch.equal(outs[k][1], want[k][1])


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    """A cache of two planes of 4.3e9 codes, its last blocks in use, rows 2^28 elements apart: bit
    for bit as the same blocks in a small cache with packed rows."""
    hkv, d, bs, tokens = 8, 128, 16, 40
    nb = (1 << 32) // (bs * hkv * d) + 64
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of device memory")
    pool = torch.empty(2, nb, bs, hkv, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.zeros(2, nb, hkv, device="cuda")
    small, small_scales = H.kv8_pool(64, bs, hkv, d)
    ids = torch.tensor([nb - 1, 3, nb - 64], dtype=torch.int32, device="cuda")
    near = torch.tensor([63, 3, 0], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(9)
    k, v = (torch.randn(hkv, tokens, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    big = torch.empty(((tokens - 1) << 28) + hkv * d, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((hkv, tokens, d), (d, 1 << 28, 1))
    far.copy_(k)
    slot = lambda t: (t.long()[:, None] * bs + torch.arange(bs, device="cuda")).flatten()[:tokens]  # noqa: E731
    H.kv8_append(pool, scales, far, v, slot(ids))
    H.kv8_append(small, small_scales, k, v, slot(near))
    out = far.zero_()
    gk, gv = H.kv8_gather(small, small_scales, near, 0, 0, tokens)
    rows = torch.empty_like(big).as_strided(out.shape, out.stride())
    H.kv8_gather(pool, scales, ids, 0, 0, tokens, k_out=out, v_out=rows)
    assert torch.equal(out, gk) and torch.equal(rows, gv)
    q = torch.randn(2, 32, d, generator=g, device="cuda").bfloat16()
    tables, near_tables = (torch.stack([t, t.flip(0)]) for t in (ids, near))
    lens = torch.tensor([tokens, 17], dtype=torch.int32, device="cuda")
    got = H.kv8_decode_partial(q, pool, scales, tables, 0, tokens, seq_lens=lens)
    want = H.kv8_decode_partial(q, small, small_scales, near_tables, 0, tokens, seq_lens=lens)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("as_handle", [False, True])
def test_memory_made_by_a_call_is_its_streams(gpu, monkeypatch, as_handle):
    """Outputs and workspaces that a call makes come from the memory of the stream it is given."""
    pool, sc = H.kv8_pool(20, 16, 2, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens, one = torch.arange(20, **i32).view(2, 10), torch.full((2,), 100, **i32), torch.ones(2, **i32)
    q, rows = torch.randn(2, 8, 64, device="cuda", dtype=torch.bfloat16), torch.randn(8, 100, 64, device="cuda", dtype=torch.bfloat16)
    sc.fill_(1)
    s = torch.cuda.Stream()
    handle = s.cuda_stream if as_handle else s
    calls = [lambda st: H.kv_plan_step(lens, one, table.clone(), torch.zeros(20, **i32), torch.zeros(1, **i32), 16, capacity=2, stream=st),
             lambda st: H.kv8_gather(pool, sc, table[0], 0, 0, 100, stream=st),
             lambda st: H.kv8_decode_partial(q, pool, sc, table, 0, 100, seq_lens=lens, stream=st),
             lambda st: H.kv8_decode_ring_replay(q, pool, sc, [(table, lens, 100)], 0, stream=st),
             lambda st: H.kv8_ring_attention_replay_paged(rows, pool, sc, table[0], [60, 40], stream=st)]
    empty, seen = torch.empty, []

    def watched(*args, **kw):
        seen.append(torch.cuda.current_stream().cuda_stream)
        return empty(*args, **kw)

    torch.cuda.synchronize()
    for call in calls:
        want = call(None)
        torch.cuda.synchronize()
        monkeypatch.setattr(torch, "empty", watched)
        seen.clear()
        got = call(handle)
        monkeypatch.setattr(torch, "empty", empty)
        assert len(seen) >= 2 and set(seen) == {s.cuda_stream}
        s.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


# ---- refusals (no GPU) ----
P = 256  # a pointer that is never followed: every call below is refused on the host


def _pool(**kw):
    f = dict(data=P, num_blocks=8, block_size=16, num_kv_heads=2, head_dim=64, elem_bytes=1)
    f.update(kw)
    return H.PagedPool(*[f[n] for n, _ in H.PagedPool._fields_])


def _desc(**kw):
    f = dict(dtype=2, batch=2, num_q_heads=8, num_kv_heads=2, head_dim=64, reserved0=0, t0=0, t1=64, table_stride=4,
             table_len=4, scale=0.125)
    f.update(kw)
    return H.DecodeDesc(*[f[n] for n, _ in H.DecodeDesc._fields_])


BAD = [dict(pool=dict(data=None)), dict(pool=dict(elem_bytes=2)), dict(pool=dict(num_blocks=0)), dict(pool=dict(block_size=24)),
       dict(pool=dict(num_kv_heads=4)), dict(pool=dict(head_dim=128)), dict(pool=dict(data=P + 8)),
       dict(desc=dict(head_dim=136), pool=dict(head_dim=136)), dict(desc=dict(dtype=3)), dict(desc=dict(dtype=0)),
       dict(desc=dict(batch=0)), dict(desc=dict(num_q_heads=0)), dict(desc=dict(num_q_heads=7)), dict(desc=dict(num_q_heads=34)),
       dict(desc=dict(scale=0.0)), dict(desc=dict(scale=-1.0)), dict(scales=None), dict(fmt=0), dict(fmt=3),
       dict(q=H.View(None, 64, 512)), dict(q=H.View(P + 2, 64, 512)), dict(q=H.View(P, 65, 512)), dict(q=H.View(P, 64, 0))]


@pytest.mark.parametrize("bad", BAD + [dict(desc=dict(t0=-1)), dict(desc=dict(t0=65)), dict(desc=dict(t1=65)),
                                       dict(desc=dict(table_len=0)), dict(desc=dict(table_stride=3)), dict(tables=None),
                                       dict(o=None), dict(lse=None), dict(o=P + 4)], ids=str)
def test_decode_partial_refusals(bad):
    kw = dict(scales=P, fmt=1, q=H.View(P, 64, 512), tables=P, o=P, lse=P)
    kw.update({k: v for k, v in bad.items() if k in kw})
    rc = H.lib().hcp_kv8_decode_partial(ctypes.byref(_desc(**bad.get("desc", {}))), ctypes.byref(_pool(**bad.get("pool", {}))),
                                        kw["scales"], kw["fmt"], kw["q"], kw["tables"], None, kw["o"], kw["lse"], P, 1 << 30, None)
    assert rc == -6 and H.last_error().startswith("hcp_kv8_decode_partial:")


@pytest.mark.parametrize("bad", BAD + [dict(n=0), dict(n=65), dict(seed=2), dict(seed=-1), dict(shard=(None, 4, 4, None, 10)),
                                       dict(shard=(P, 4, 4, None, 65)), dict(shard=(P, 3, 4, None, 10)),
                                       dict(shard=(P, 4, 0, None, 10)), dict(shard=(P, 4, 4, None, -1)),
                                       dict(out=H.View(None, 64, 512)), dict(out=H.View(P, 64, 500)), dict(out=H.View(P + 2, 64, 512))],
                         ids=str)
def test_decode_ring_refusals(bad):
    kw = dict(scales=P, fmt=1, q=H.View(P, 64, 512), n=2, seed=0, out=H.View(P, 64, 512), shard=(P, 4, 4, None, 64))
    kw.update({k: v for k, v in bad.items() if k in kw})
    shards = (H.DecodeShard * 65)(*[H.DecodeShard(*kw["shard"])] * 65)
    rc = H.lib().hcp_kv8_decode_ring_replay(ctypes.byref(_desc(**bad.get("desc", {}))), ctypes.byref(_pool(**bad.get("pool", {}))),
                                            kw["scales"], kw["fmt"], kw["q"], kw["n"], shards, kw["seed"], kw["out"], None, P,
                                            1 << 30, None)
    assert rc == -6 and H.last_error().startswith("hcp_kv8_decode_ring_replay:")


def test_decode_null_and_python_refusals():
    lib, v = H.lib(), H.View(P, 64, 512)
    assert lib.hcp_kv8_decode_partial(None, None, None, 0, v, None, None, None, None, None, 0, None) == -6
    assert lib.hcp_kv8_decode_ring_replay(None, None, None, 0, v, 0, None, 0, v, None, None, 0, None) == -6
    assert lib.hcp_kv8_decode_workspace_size(None, None) == 0
    assert lib.hcp_kv8_decode_ring_workspace_size(None, None, 1, None) == 0
    pool, sc = H.kv8_pool(4, 16, 2, 64, torch.int8, device="cpu")
    q, table = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32)
    for args, kw in (((q[:, :, :32], pool, sc, table, 0, 20), {}), ((q, pool.float(), sc, table, 0, 20), {}),
                     ((q, pool, sc[:1], table, 0, 20), {}), ((q, pool, sc, table.long(), 0, 20), {}),
                     ((q, pool, sc, table[:2], 0, 20), {}), ((q, pool, sc, table, 0, 20), dict(seq_lens=torch.zeros(3))),
                     ((q, pool, sc, table, 0, 20), dict(o=torch.zeros(3, 4, 64, dtype=torch.bfloat16))),
                     ((q, pool, sc, table, 0, 20), dict(lse=torch.zeros(4, 3)))):
        with pytest.raises(ValueError):
            H.kv8_decode_partial(*args, **kw)
    with pytest.raises(ValueError):
        H.kv8_decode_ring_replay(q, pool, sc, [(table[:2], None, 20)], 0)


@pytest.mark.parametrize("heads", [(32, 8, 128), (16, 2, 128), (14, 2, 64), (8, 1, 96), (40, 5, 64)])
@pytest.mark.parametrize("batch", [1, 3, 40, 300])
def test_decode_workspace_covers_every_shorter_context(heads, batch):
    hq, hkv, d = heads
    pool = _pool(num_kv_heads=hkv, head_dim=d)
    sizes, rings = [], []
    for tokens in [*range(1, 1200, 13), 2048, 4099, 16384, 131072]:
        desc = _desc(batch=batch, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, t1=tokens)
        sizes.append(H.lib().hcp_kv8_decode_workspace_size(ctypes.byref(desc), ctypes.byref(pool)))
        shards = (H.DecodeShard * 3)(*[H.DecodeShard(P, 1 << 14, 1 << 14, None, t) for t in (tokens, tokens // 2, tokens // 7)])
        rings.append(H.lib().hcp_kv8_decode_ring_workspace_size(ctypes.byref(desc), ctypes.byref(pool), 3, shards))
    for s in (sizes, rings):
        assert all(a <= b for a, b in zip(s, s[1:])), (batch, heads)


def test_decode_ring_refuses_an_out_of_strided_rows():
    # strides of rows and heads that fit each other, but two elements from one dim to the next
    pool, sc = H.kv8_pool(4, 16, 2, 64, device="cpu")
    q, table = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32)
    for out in (torch.zeros(3, 4, 64, 2, dtype=q.dtype)[..., 0], torch.zeros(3, 64, 4, dtype=q.dtype).transpose(1, 2)):
        with pytest.raises(ValueError, match="contiguous rows"):
            H.kv8_decode_ring_replay(q, pool, sc, [(table, None, 20)], 0, out=out)
    with pytest.raises(ValueError, match="GPU"):  # a wider row's slice is taken
        H.kv8_decode_ring_replay(q, pool, sc, [(table, None, 20)], 0, out=torch.zeros(3, 4, 72, dtype=q.dtype)[..., :64])
