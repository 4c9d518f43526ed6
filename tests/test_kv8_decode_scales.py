"""Decode attention over the 8-bit paged cache where its scales are zero, tiny or far apart,
against the plain restatement in 64 bits (kv8_reference): any finite scale >= 0 is allowed."""
import math

import numpy as np
import pytest
import torch

import hcp_ring_amd as H
import kv8_reference as R
from test_kv8_decode import SCORE, compare, inputs, reference, tolerance

# One wave; waves that meet in LDS; lone waves over a row of sequences, two padded; four heads a
# workgroup; four and sixteen waves that meet, over a row of sequences.
SPLITS = {
    # batch, Hq, Hkv, D, tokens of the longest sequence
    "one_wave": (2, 4, 1, 64, 30),
    "direct": (3, 8, 2, 128, 200),
    "lone": (2, 8, 2, 128, 3000),
    "padded": (6, 16, 2, 96, 2000),
    "heads": (3, 8, 8, 64, 4000),
    "meet4": (3, 8, 2, 128, 4000),
    "meet16": (1, 16, 1, 128, 30000),
}


def setup(seed, split, bs, fmt):
    b, hq, hkv, d, tokens = SPLITS[split]
    return inputs(seed, b, hq, hkv, d, bs, "bf16", fmt, tokens)


def decode(lens, codes, scales, fmt, tables, qt):
    pool, sc = R.to_device(codes, scales, fmt)
    return H.kv8_decode_partial(qt, pool, sc, torch.from_numpy(tables[0]).cuda(), 0, int(lens[0].max()),
                                seq_lens=torch.from_numpy(lens[0].astype(np.int32)).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 32])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("split", SPLITS)
def test_v_scales_of_zero(gpu, split, fmt, bs):
    # everywhere: rows of 0; over each sequence's first tokens and in every second stretch of 64
    # after them, so that waves begin with, meet and end in them: those tokens count as V = 0
    r, lens, codes, scales, tables, qt, q = setup(50, split, bs, fmt)
    none = scales.copy()
    none[1] = 0
    want, want_lse = reference(q, codes, none, fmt, tables, lens)
    o, lse = decode(lens, codes, none, fmt, tables, qt)
    assert (o == 0).all()
    compare(o, lse, want, want_lse, 0.0)
    some = scales.copy()
    some[1, tables[0][:, np.arange(tables[0].shape[1]) * bs // 64 % 2 == 0]] = 0
    want, want_lse = reference(q, codes, some, fmt, tables, lens)
    o, lse = decode(lens, codes, some, fmt, tables, qt)
    compare(o, lse, want, want_lse, R.LARGEST[fmt] * scales.max())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("split", SPLITS)
def test_v_scales_down_to_the_smallest(gpu, split, fmt):
    # V scales of 2^-110 to 2^-126, beside 0; the rows as near to the largest V as ordinary ones,
    # but for a result's own rounding at the smallest normal number
    r, lens, codes, scales, tables, qt, q = setup(51, split, 16, fmt)
    scales[1] = 2.0 ** r.integers(-126, -109, scales[1].shape)
    scales[1, tables[0][:, 2::5]] = 0
    want, want_lse = reference(q, codes, scales, fmt, tables, lens)
    o, lse = decode(lens, codes, scales, fmt, tables, qt)
    err = np.abs(o.double().cpu().numpy() - want).max()
    assert err <= tolerance(R.LARGEST[fmt] * scales[1].max(), torch.float32) + 2.0 ** -126
    assert np.abs(lse.double().cpu().numpy() - want_lse)[np.isfinite(want_lse)].max() <= 2 * SCORE + 2.0 ** -16


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_v_scales_fall_as_scores_rise(gpu, fmt):
    # later tokens score up to 100 higher and have V scales down to 0: each step's maximum rises
    # while nothing of V follows
    b, tokens, bs, d = 2, 160, 16, 128
    _, lens, codes, scales, tables, qt, q = inputs(52, b, 4, 1, d, bs, "bf16", fmt, tokens)
    lens[0][:] = tokens
    codes[0] = 0x38 if fmt == "e4m3" else 1  # 1: scores are q's sum times the scale
    q = np.ones_like(q)
    for e in range(tokens // bs):
        scales[0, tables[0][:, e]] = 10.0 * e / math.sqrt(d)
        scales[1, tables[0][:, e]] = 2.0 ** (-12.0 * e) if e < 8 else 0
    want, want_lse = reference(q, codes, scales, fmt, tables, lens)
    o, lse = decode(lens, codes, scales, fmt, tables, torch.ones_like(qt))
    err = np.abs(o.double().cpu().numpy() - want).max(axis=(1, 2))
    # |S| <= 100 here: SCORE counts up to 2^6
    assert (err <= np.abs(want).max(axis=(1, 2)) * (4 * SCORE + 2.0 ** -18)).all()
    assert np.abs(lse.double().cpu().numpy() - want_lse).max() <= 4 * SCORE


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("tokens", [1, 5, 16, 33, 100, 3000])
def test_fresh_pool(gpu, tokens, fmt):
    # nothing appended yet (a warm-up): equal scores, V = 0
    pool, sc = H.kv8_pool(2 * 200, 16, 2, 64, R.TORCH[fmt])
    table = torch.arange(400, dtype=torch.int32, device="cuda").view(2, 200)
    q = torch.randn(2, 8, 64, device="cuda", dtype=torch.bfloat16)
    lens = torch.tensor([tokens, max(tokens - 3, 0)], dtype=torch.int32, device="cuda")
    for out, lse in (H.kv8_decode_partial(q, pool, sc, table, 0, tokens, seq_lens=lens),
                     H.kv8_decode_ring_replay(q, pool, sc, [(table, lens, tokens), (table, lens, tokens)], 0)):
        assert (out == 0).all()
        n = lens.double()[:, None] * (1 if out.dtype == torch.float32 else 2)
        want = torch.log(n).expand(2, 8)
        assert torch.equal(torch.isneginf(lse), n.expand(2, 8) == 0)
        fin = torch.isfinite(want)
        assert (lse.double()[fin] - want[fin]).abs().max() <= 2.0 ** -16


FAR = [  # log2 of the weight and of the V scale, of the tokens of even blocks and of odd ones
    (25, -20, -35, 20),
    (-35, 20, 25, -20),
    (0, -100, -110, 100),  # the small weights carry the row
    (-118, 100, 0, -100),  # so that 2^14 over their sum is past fp32 with their scale
    (0, -100, -300, 60),   # and here they are nothing
    (0, 0, -200, 120),
    (0, -126, -60, 0),
    (0, 60, 3, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("tokens", [32, 100, 3000])
@pytest.mark.parametrize("far", FAR, ids=str)
def test_neighbouring_blocks_of_very_different_scales(gpu, far, tokens, fmt):
    # two blocks of one step: what a token weighs is its own softmax weight times its own scale
    b, bs, d = 2, 16, 128
    _, lens, codes, scales, tables, qt, q = inputs(53, b, 4, 1, d, bs, "bf16", fmt, tokens)
    lens[0][:] = [tokens, tokens - 16]
    one = 0x38 if fmt == "e4m3" else 1  # K rows of one value: a score is its sign times the scale
    for e in range(tables[0].shape[1]):
        s, v = far[2 * (e % 2): 2 * (e % 2) + 2]
        codes[0, tables[0][:, e]] = one if s >= 0 else (one | 0x80 if fmt == "e4m3" else 0xff)
        scales[0, tables[0][:, e]] = abs(s) * math.log(2.0) / math.sqrt(d)
        scales[1, tables[0][:, e]] = 2.0 ** v
    want, want_lse = reference(np.ones_like(q), codes, scales, fmt, tables, lens)
    o, lse = decode(lens, codes, scales, fmt, tables, torch.ones_like(qt))
    err = np.abs(o.double().cpu().numpy() - want).max(axis=(1, 2))
    # |S| <= 300 ln 2 is rounded to 2^-24 of it by scale and product and by each of 128 sums at most:
    # 2^-24 * 208 * (2 * 136) < 2^-8 at the very worst, 2^-12.4 with sqrt(136); against a row's own largest
    assert (err <= np.abs(want).max(axis=(1, 2)) * 2.0 ** -12 + 2.0 ** -126).all(), err / np.abs(want).max(axis=(1, 2))
    assert np.abs(lse.double().cpu().numpy() - want_lse).max() <= 2.0 ** -12


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("split", SPLITS)
def test_scores_of_the_largest_size(gpu, split, sign, fmt):
    # K scales of 2^20 and scores all negative or all positive, to 2^23.5: one token of each sequence has all the weight
    r, lens, codes, scales, tables, qt, q = setup(54, split, 16, fmt)
    scales[0] = 2.0 ** 20
    one = (0x38 if sign > 0 else 0xb8) if fmt == "e4m3" else (1 if sign > 0 else 0xff)
    codes[0] = one if sign < 0 else 0  # a score is the scale times sum(code) / sqrt(D)
    b, hq, hkv, d, tokens = SPLITS[split]
    for i in range(b):
        if lens[0][i]:
            best = int(r.integers(lens[0][i]))
            codes[0, tables[0][i, best // 16], best % 16, :, ::2] = one if sign > 0 else 0
    want, want_lse = reference(np.ones_like(q), codes, scales, fmt, tables, lens)
    o, lse = decode(lens, codes, scales, fmt, tables, torch.ones_like(qt))
    err = np.abs(o.double().cpu().numpy() - want).max()
    assert err <= tolerance(R.LARGEST[fmt] * scales[1].max(), torch.float32)
    got = lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(got), np.isneginf(want_lse))
    fin = np.isfinite(want_lse)
    # whole products and sums; scale, its log2 e, ln 2 and the products with them round, and the largest score
    # against its own fp32 maximum: 8 roundings
    assert (np.abs(got - want_lse)[fin] <= np.abs(want_lse[fin]) * 8 * 2.0 ** -24).all()
