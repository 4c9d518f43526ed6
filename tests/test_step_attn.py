"""Attention of a serving step over the paged cache against softmax(q k^T scale) v in 64 bits,
sequence by sequence.

Bound of an output element.  A score is a sum of D exact products in fp32: off by at most
(D + 8) 2^-24 sum |q_d k_d| scale =: s (the scale and the subtraction of the maximum among the
8), so a weight by a factor within e^s (1 + 2^-21) (the exponential is within 2^-22).  A weight
enters the product with V rounded to the 16-bit type (half a step: eps / 2 of it) in one term,
two or three: r = (eps / 2)^terms.  Normalised sums of weights and |v| then move by at most
(2 s + 2^-20 + r) A with A = sum w |v|, parts of a row that are joined by another 2^-17 A (their
LSE, rounded to 2^-24 of its size below 32, its difference and the exponential of it), and the
output rounds once: eps(out) / 2 |o|.  The LSE moves by s, 2^-20 and its own rounding."""
import ctypes
import math

import numpy as np
import pytest
import torch

import hcp_ring_amd as H

I32 = torch.int32
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


class Step:
    """A step: new[b] tokens of sequence b, lens[b] tokens of its own with them, a prefix each or -1."""

    def __init__(self, new, lens, hq=8, hkv=2, d=128, bs=16, ids=None, plens=(), dtype="bf16", causal=True, seed=0, spare=3,
                 extra=0, big=1.0):
        self.new, self.lens, self.plens = np.asarray(new), np.asarray(lens), np.asarray(plens, dtype=np.int64)
        self.ids = np.full(len(new), -1) if ids is None else np.asarray(ids)
        self.hq, self.hkv, self.d, self.bs, self.causal = hq, hkv, d, bs, causal
        g = torch.Generator().manual_seed(seed)
        self.tokens = int(self.new.sum()) + extra
        self.starts = np.concatenate([[0], np.cumsum(self.new)])
        used = np.concatenate([-(-self.lens // bs), -(-self.plens // bs)]).astype(np.int64)
        total = int(used.sum()) + spare
        perm = torch.randperm(total, generator=g).numpy()
        # what no sequence holds is NaN: rows past a length, spare blocks
        self.pool = (torch.randn(2, total, bs, hkv, d, generator=g) * big).to(DT[dtype])
        free = np.ones((total, bs), bool)
        first = np.concatenate([[0], np.cumsum(used)])
        width, pwidth = max(1, int(used[: len(new)].max()) + 1), max(1, int(used[len(new):].max()) + 1) if len(self.plens) else 1
        self.tables, self.ptables = np.full((len(new), width), -7), np.full((len(self.plens), pwidth), -7)
        for i, n in enumerate(list(self.lens) + list(self.plens)):
            blocks = perm[first[i]: first[i + 1]]
            (self.tables[i] if i < len(new) else self.ptables[i - len(new)])[: len(blocks)] = blocks
            for t in range(int(n)):
                free[blocks[t // bs], t % bs] = False
        self.pool[:, torch.from_numpy(free)] = float("nan")
        self.q = torch.randn(self.tokens, hq, d, generator=g).to(DT[dtype])

    def device(self, dev="cuda"):
        t = lambda x: torch.tensor(np.asarray(x), dtype=I32, device=dev)  # noqa: E731
        p = len(self.plens) > 0
        return dict(q=self.q.to(dev).permute(1, 0, 2), pool=self.pool.to(dev), tables=t(self.tables), starts=t(self.starts),
                    lens=t(self.lens), ptables=t(self.ptables) if p else None, ids=t(self.ids) if p else None,
                    plens=t(self.plens) if p else None)

    def run(self, out=None, lse=None, x=None, **kw):
        x = x or self.device()
        plan = H.step_attn_plan(x["q"], x["pool"], x["tables"], x["starts"], x["lens"], x["ptables"], x["ids"], x["plens"],
                                causal=self.causal)
        return H.step_attn(x["q"], x["pool"], x["tables"], plan, x["ptables"], causal=self.causal, out=out, lse=lse, **kw)

    def rows(self, plane, table, n):
        return self.pool[plane, torch.from_numpy(table[: -(-n // self.bs)])].flatten(0, 1)[:n]

    def reference(self):
        """(o, A, lse, s) in fp64: o and A [Hq, T, D], lse and s [Hq, T]; rows of no sequence NaN."""
        shape = (self.hq, self.tokens, self.d)
        o, mag, lse, s = (torch.full(shape[: 2 + i], float("nan"), dtype=torch.float64) for i in (1, 1, 0, 0))
        rep = self.hq // self.hkv
        for b, n in enumerate(self.new):
            if n == 0:
                continue
            k, v = (torch.cat([self.rows(p, self.ptables[self.ids[b]], int(self.plens[self.ids[b]])) if self.ids[b] >= 0
                               else self.pool[p, 0, :0], self.rows(p, self.tables[b], int(self.lens[b]))]).double().cuda() for p in (0, 1))
            shared = k.shape[0] - int(self.lens[b])
            at = slice(int(self.starts[b]), int(self.starts[b]) + int(n))
            q = self.q[at].double().cuda()
            i, j = torch.arange(int(n)).cuda()[:, None], torch.arange(k.shape[0]).cuda()[None, :]
            seen = (j < shared) | (j - shared <= int(self.lens[b]) - int(n) + i) if self.causal else torch.ones(int(n), k.shape[0], dtype=torch.bool).cuda()
            for h in range(self.hq):
                kk, vv = k[:, h // rep], v[:, h // rep]
                x = (q[:, h] @ kk.T / math.sqrt(self.d)).masked_fill(~seen, -math.inf)
                lse[h, at] = torch.logsumexp(x, 1).cpu()
                w = torch.exp(x - torch.logsumexp(x, 1, keepdim=True)).nan_to_num(0.0)
                o[h, at], mag[h, at] = (w @ vv).cpu(), (w @ vv.abs()).cpu()
                size = (q[:, h].abs() @ kk.abs().T / math.sqrt(self.d)).masked_fill(~seen, 0.0)
                s[h, at] = (size.amax(1).cpu() if size.shape[1] else 0.0) * (self.d + 8) * 2.0 ** -24
        return o, mag, lse, s


def check(step, out, lse, ref=None, terms=1, rows=slice(None)):
    o, mag, want, s = (t[:, rows] for t in (ref or step.reference()))
    out, lse = out[:, rows], lse[:, rows]
    live = ~torch.isnan(want)
    half = torch.finfo(step.q.dtype).eps / 2
    r = half ** terms
    got = out.double().cpu()
    bound = (2 * s[..., None] + 2.0 ** -20 + r + 2.0 ** -17) * mag + torch.finfo(out.dtype).eps / 2 * o.abs() + 1e-30
    if out.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    err = (got - o).abs()
    worst = (err / bound)[live]
    assert bool((worst <= 1).all()), float(worst.nan_to_num(1e30).max())
    l = lse.double().cpu()
    empty = live & (want == -math.inf)
    assert bool((l[empty] == -math.inf).all()) and bool((got[empty] == 0).all())
    some = live & ~empty
    assert bool(((l - want).abs()[some] <= (s + 2.0 ** -19 * (1 + want.abs()))[some]).all())
    assert H.fetch_device_errors() == 0


HEADS = [(32, 8, 128), (16, 2, 128), (14, 2, 64), (8, 1, 96), (4, 4, 32), (24, 2, 72), (6, 2, 8), (40, 1, 128), (3, 3, 112)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", HEADS)
def test_decode_of_ragged_sequences(gpu, heads, dtype):
    hq, hkv, d = heads
    step = Step([1] * 7, [1, 130, 16, 517, 33, 2, 1000], hq, hkv, d, dtype=dtype, seed=1)
    check(step, *step.run())
    out = torch.empty(hq, 7, d, dtype=torch.float32, device="cuda")
    check(step, *step.run(out=out), terms=2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("causal", [True, False])
def test_chunks_and_single_tokens_together(gpu, heads, dtype, causal):
    hq, hkv, d = heads
    step = Step([1, 70, 0, 5, 300, 1], [40, 70, 9, 133, 450, 1], hq, hkv, d, bs=32, dtype=dtype, seed=2, causal=causal)
    check(step, *step.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", HEADS)
def test_shared_prefixes(gpu, heads, dtype):
    """Prefixes behind many sequences, behind one, behind a long run of tokens, and empty."""
    hq, hkv, d = heads
    ids = [0, 1, 0, -1, 2, 0, 3, 0, 0, 4, 4, 0]
    step = Step([1, 1, 2, 1, 1, 1, 1, 40, 1, 1, 1, 0], [1, 20, 3, 70, 5, 33, 9, 60, 64, 18, 1, 4], hq, hkv, d, ids=ids,
                plens=[517, 64, 31, 0, 16], dtype=dtype, seed=3)
    check(step, *step.run())


@pytest.mark.gpu
@pytest.mark.parametrize("ctx", [1000, 4500, 9000, 40000])
@pytest.mark.parametrize("heads", [(8, 1, 128), (4, 2, 64), (12, 3, 96)])
def test_one_sequence_over_the_whole_gpu(gpu, heads, ctx):
    """A few units cut among all workgroups: up to 256 parts of a row are joined, of a number that
    is no multiple of what a lane loads at a time."""
    hq, hkv, d = heads
    for new in (1, 2, 40):
        step = Step([new], [ctx + new], hq, hkv, d, seed=ctx)
        check(step, *step.run())


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [(32, 8, 128), (16, 2, 128), (14, 2, 64), (8, 1, 96), (24, 6, 72), (12, 4, 40)])
def test_long_chunks(gpu, heads, dtype, causal):
    """Steps of enough work for tiles of 256 rows: prompt chunks that end inside tiles, behind
    cached tokens, a prefix of their own and one that many decoding sequences share."""
    hq, hkv, d = heads
    new = [1] * 40 + [1500, 700, 33] + [1] * 60
    r = np.random.default_rng(15)
    lens = np.asarray(new) + r.integers(0, 300, len(new))
    lens[40:43] += [4000, 2111, 0]
    ids = [0] * 30 + [-1] * 10 + [1, 0, -1] + [0] * 60
    step = Step(new, lens, hq, hkv, d, ids=ids, plens=[1111, 300], dtype=dtype, seed=15, causal=causal)
    ref = step.reference()
    check(step, *step.run(), ref=ref)
    out = torch.empty(hq, step.tokens, d, dtype=torch.float32, device="cuda")
    check(step, *step.run(out=out), ref=ref, terms=2)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64), (8, 1, 96)])
def test_fp32_rows_carry_small_weights(gpu, heads):
    """One key far above thousands whose weights are e^-17 each: a tenth of a thousandth of the sum,
    below what one fp16 or bf16 term of a weight next to it holds."""
    hq, hkv, d = heads
    for dtype in ("bf16", "f16"):
        step = Step([1, 5, 130], [9000, 4000, 6000], hq, hkv, d, dtype=dtype, seed=7)
        step.q[:] = 1.0
        k = step.pool[0]
        k[~torch.isnan(k)] = 0.0
        peak = 17.0 / math.sqrt(d)  # a score of 17 where every dim of the key is this
        for b in range(3):
            step.pool[0, step.tables[b, 0], 0] = peak
        out = torch.empty(hq, step.tokens, d, dtype=torch.float32, device="cuda")
        check(step, *step.run(out=out), terms=2)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_lengths_of_nothing_and_tokens_not_served(gpu, causal):
    """Sequences without tokens, without keys, with fewer tokens held than new ones (a step that did
    not serve them), behind a prefix or not; rows past the last sequence stay as they are."""
    step = Step([0, 1, 4, 3, 0, 2, 40], [5, 0, 2, 0, 0, 1, 7], 8, 2, 128, ids=[-1, -1, 0, 0, 0, 0, -1], plens=[37], seed=4,
                causal=causal, extra=9)
    out = torch.full((8, step.tokens, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((8, step.tokens), 5.0, device="cuda")
    check(step, *step.run(out=out, lse=lse))
    assert bool((out[:, -9:] == 5.0).all()) and bool((lse[:, -9:] == 5.0).all())


@pytest.mark.gpu
def test_new_tokens_of_every_count(gpu):
    """Every number of new tokens from 1 to 70 (tiles that end anywhere), over two prefixes."""
    n = list(range(1, 71))
    step = Step(n, [i + (i * 37) % 90 for i in n], 8, 2, 64, ids=[i % 3 - 1 for i in n], plens=[100, 259], seed=5)
    check(step, *step.run())


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 48, 80, 128, 1024])
def test_block_sizes(gpu, bs):
    step = Step([1, 3, 200, 1, 1], [1, 77, 1333, 600, 16], 16, 2, 128, bs=bs, ids=[0, 0, 0, 0, -1], plens=[1029], seed=6)
    check(step, *step.run())


@pytest.mark.gpu
def test_views_of_any_strides(gpu):
    """Head-major q and out, rows apart, tables that are parts of wider ones."""
    step = Step([1, 50, 2], [70, 90, 300], 8, 2, 96, ids=[0, -1, 0], plens=[64], seed=8)
    x = step.device()
    want = step.run(x=x)
    q = torch.zeros(8, step.tokens + 3, 128, dtype=torch.bfloat16, device="cuda")[:, 1: step.tokens + 1, 16: 112]
    q.copy_(x["q"])
    wide = torch.full((3, x["tables"].shape[1] + 5), -9, dtype=I32, device="cuda")
    wide[:, : x["tables"].shape[1]] = x["tables"]
    out = torch.full((8, step.tokens, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    got = step.run(x=dict(x, q=q, tables=wide[:, : x["tables"].shape[1]]), out=out[..., :96])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert bool((out[..., 96:] == 3.0).all())
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
def test_many_sequences_and_prefixes(gpu):
    """The most sequences and prefixes that a step takes, in no order."""
    r = np.random.default_rng(9)
    b, p = 4096, 1024
    new = (r.random(b) < 0.3).astype(int)
    step = Step(new, r.integers(0, 20, b) + new, 2, 1, 32, ids=r.integers(-1, p, b), plens=r.integers(0, 40, p), seed=9)
    check(step, *step.run())


@pytest.mark.gpu
def test_blocks_past_four_gigabytes(gpu):
    """Blocks whose bytes lie past 2^32 in either plane."""
    hq, hkv, d, bs = 8, 8, 128, 16
    step = Step([1, 3, 140], [40, 33, 170], hq, hkv, d, bs=bs, ids=[0, 0, -1], plens=[50], seed=10, spare=0)
    small, n = step.pool, step.pool.shape[1]
    blocks = (9 << 30) // (2 * bs * hkv * d * 2)  # 4.5 GiB a plane
    big = torch.zeros(2, blocks, bs, hkv, d, dtype=torch.bfloat16, device="cuda")
    x = step.device()
    big[:, blocks - n:] = small.cuda()
    move = lambda t: torch.where(t >= 0, t + blocks - n, t).to(I32)  # noqa: E731
    got = step.run(x=dict(x, pool=big, tables=move(x["tables"]), ptables=move(x["ptables"])))
    check(step, *got)


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_with_their_sequence(gpu):
    step = Step([1, 40, 1, 3], [90, 70, 5, 30], 8, 2, 128, ids=[0, -1, 0, -1], plens=[48], seed=11)
    x = step.device()
    want, want_lse = (t.clone() for t in step.run(x=x))
    first, last = int(step.tables[1, 0]), int(step.tables[1, 60 // 16])
    x["pool"][0, last, 60 % 16], x["pool"][1, first, 3] = float("nan"), float("inf")  # a key of tokens 30 .., a value of all
    out, lse = step.run(x=x)
    for b, at in ((0, slice(0, 1)), (2, slice(41, 42)), (3, slice(42, 45))):
        assert torch.equal(out[:, at], want[:, at]) and torch.equal(lse[:, at], want_lse[:, at])
    # own key 60 of sequence 1 is seen by its tokens 30 .. 39; its K reaches no other's LSE
    assert torch.equal(lse[:, 1: 31], want_lse[:, 1: 31]) and bool(lse[:, 31: 41].isnan().all())
    assert not bool(out[:, 1: 41].isfinite().all(-1).any())


@pytest.mark.gpu
def test_a_nan_key_in_a_long_chunk_is_not_lost(gpu):
    """Tiles of 256 rows, some of them joined of parts: the rows that see the key are NaN, and their
    LSE too, the ones before it as they were.  The 8 tokens of a wave take their maxima anew
    together, so those beside token 700 may round otherwise: they stay within the bounds."""
    step = Step([1500, 1], [5500, 40], 32, 8, 128, seed=16)
    ref = step.reference()
    x = step.device()
    want, want_lse = (t.clone() for t in step.run(x=x))
    x["pool"][0, int(step.tables[0, 4700 // 16]), 4700 % 16] = float("nan")  # seen by tokens 700 ..
    out, lse = step.run(x=x)
    assert torch.equal(lse[:, :696], want_lse[:, :696]) and torch.equal(out[:, :696], want[:, :696])
    check(step, out, lse, ref=ref, rows=slice(0, 700))
    assert bool(lse[:, 700: 1500].isnan().all()) and bool(out[:, 700: 1500].isnan().all())
    assert torch.equal(out[:, 1500:], want[:, 1500:]) and torch.equal(lse[:, 1500:], want_lse[:, 1500:])


@pytest.mark.gpu
@pytest.mark.parametrize("first", [1, 200, 600])
def test_a_short_sequence_before_long_ones(gpu, first):
    """The first unit of the work is short against a worker's share, and is still done."""
    for new, lens in (([1] * 24, [first] + [12000] * 23), ([1] * 24, [12000] * 23 + [first])):
        step = Step(new, lens, 16, 8, 64, seed=17)
        out = torch.full((16, 24, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
        check(step, *step.run(out=out))
    step = Step([40, 3000], [40 + first, 6000], 16, 8, 64, seed=18)
    out = torch.full((16, 3040, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    check(step, *step.run(out=out))


@pytest.mark.gpu
def test_bad_ids_lengths_and_plans_set_their_flags(gpu):
    step = Step([1, 40, 1], [90, 70, 5], 8, 2, 128, ids=[0, -1, 0], plens=[48], seed=12)
    x = step.device()
    # a block id outside the pool: its tokens are rows of zeros
    for bad in (-1, x["pool"].shape[1], 2 ** 30):
        y = dict(x, tables=x["tables"].clone())
        y["tables"][1, 1] = bad
        out, lse = step.run(x=y)
        assert H.fetch_device_errors() == 1
        zero = Step([1, 40, 1], [90, 70, 5], 8, 2, 128, ids=[0, -1, 0], plens=[48], seed=12)
        zero.pool[:, zero.tables[1, 1]] = 0.0
        check(zero, out, lse)
    # lengths and ids that do not fit
    t = lambda v: torch.tensor(v, dtype=I32, device="cuda")  # noqa: E731
    for kw in (dict(lens=t([90, -70, 5])), dict(lens=t([90, 1 << 20, 5])), dict(ids=t([0, 1, 0])), dict(ids=t([0, -2, 0])),
               dict(plens=t([-1])), dict(plens=t([1 << 30])), dict(starts=t([0, 1, 0, 42])), dict(starts=t([-5, 1, 41, 42]))):
        y = dict(x, **kw)
        y["pool"] = torch.nan_to_num(x["pool"], nan=0.0)
        y["tables"], y["ptables"] = x["tables"].clamp(min=0), x["ptables"].clamp(min=0)
        step.run(x=y)
        assert H.fetch_device_errors() == 8, list(kw)
    # a plan of another shape
    plan = H.step_attn_plan(x["q"], x["pool"], x["tables"], x["starts"], x["lens"], x["ptables"], x["ids"], x["plens"])
    out = torch.full((8, 42, 128), 2.0, dtype=torch.bfloat16, device="cuda")
    H.step_attn(x["q"], x["pool"], x["tables"], plan, x["ptables"], causal=False, out=out)
    assert H.fetch_device_errors() == 8 and bool((out == 2.0).all())
    H.step_attn(x["q"], x["pool"], x["tables"], torch.zeros_like(plan), x["ptables"], out=out)
    assert H.fetch_device_errors() == 8 and bool((out == 2.0).all())
    H.step_attn(x["q"][:, :41], x["pool"], x["tables"], plan, x["ptables"], out=out[:, :41])
    assert H.fetch_device_errors() == 8 and bool((out == 2.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[0, 200, 0, 200, 0, 200, 0, 200, 0], [0, 30, 10, 200, 199, 200, -4, 200, 200],
                                    [0, 3, 0, 4, 1, 5, 2, 200, 0]])
@pytest.mark.parametrize("prefix", [False, True])
def test_starts_that_fall_give_every_token_to_one_sequence(gpu, starts, prefix):
    """What earlier sequences have is left out of later ones: the plan has room for every token once."""
    new = [0 if t0 < 0 or t1 < t0 else max(t1 - max(starts[: b + 1]), 0) for b, (t0, t1) in enumerate(zip(starts, starts[1:]))]
    assert sum(new) == 200
    step = Step(new, [260 + 7 * b for b in range(8)], 8, 2, 64, ids=[b // 2 % 2 for b in range(8)] if prefix else None,
                plens=[40, 300] if prefix else (), seed=17)
    x = step.device()
    x["starts"] = torch.tensor(starts, dtype=I32, device="cuda")
    size = H.step_attn_plan_size(x["q"], x["pool"], x["tables"], x["ptables"])
    room = torch.full((size + (1 << 20),), 90, dtype=torch.uint8, device="cuda")
    plan = H.step_attn_plan(x["q"], x["pool"], x["tables"], x["starts"], x["lens"], x["ptables"], x["ids"], x["plens"], plan=room[:size])
    assert H.fetch_device_errors() == 8 and bool((room[size:] == 90).all())
    check(step, *H.step_attn(x["q"], x["pool"], x["tables"], plan, x["ptables"]))


@pytest.mark.gpu
def test_two_calls_at_once_share_a_plan(gpu):
    """One plan, two streams, each with a workspace of its own."""
    step = Step([1, 1, 300, 5], [9000, 700, 2000, 40], 16, 2, 128, ids=[0, 0, -1, 0], plens=[3000], seed=13)
    x = step.device()
    plan = H.step_attn_plan(x["q"], x["pool"], x["tables"], x["starts"], x["lens"], x["ptables"], x["ids"], x["plens"])
    want = H.step_attn(x["q"], x["pool"], x["tables"], plan, x["ptables"])
    q2 = torch.flip(x["q"], (2,)).contiguous()
    want2 = H.step_attn(q2, x["pool"], x["tables"], plan, x["ptables"])
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        got = H.step_attn(x["q"], x["pool"], x["tables"], plan, x["ptables"], stream=a)
        got2 = H.step_attn(q2, x["pool"], x["tables"], plan, x["ptables"], stream=b)
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got + got2, want + want2))


@pytest.mark.gpu
def test_a_captured_step_follows_the_lengths(gpu):
    """Step plan, norms with append, attention plan and attention in one graph, replayed as the
    sequences grow behind two prefixes; every replay against the same calls made eagerly and
    against 64 bits.  The prefixes' blocks lie outside the free ones; the sequences' rows hold their
    own tokens only."""
    hq, hkv, d, bs, b, cap, nb = 8, 2, 64, 16, 5, 40, 64
    g = torch.Generator().manual_seed(14)
    t = lambda v: torch.tensor(v, dtype=I32, device="cuda")  # noqa: E731
    plens, ids = t([70, 33]), t([0, 1, 0, -1, 0])
    ptables = torch.full((2, 5), -1, dtype=I32, device="cuda")
    ptables[0] = t([3, 60, 7, 1, 22])
    ptables[1, :3] = t([9, 2, 50])
    taken = set(ptables.flatten().tolist())
    free_ids = [i for i in range(nb) if i not in taken]
    table = H.rope_table(d, 400)
    wq, wk = (1 + 0.1 * torch.randn(2, d, generator=g)).to(torch.bfloat16).cuda()
    pool0 = torch.randn(2, nb, bs, hkv, d, generator=g).to(torch.bfloat16).cuda()
    shift = torch.where(ids >= 0, plens[ids.clamp(min=0).long()], 0)

    def state():
        return dict(lens=t([0] * b), tables=torch.full((b, 8), -1, dtype=I32, device="cuda"), free=t(free_ids + [-1] * (nb - len(free_ids))),
                    count=t([len(free_ids)]), pool=pool0.clone(), new=t([0] * b), x=torch.zeros(cap, hq + 2 * hkv, d, dtype=torch.bfloat16,
                                                                                                device="cuda"),
                    out=torch.zeros(cap, hq, d, dtype=torch.bfloat16, device="cuda").permute(1, 0, 2), lse=torch.zeros(hq, cap, device="cuda"),
                    seq=torch.zeros(cap, dtype=torch.int64, device="cuda"))

    def step(s):
        slots, pos, starts, _, _ = H.kv_plan_step(s["lens"], s["new"], s["tables"], s["free"], s["count"], bs, capacity=cap,
                                                  seq_lens_out=s["lens"], free_count_out=s["count"])
        q, k, v = (s["x"][:, i:j].permute(1, 0, 2) for i, j in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
        at = pos + shift[s["seq"]]  # positions behind the prefixes
        qn = H.qk_norm_rope_append(q, k, v, wq, wk, s["pool"], slots, at, table)
        plan = H.step_attn_plan(qn, s["pool"], s["tables"], starts, s["lens"], ptables, ids, plens)
        H.step_attn(qn, s["pool"], s["tables"], plan, ptables, out=s["out"], lse=s["lse"])
        return qn, starts

    steps = [[7, 3, 1, 12, 0], [1, 1, 1, 1, 9], [1, 1, 1, 1, 1], [4, 1, 20, 1, 1], [1, 1, 1, 1, 1]]
    eager, graphed = state(), state()
    step(state())  # warm: loads the kernels
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qn_g, _ = step(graphed)
    for name, v in state().items():
        graphed[name].copy_(v)
    for i, new in enumerate(steps):
        x = torch.randn(cap, hq + 2 * hkv, d, generator=g).to(torch.bfloat16).cuda()
        seq = torch.tensor(np.repeat(np.arange(b), new).tolist() + [0] * (cap - sum(new))).cuda()
        for s in (eager, graphed):
            s["x"].copy_(x)
            s["seq"].copy_(seq)
            s["new"].copy_(t(new))
        qn, _ = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        n = sum(new)
        for name in ("lens", "tables", "free", "count", "pool"):
            assert torch.equal(eager[name], graphed[name]), (i, name)
        assert torch.equal(eager["out"][:, :n], graphed["out"][:, :n]) and torch.equal(eager["lse"][:, :n], graphed["lse"][:, :n])
        assert torch.equal(qn[:, :n], qn_g[:, :n])
        ref = Step(new, eager["lens"].tolist(), hq, hkv, d, ids=ids.tolist(), plens=plens.tolist())
        ref.pool, ref.q = eager["pool"].cpu(), qn[:, :n].permute(1, 0, 2).cpu()
        ref.tables, ref.ptables = eager["tables"].cpu().numpy(), ptables.cpu().numpy()
        check(ref, eager["out"][:, :n], eager["lse"][:, :n])


# ---------------------------------------------------------------------------------
# refusals (no GPU)
# ---------------------------------------------------------------------------------
AT = 1 << 20
DESC = dict(dtype=2, batch=3, num_q_heads=8, num_kv_heads=2, head_dim=128, reserved0=0, t0=0, t1=0, table_stride=6, table_len=5, scale=0.1)
POOL = (AT, 9, 16, 2, 128, 2)


def _call(fn, null=False, pool=POOL, tokens=4, causal=1, prefixes=0, shard=(AT, 3, 3, AT, 0), ids=AT, plan=AT, plan_bytes=1 << 30, q=AT,
          out=AT, out_dtype=2, stride=1024, ostride=1024, tables=AT, ws=AT, ws_bytes=1 << 40, starts=AT, lens=AT, **kw):
    """Either entry with addresses that are never read: a call that is not refused would need a GPU."""
    L, d = H.lib(), None if null else ctypes.byref(H.DecodeDesc(**dict(DESC, **kw)))
    p = None if pool is None else ctypes.byref(H.PagedPool(*pool))
    sh = None if shard is None else ctypes.byref(H.DecodeShard(*shard))
    if fn == "plan":
        return L.hcp_step_attn_plan(d, p, tokens, causal, starts, lens, prefixes, sh, ids, plan, plan_bytes, None)
    return L.hcp_step_attn(d, p, tokens, causal, H.View(q, 128, stride), tables, prefixes, sh, plan, plan_bytes, out_dtype,
                           H.View(out, 128, ostride), AT, ws, ws_bytes, None)


BAD = [dict(null=True), dict(dtype=3), dict(batch=0), dict(batch=4097), dict(num_q_heads=7), dict(num_q_heads=0), dict(num_kv_heads=0),
       dict(num_q_heads=514), dict(head_dim=136), dict(head_dim=124), dict(head_dim=64), dict(table_len=0), dict(table_stride=4),
       dict(table_len=1 << 28, table_stride=1 << 28), dict(tokens=-1), dict(tokens=1 << 29), dict(causal=2), dict(prefixes=-1), dict(prefixes=1025),
       dict(prefixes=2, shard=None), dict(prefixes=2, shard=(AT, 2, 3, AT, 0)), dict(prefixes=2, shard=(AT, 3, 0, AT, 0)),
       dict(pool=None), dict(pool=(0, 9, 16, 2, 128, 2)), dict(pool=(AT + 8, 9, 16, 2, 128, 2)), dict(pool=(AT, 0, 16, 2, 128, 2)),
       dict(pool=(AT, 9, 24, 2, 128, 2)), dict(pool=(AT, 9, 16, 4, 128, 2)), dict(pool=(AT, 9, 16, 2, 128, 4)),
       dict(pool=(AT, 9, 1 << 21, 2, 128, 2)), dict(plan=None), dict(plan=AT + 16), dict(plan_bytes=100)]


@pytest.mark.parametrize("fn", ["plan", "attn"])
@pytest.mark.parametrize("kw", BAD)
def test_bad_arguments_are_refused(hcp, fn, kw):
    assert _call(fn, **kw) == -6 and H.last_error()


@pytest.mark.parametrize("kw", [dict(starts=None), dict(lens=None), dict(prefixes=2, shard=(AT, 3, 3, None, 0)), dict(prefixes=2, ids=None)])
def test_a_plan_refuses_null_lengths(hcp, kw):
    assert _call("plan", **kw) == -6


@pytest.mark.parametrize("kw", [dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(tables=None), dict(out_dtype=1),
                                dict(prefixes=2, shard=(None, 3, 3, None, 0)), dict(ws=None), dict(ws=AT + 16), dict(ws_bytes=1000), dict(q=0),
                                dict(q=AT + 8), dict(stride=1028), dict(out=0), dict(out=AT + 8), dict(ostride=1028),
                                dict(out_dtype=3, ostride=1026)])
def test_the_attention_refuses_bad_views_and_workspaces(hcp, kw):
    assert _call("attn", **kw) == -6


def test_nothing_to_do_and_sizes(hcp):
    assert _call("attn", tokens=0) == 0
    d = H.DecodeDesc(**DESC)
    L = H.lib()
    assert L.hcp_step_attn_plan_size(None, 4, 0) == 0 and L.hcp_step_attn_workspace_size(None, 4, 0) == 0
    assert L.hcp_step_attn_plan_size(ctypes.byref(d), -1, 0) == 0 and L.hcp_step_attn_workspace_size(ctypes.byref(d), 4, 2000) == 0
    sizes = [(L.hcp_step_attn_plan_size(ctypes.byref(d), n, p), L.hcp_step_attn_workspace_size(ctypes.byref(d), n, p))
             for n in (1, 5, 700) for p in (0, 3)]
    assert all(a > 0 and b > 0 for a, b in sizes)


def test_bindings_refuse_what_does_not_fit(hcp):
    step = Step([1, 2], [3, 4], 4, 2, 64, ids=[0, -1], plens=[5])
    x = step.device("cpu")
    args = [x[k] for k in ("q", "pool", "tables", "starts", "lens", "ptables", "ids", "plens")]
    for i, bad in ((0, x["q"].half()), (1, x["pool"][0]), (1, x["pool"].half()), (2, x["tables"].long()), (2, x["tables"][0]), (3, x["starts"][:2]),
                   (3, x["starts"].long()), (4, x["lens"][:1]), (5, x["ptables"].long()), (6, None), (6, x["ids"][:1]), (7, None),
                   (7, x["plens"].float()), (0, x["q"])):
        with pytest.raises(ValueError):  # the last: tensors on the CPU
            H.step_attn_plan(*(args[:i] + [bad] + args[i + 1:]))
    plan = torch.zeros(1 << 16, dtype=torch.uint8)
    for kw in (dict(out=torch.zeros(4, 3, 32)), dict(lse=torch.zeros(4, 2)), dict(lse=torch.zeros(4, 3).half()), dict(plan=plan[::2]), dict()):
        with pytest.raises(ValueError):
            H.step_attn(x["q"], x["pool"], x["tables"], kw.pop("plan", plan), x["ptables"], **kw)


def test_bindings_refuse_tables_whose_rows_overlap(hcp):
    """An expanded row, or rows closer than their length, would be read at other places than the tensor's."""
    step = Step([1, 2], [3, 4], 4, 2, 64, ids=[0, -1], plens=[5, 3])
    x = step.device("cpu")
    for key in ("tables", "ptables"):
        row = torch.zeros(64, dtype=torch.int32)
        for bad in (row[:5].expand(2, 5), row.as_strided((2, 5), (4, 1))):
            y = dict(x, **{key: bad})
            with pytest.raises(ValueError, match="overlap"):
                H.step_attn_plan(*(y[k] for k in ("q", "pool", "tables", "starts", "lens", "ptables", "ids", "plens")))
            with pytest.raises(ValueError, match="overlap"):
                H.step_attn(y["q"], y["pool"], y["tables"], torch.zeros(1 << 16, dtype=torch.uint8), y["ptables"])
