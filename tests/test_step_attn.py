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
            seen = (j - shared <= int(self.lens[b]) - int(n) + i) if self.causal else torch.ones(int(n), k.shape[0], dtype=torch.bool).cuda()
            for h in range(self.hq):
                kk, vv = k[:, h // rep], v[:, h // rep]
                x = (q[:, h] @ kk.T / math.sqrt(self.d)).masked_fill(~seen, -math.inf)
                lse[h, at] = torch.logsumexp(x, 1).cpu()
                w = torch.exp(x - torch.logsumexp(x, 1, keepdim=True)).nan_to_num(0.0)
                o[h, at], mag[h, at] = (w @ vv).cpu(), (w @ vv.abs()).cpu()
                size = (q[:, h].abs() @ kk.abs().T / math.sqrt(self.d)).masked_fill(~seen, 0.0)
                s[h, at] = (size.amax(1).cpu() if size.shape[1] else 0.0) * (self.d + 8) * 2.0 ** -24
        return o, mag, lse, s


def check(step, out, lse, ref=None, terms=1):
    o, mag, want, s = ref or step.reference()
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
