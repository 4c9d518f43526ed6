"""Cases that time a serving step's operators over the paged K/V cache: the norms of the
queries and keys of each head with the position rotation (dense, and with the append to
the cache through a slot map), and the step's attention (a batch of sequences with one or
many new tokens each, behind what the cache holds of them and behind prefixes that several
of them share).

A cache is a pool [2, num_blocks, block_size, Hkv, D] (plane 0 = K, plane 1 = V).  Head
layouts are those of bench.py and the tests (Llama-3-8B, Qwen2.5-3B, Qwen2-0.5B) and one
generic one of 96 dims.
"""
from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TORCH_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6

# attention heads: query heads, KV heads, head dim (Llama-3-8B, Qwen2.5-3B, Qwen2-0.5B, generic)
LLAMA = dict(hq=32, hkv=8, d=128)
QWEN3B = dict(hq=16, hkv=2, d=128)
QWEN05B = dict(hq=14, hkv=2, d=64)
GENERIC = dict(hq=8, hkv=1, d=96)


def _attn(name, **kw):
    """A step: `batch` sequences, `long` of them with up to `new` tokens, the others with `few`; up to
    `ctx` tokens of their own in the cache before; `prefixes` shared ones of up to `prefix` tokens."""
    case = dict(name=name, kind="attn", few=1, long=0, new=0, prefixes=0, prefix=0, causal=True, out="same", bs=16,
                dtype="bf16")
    case.update(kw)
    return case


def listed():
    return [
        # One new token of one sequence: latency counts.
        dict(name="append_1", kind="append", tokens=1, prompt=False, **LLAMA, rot=128, pairs=False, dtype="bf16", bs=16),
        # The decode step of a serving batch, fp16.
        dict(name="append_decode_64", kind="append", tokens=64, prompt=False, **QWEN3B, rot=128, pairs=False, dtype="f16", bs=32),
        # A long prompt.
        dict(name="append_prompt_32k", kind="append", tokens=32768, prompt=True, **LLAMA, rot=128, pairs=False, dtype="bf16", bs=16),
        # A prompt of odd length of a model that rotates half of its dims, in neighbouring pairs, fp32 activations.
        dict(name="norm_pairs_2085", kind="norm", tokens=2085, prompt=True, **GENERIC, rot=48, pairs=True, dtype="f32", bs=16),
        # One short chat sequence's token; fp32 rows, as a ring packet or a merge takes them.
        _attn("decode_1x130", batch=1, ctx=130, **LLAMA, out="f32"),
        # A full serving batch at 16k context, nothing shared.
        _attn("decode_64x16k", batch=64, ctx=16384, **LLAMA),
        # The same batch sampling from one long shared prompt, a few hundred tokens each of their own.
        _attn("shared_64x16k", batch=64, ctx=700, prefixes=1, prefix=16384, **LLAMA),
        # A large batch over a few system prompts, some sequences with none.
        _attn("shared_256x2k", batch=256, ctx=517, prefixes=3, prefix=2085, **QWEN3B, dtype="f16", bs=32),
        # Five drafted tokens of each sequence checked at once, behind a shared prompt.
        _attn("draft_32x5", batch=32, few=5, ctx=1531, prefixes=2, prefix=1027, **QWEN05B),
        # Prompt chunks behind cached contexts beside decoding sequences.
        _attn("mixed_43", batch=43, long=3, new=1531, ctx=8192, **LLAMA),
        # A peer domain's shard for a chunk of queries: no mask, fp32 partial rows.
        _attn("peer_512x2k", batch=1, long=1, new=512, ctx=1573, **GENERIC, dtype="f16", causal=False, out="f32", bs=32),
        # A long prompt at once.
        _attn("prompt_16k", batch=1, long=1, new=16384, ctx=0, **LLAMA),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "norm", "decode", "shared", "shared", "draft", "mixed", "prompt"])
    heads = dict(rng.choice([LLAMA, QWEN3B, QWEN05B, GENERIC]))
    more = dict(heads, dtype=rng.choice(["bf16", "bf16", "f16"]), bs=rng.choice([16, 16, 32, 64, 128]))
    if kind in ("append", "norm"):
        more["rot"] = rng.choice([heads["d"], heads["d"], heads["d"] // 2, 0])
        if kind == "norm":
            more["dtype"] = rng.choice(["bf16", "f16", "f32"])
        return dict(kind=kind, tokens=_log_int(rng, 1, 32768), prompt=rng.random() < 0.5, pairs=rng.random() < 0.3, **more)
    more["out"] = rng.choice(["same", "same", "f32"])
    batch = _log_int(rng, 1, 256)
    most = min(16384, (1 << 20) // batch)  # own tokens of a sequence: no more than 64 x 16384 in all
    if kind == "decode":
        case = dict(batch=batch, ctx=_log_int(rng, 1, most))
    elif kind == "shared":
        case = dict(batch=batch, ctx=_log_int(rng, 1, min(most, 2048)), prefixes=rng.randint(1, 4), prefix=_log_int(rng, 16, 16384))
    elif kind == "draft":
        case = dict(batch=min(batch, 64), few=rng.randint(2, 8), ctx=_log_int(rng, 1, min(most, 4096)),
                    prefixes=rng.randint(0, 2), prefix=_log_int(rng, 16, 4096))
    elif kind == "mixed":
        case = dict(batch=min(batch, 64), long=rng.randint(1, min(batch, 4)), new=_log_int(rng, 2, 2048),
                    ctx=_log_int(rng, 1, min(most, 8192)), prefixes=rng.randint(0, 2), prefix=_log_int(rng, 16, 2048))
    else:
        case = dict(batch=1, long=1, new=_log_int(rng, 16, 8192), ctx=rng.choice([0, _log_int(rng, 1, 4096)]),
                    causal=rng.random() < 0.75)
    case = _attn("", **dict(more, **case))
    del case["name"]
    return case


# ---------------------------------------------------------------------------------
# inputs (made from the seed alone)
# ---------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normals(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=TORCH_DTYPE[dtype])


def _perm(g, n):
    return torch.randperm(n, generator=g, device=DEVICE).to(torch.int32)


def _ints(v, dtype=torch.int32):
    return torch.tensor(np.asarray(v), dtype=dtype, device=DEVICE)


def _cos_sin(rot, rows):
    """cos and sin of position * 10000^(-2j/rot), [2, rows, rot/2] fp32."""
    j = torch.arange(rot // 2, device=DEVICE, dtype=torch.float64)
    a = torch.arange(rows, device=DEVICE, dtype=torch.float64)[:, None] * torch.pow(10000.0, -2.0 * j / rot)[None, :]
    return torch.stack([torch.cos(a), torch.sin(a)]).float()


def _norm_inputs(case, seed):
    """A step's projected rows [T, (Hq + 2 Hkv) D], the norms' weights, positions, and a slot a token."""
    g = _gen(seed)
    t, hq, hkv, d, bs = case["tokens"], case["hq"], case["hkv"], case["d"], case["bs"]
    rows = 32768 + 512
    x = _normals(g, (t, hq + 2 * hkv, d), case["dtype"])
    x[:, : hq + hkv].mul_(3.0)
    w = [(1.0 + 0.2 * _normals(g, (d,), "f32")).to(TORCH_DTYPE[case["dtype"]]) for _ in range(2)]
    if case["prompt"]:  # one sequence's next tokens, behind what is cached of it
        first = int(np.random.default_rng(seed).integers(0, 512))
        pos = torch.arange(first, first + t, device=DEVICE)
        at = pos - first // bs * bs
        perm = _perm(g, (t + bs - 1) // bs + 1).long()
        slots = perm[at // bs] * bs + at % bs
    else:  # a token of each sequence, in a block of its own
        pos = torch.randint(0, rows, (t,), generator=g, device=DEVICE)
        perm = _perm(g, t).long()
        slots = perm * bs + pos % bs
    st = dict(q=x[:, :hq].permute(1, 0, 2), k=x[:, hq: hq + hkv].permute(1, 0, 2), v=x[:, hq + hkv:].permute(1, 0, 2),
              wq=w[0], wk=w[1], pos=pos if case["rot"] else None, table=_cos_sin(case["rot"], rows) if case["rot"] else None,
              slots=slots)
    if case["kind"] == "append":
        st["pool"] = _normals(g, (2, perm.numel(), bs, hkv, d), case["dtype"])
    return st


def _step(case):
    """(new tokens, tokens held of its own with the new ones, prefix or -1) of every sequence, and the prefixes' lengths."""
    b, n = case["batch"], case["prefixes"]
    r = np.random.default_rng([b, case["ctx"], case["new"], case["few"], case["prefix"], n])
    new = np.full(b, case["few"])
    held = r.integers(case["ctx"] // 2, case["ctx"] + 1, b)
    held[0] = case["ctx"]
    ids = np.full(b, -1)
    if n:
        ids = r.integers(0, n, b)
        ids[8::8] = -1  # every eighth sequence shares nothing
    for i, at in enumerate(r.permutation(b)[: case["long"]]):
        new[at] = case["new"] if i == 0 else r.integers(max(1, case["new"] // 2), case["new"] + 1)
    lens = np.sort(r.integers(max(1, case["prefix"] // 2), case["prefix"] + 1, n))[::-1].copy() if n else np.zeros(0, np.int64)
    if n:
        lens[0] = case["prefix"]
    return new, held + new, ids, lens


def _attn_inputs(case, seed):
    g = _gen(seed)
    new, lens, ids, plens = _step(case)
    bs = case["bs"]
    t = int(new.sum())
    q = _normals(g, (t, case["hq"], case["d"]), case["dtype"]).permute(1, 0, 2)
    width, pwidth = -(-int(lens.max()) // bs), -(-case["prefix"] // bs) if case["prefixes"] else 0
    used = np.concatenate([-(-lens // bs), -(-plens // bs)])
    pool = _normals(g, (2, int(used.sum()), bs, case["hkv"], case["d"]), case["dtype"])
    perm = _perm(g, int(used.sum()))
    first = np.concatenate([[0], np.cumsum(used)])[:-1]

    def tables(starts, counts, n):
        col = torch.arange(n, device=DEVICE)
        at = _ints(starts, torch.int64)[:, None] + col[None, :]
        return torch.where(col[None, :] < _ints(counts)[:, None], perm[at.clamp(max=perm.numel() - 1)], -1).to(torch.int32)

    b = case["batch"]
    st = dict(q=q, pool=pool, tables=tables(first[:b], used[:b], width), starts=_ints(np.concatenate([[0], np.cumsum(new)])),
              lens=_ints(lens), prefix_tables=None, prefix_ids=None, prefix_lens=None)
    if case["prefixes"]:
        st.update(prefix_tables=tables(first[b:], used[b:], pwidth), prefix_ids=_ints(ids), prefix_lens=_ints(plens))
    return st


INPUTS = {"norm": _norm_inputs, "append": _norm_inputs, "attn": _attn_inputs}


def _package():
    return importlib.import_module("hetero-cp-ringattn_amd")


def prepare(case, seed):
    st = dict(INPUTS[case["kind"]](case, seed), case=case)
    q = st["q"]
    hq, t, d = q.shape
    out = torch.float32 if case.get("out") == "f32" else q.dtype
    st["o"] = torch.empty(t, hq, d, dtype=out, device=DEVICE).permute(1, 0, 2)
    if case["kind"] == "norm":
        st["ko"] = torch.empty(t, case["hkv"], d, dtype=q.dtype, device=DEVICE).permute(1, 0, 2)
    if case["kind"] == "attn":
        st["lse"] = torch.empty(hq, t, dtype=torch.float32, device=DEVICE)
        st["host"] = _step(case)  # the scheduler's own record of the step
        if own:  # made once a step; every layer's call takes it
            H = _package()
            st["plan"] = H.step_attn_plan(q, st["pool"], st["tables"], st["starts"], st["lens"], st["prefix_tables"],
                                          st["prefix_ids"], st["prefix_lens"], causal=case["causal"])
            n = H.step_attn_workspace_size(q, st["pool"], st["tables"], st["prefix_tables"])
            st["ws"] = torch.empty(max(1, n), dtype=torch.uint8, device=DEVICE)
    return st


# ---------------------------------------------------------------------------------
# one pass: the framework's calls, or the plain forms
# ---------------------------------------------------------------------------------
def run(st):
    kind = st["case"]["kind"]
    if own:
        return _run_own(st, kind)
    return PLAIN[kind](st)


def _run_own(st, kind):
    H, pairs = _package(), st["case"].get("pairs")
    if kind == "norm":
        return H.qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["pos"], st["table"], eps=EPS, pairs=pairs, q_out=st["o"],
                              k_out=st["ko"])
    if kind == "append":
        H.qk_norm_rope_append(st["q"], st["k"], st["v"], st["wq"], st["wk"], st["pool"], st["slots"], st["pos"], st["table"],
                              eps=EPS, pairs=pairs, q_out=st["o"])
        return st["o"], st["pool"]
    return H.step_attn(st["q"], st["pool"], st["tables"], st["plan"], st["prefix_tables"], causal=st["case"]["causal"],
                       out=st["o"], lse=st["lse"], workspace=st["ws"])


def _normed(st, x, w):
    """Norm and rotation of [H, T, D] rows in fp32."""
    case = st["case"]
    x, rot = x.float(), case["rot"]
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    if not rot:
        return y
    cos, sin = st["table"][:, st["pos"]]
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if case["pairs"] else (y[..., : rot // 2], y[..., rot // 2: rot])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([c, d], -1).flatten(-2) if case["pairs"] else torch.cat([c, d], -1)
    return torch.cat([turned, y[..., rot:]], -1)


def _plain_norm(st):
    st["o"].copy_(_normed(st, st["q"], st["wq"]))
    st["ko"].copy_(_normed(st, st["k"], st["wk"]))
    return st["o"], st["ko"]


def _plain_append(st):
    pool = st["pool"]
    rows = pool.view(2, -1, *pool.shape[3:])
    st["o"].copy_(_normed(st, st["q"], st["wq"]))
    rows[0][st["slots"]] = _normed(st, st["k"], st["wk"]).permute(1, 0, 2).to(pool.dtype)
    rows[1][st["slots"]] = st["v"].permute(1, 0, 2)
    return st["o"], pool


def _attend(s, v):
    """(softmax(s) @ v, log-sum-exp) over the last axis; a row without a key gives 0 and -inf."""
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0), (m + torch.log(total)).squeeze(-1)


def _plain_alike(st, at, n, first):
    """Sequences `at` with n new tokens each, whose first rows of q are `first`, at once."""
    case = st["case"]
    hkv, d, bs = case["hkv"], case["d"], case["bs"]
    rep, b = case["hq"] // hkv, at.numel()
    blocks, lens = st["tables"][at], st["lens"][at]
    col = torch.arange(blocks.shape[1] * bs, device=DEVICE)[None, None, :]
    row = torch.arange(n, device=DEVICE)[None, :, None]
    seen = col < (lens[:, None, None] - n + row + 1 if case["causal"] else lens[:, None, None])
    seen = seen.expand(b, n, -1)
    if st["prefix_tables"] is not None:
        ids = st["prefix_ids"][at].long()
        blocks = torch.cat([st["prefix_tables"][ids.clamp(min=0)], blocks], 1)
        col = torch.arange(st["prefix_tables"].shape[1] * bs, device=DEVICE)[None, :]
        shared = (col < st["prefix_lens"][ids.clamp(min=0)][:, None]) & (ids >= 0)[:, None]
        seen = torch.cat([shared[:, None, :].expand(b, n, -1), seen], 2)
    rows = (first[:, None] + torch.arange(n, device=DEVICE)[None, :]).reshape(-1)
    q = st["q"][:, rows].float().view(hkv, rep, b, n, d).permute(2, 0, 1, 3, 4).reshape(b, hkv, rep * n, d)
    k, v = (st["pool"][p][blocks.clamp(min=0).long()].float().view(b, -1, hkv, d) for p in range(2))
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(b, hkv, rep, n, -1) / math.sqrt(d)
    s = torch.where(seen[:, None, None], s, -math.inf).view(b, hkv, rep * n, -1)
    o, lse = _attend(s, v.permute(0, 2, 1, 3).contiguous())
    st["o"][:, rows] = o.view(b, hkv * rep, n, d).permute(1, 0, 2, 3).reshape(hkv * rep, b * n, d).to(st["o"].dtype)
    st["lse"][:, rows] = lse.view(b, hkv * rep, n).permute(1, 0, 2).reshape(hkv * rep, b * n)


def _plain_attn(st):
    case, (new, _, _, _) = st["case"], st["host"]
    starts = np.concatenate([[0], np.cumsum(new)])
    for n in np.unique(new):  # one batch for the sequences of each number of new tokens
        at = np.flatnonzero(new == n)
        _plain_alike(st, _ints(at, torch.int64), int(n), _ints(starts[at], torch.int64))
    return st["o"], st["lse"]


PLAIN = {"norm": _plain_norm, "append": _plain_append, "attn": _plain_attn}


# ---------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------
def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] != "attn":
        t, heads = case["tokens"], hq + hkv * (2 if case["kind"] == "append" else 1)
        index = (8 if case["rot"] else 0) + (8 if case["kind"] == "append" else 0)
        return {"bytes": 2 * t * heads * d * es + t * (4 * case["rot"] + index) + 2 * d * es,
                "flops": t * (hq + hkv) * (4 * d + 3 * case["rot"])}
    new, lens, ids, plens = _step(case)
    t = int(new.sum())
    used = plens[np.unique(ids[ids >= 0])].sum() if case["prefixes"] else 0
    pairs = new * lens - (new * (new - 1) // 2 if case["causal"] else 0)
    if case["prefixes"]:
        pairs = pairs + new * np.where(ids >= 0, plens[ids], 0)
    out = 4 if case["out"] == "f32" else es
    return {"bytes": 2 * int(lens.sum() + used) * hkv * d * es + t * hq * (d * (es + out) + 4), "flops": 4 * d * hq * int(pairs.sum())}


# ---------------------------------------------------------------------------------
# 64-bit results
# ---------------------------------------------------------------------------------
def _turn64(x, w, cos, sin, rot, pairs):
    """Rows [n, D] of one head in fp64: the norm, then each plane (i, j) turned by its angle."""
    y = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + EPS) * w.double()
    z = y.clone()
    if rot:
        i = torch.arange(rot // 2, device=DEVICE)
        i, j = (2 * i, 2 * i + 1) if pairs else (i, i + rot // 2)
        z[:, i] = y[:, i] * cos - y[:, j] * sin
        z[:, j] = y[:, i] * sin + y[:, j] * cos
    return z


def _exact_norm(case, st):
    cos, sin = st["table"].double()[:, st["pos"]] if case["rot"] else (None, None)
    q, k = (torch.stack([_turn64(h, w, cos, sin, case["rot"], case["pairs"]) for h in x])
            for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])))
    if case["kind"] == "norm":
        return q, k
    pool = st["pool"].double()
    blk, at = st["slots"] // case["bs"], st["slots"] % case["bs"]
    pool[0, blk, at] = k.transpose(0, 1)
    pool[1, blk, at] = st["v"].double().transpose(0, 1)
    return q, pool


def exact(case, seed):
    st = INPUTS[case["kind"]](case, seed)
    if case["kind"] != "attn":
        return _exact_norm(case, st)
    new, lens, ids, plens = _step(case)
    bs, rep, d = case["bs"], case["hq"] // case["hkv"], case["d"]
    o = torch.zeros(case["hq"], int(new.sum()), d, dtype=torch.float64, device=DEVICE)
    lse = torch.zeros(o.shape[:2], dtype=torch.float64, device=DEVICE)
    end = 0
    for b in range(case["batch"]):
        n, own_keys = int(new[b]), int(lens[b])
        end += n
        blocks = [st["tables"][b, : -(-own_keys // bs)].long()]
        shared = int(plens[ids[b]]) if ids[b] >= 0 else 0
        if shared:
            blocks.insert(0, st["prefix_tables"][int(ids[b]), : -(-shared // bs)].long())
        k, v = (torch.cat([st["pool"][p, x].flatten(0, 1)[:m] for x, m in zip(blocks, [shared, own_keys][-len(blocks):])])
                for p in range(2))
        for h in range(case["hq"]):
            s = torch.mm(st["q"][h, end - n: end].double(), k[:, h // rep].double().t().contiguous()) / math.sqrt(d)
            if case["causal"] and n > 1:  # new token i stands behind all but n - 1 - i of the keys
                s = s.masked_fill_(torch.ones(n, n, dtype=torch.bool, device=DEVICE).triu_(1), -math.inf) if s.shape[1] == n else \
                    torch.cat([s[:, :-n], s[:, -n:].masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEVICE).triu_(1), -math.inf)], 1)
            lse[h, end - n: end] = torch.logsumexp(s, 1)
            o[h, end - n: end] = torch.mm(s.sub_(lse[h, end - n: end, None]).exp_(), v[:, h // rep].double())
    return o, lse
