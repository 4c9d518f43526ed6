"""Cases that time the 8-bit paged K/V cache's operators: the step plan (block tables and
slots from request lengths), the quantising append, the decode attention over the cache
(partial and Q-ring), and the dequantising gather with the prefill that stands on it.

A cache is a pool of codes [2, num_blocks, block_size, Hkv, D] (plane 0 = K, plane 1 = V;
float8_e4m3fn or int8) and a scale for each plane, block and head [2, num_blocks, Hkv]
fp32: a code stands for scale * code.  Head layouts are those of bench.py and the tests
(Llama-3-8B, Qwen2.5-3B, Qwen2-0.5B) and one generic one of 96 dims.
"""
from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TORCH_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODE_DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}

# attention heads: query heads, KV heads, head dim (Llama-3-8B, Qwen2.5-3B, Qwen2-0.5B, generic)
LLAMA = dict(hq=32, hkv=8, d=128)
QWEN3B = dict(hq=16, hkv=2, d=128)
QWEN05B = dict(hq=14, hkv=2, d=64)
GENERIC = dict(hq=8, hkv=1, d=96)


def listed():
    return [
        # The plan of a decode step of a few interactive sequences: one new token each.
        dict(name="plan_decode_16", kind="plan", batch=16, ctx=2085, chunk=1, prefills=0, ended=0, bs=16, spare=64),
        # A full serving batch's decode step, a few sequences ended since the last one.
        dict(name="plan_decode_256", kind="plan", batch=256, ctx=4096, chunk=1, prefills=0, ended=5, bs=16, spare=2048),
        # A mixed step of a large batch: decode tokens beside prompt chunks, a few requests ended,
        # too few free blocks for the last prompts.
        dict(name="plan_mixed_1000", kind="plan", batch=1000, ctx=8192, chunk=1531, prefills=40, ended=3, bs=16, spare=600),
        # The append of a decode step: one token of each of 64 sequences, blocks partly filled.
        dict(name="append_decode_64", kind="append", batch=64, tokens=1, ctx=16384, **LLAMA, dtype="bf16", fmt="e4m3", bs=16),
        # Ragged prompt tails behind cached prefixes, fp16 inputs, int8 codes.
        dict(name="append_ragged_6", kind="append", batch=6, tokens=517, ctx=1027, **QWEN3B, dtype="f16", fmt="int8", bs=16),
        # A long prompt's K/V.
        dict(name="append_prefill_32k", kind="append", batch=1, tokens=32768, ctx=0, **LLAMA, dtype="bf16", fmt="e4m3", bs=16),
        # One short chat sequence: latency counts; the partial's fp32 rows for a ring packet.
        dict(name="decode_1x130", kind="decode", batch=1, ctx=130, domains=0, **LLAMA, dtype="bf16", fmt="e4m3", bs=16),
        # A few ragged sequences over two domains' shards, int8 codes.
        dict(name="decode_qwen3b_6x2k", kind="decode", batch=6, ctx=2085, domains=2, **QWEN3B, dtype="f16", fmt="int8", bs=16),
        # A full serving batch at 16k context over three growth-sharded domains.
        dict(name="decode_llama_64x16k", kind="decode", batch=64, ctx=16384, domains=3, **LLAMA, dtype="bf16", fmt="e4m3", bs=16),
        # A cached prompt of odd length staged for a ring step, int8 codes to fp16.
        dict(name="gather_1027", kind="gather", tokens=1027, skip=13, **QWEN05B, dtype="f16", fmt="int8", bs=32),
        # A long cached prompt staged whole.
        dict(name="gather_32k", kind="gather", tokens=32768, skip=0, **LLAMA, dtype="bf16", fmt="e4m3", bs=16),
        # A cached prompt over two uneven domains, staged and folded.
        dict(name="prefill_paged8_2k", kind="prefill", chunks="1531,554", **LLAMA, dtype="bf16", fmt="e4m3", bs=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "append", "decode", "decode", "decode", "gather", "prefill"])
    heads = dict(rng.choice([LLAMA, QWEN3B, QWEN05B, GENERIC]))
    more = dict(heads, dtype=rng.choice(["bf16", "bf16", "f16"]), fmt=rng.choice(["e4m3", "e4m3", "int8"]),
                bs=rng.choice([16, 16, 32, 64, 128]))
    if kind == "plan":
        batch = _log_int(rng, 1, 1000)
        return dict(kind=kind, batch=batch, ctx=_log_int(rng, 16, 8192), chunk=_log_int(rng, 1, 1531),
                    prefills=rng.randint(0, min(batch, 40)) if rng.random() < 0.5 else 0,
                    ended=rng.randint(0, batch // 8), bs=more["bs"], spare=_log_int(rng, 16, 8192))
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, batch=_log_int(rng, 1, 256), tokens=1, ctx=_log_int(rng, 16, 4096), **more)
        return dict(kind=kind, batch=rng.randint(1, 8), tokens=_log_int(rng, 2, 4000), ctx=_log_int(rng, 16, 4096), **more)
    if kind == "decode":
        return dict(kind=kind, batch=_log_int(rng, 1, 64), ctx=_log_int(rng, 16, 16384), domains=rng.randint(0, 4), **more)
    if kind == "gather":
        return dict(kind=kind, tokens=_log_int(rng, 1, 32768), skip=rng.randint(0, 100), **more)
    s = _log_int(rng, 130, 2500)
    cut = rng.randint(1, s - 1)
    return dict(kind=kind, chunks="%d,%d" % (cut, s - cut) if rng.random() < 0.7 else str(s), **more)


# ---------------------------------------------------------------------------------
# inputs (made from the seed alone)
# ---------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normals(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=TORCH_DTYPE[dtype])


def _power(e, dtype=torch.float32):
    """2^e exactly, from its bits (e within the type's normal exponents)."""
    if dtype == torch.float32:
        return ((e.to(torch.int32) + 127) << 23).view(torch.float32)
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _cache(g, blocks, case):
    """Codes as quantised normals have them, with scales that differ from block to block."""
    shape = (2, blocks, case["bs"], case["hkv"], case["d"])
    if case["fmt"] == "e4m3":
        codes = torch.randn(shape, generator=g, device=DEVICE).mul_(110.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
        low = -8
    else:
        codes = torch.randn(shape, generator=g, device=DEVICE).mul_(32.0).round_().clamp_(-127.0, 127.0).to(torch.int8)
        low = -6
    e = torch.randint(low, low + 3, (2, blocks, case["hkv"]), generator=g, device=DEVICE)
    return codes, _power(e)


def _perm(g, n):
    return torch.randperm(n, generator=g, device=DEVICE).to(torch.int32)


def _ints(v, dtype=torch.int32):
    return torch.tensor(np.asarray(v), dtype=dtype, device=DEVICE)


def _plan_lens(case, seed):
    """Tokens held and tokens to add of every sequence (-1: it ended)."""
    r = np.random.default_rng(seed)
    b = case["batch"]
    lens = r.integers(max(1, case["ctx"] // 8), case["ctx"] + 1, b)
    new = np.ones(b, np.int64)
    order = r.permutation(b)
    for i in order[: case["prefills"]]:  # prompts: some new, some behind a cached prefix
        lens[i] = 0 if r.random() < 0.5 else lens[i]
        new[i] = r.integers(1, case["chunk"] + 1)
    new[order[b - case["ended"]:]] = -1
    return lens, new


def _plan_inputs(case, seed):
    g = _gen(seed)
    bs, b = case["bs"], case["batch"]
    lens, new = _plan_lens(case, seed)
    used = -(-lens // bs)
    width = int((-(-(case["ctx"] + case["chunk"]) // bs)))
    total = b * (-(-case["ctx"] // bs)) + case["spare"]  # blocks of the cache; some belong to nobody here
    perm = _perm(g, total)
    tables = torch.full((b, width), -1, dtype=torch.int32, device=DEVICE)
    starts = np.concatenate([[0], np.cumsum(used)])
    col = torch.arange(width, device=DEVICE)
    held = col[None, :] < _ints(used, torch.int64)[:, None]
    src = (_ints(starts[:-1], torch.int64)[:, None] + col[None, :]).clamp_(max=total - 1)
    tables = torch.where(held, perm[src], tables)
    free = torch.full((total,), -1, dtype=torch.int32, device=DEVICE)
    free[: case["spare"]] = perm[int(used.sum()): int(used.sum()) + case["spare"]]
    tokens = b + case["prefills"] * case["chunk"]  # room for the largest step
    return dict(seq_lens=_ints(lens), new_lens=_ints(new), tables=tables, free=free, free_count=_ints([case["spare"]]),
                capacity=tokens)


def _append_lens(case, seed):
    """Tokens held (from the seed) and tokens to add (from the case alone) of every sequence."""
    b = case["batch"]
    lens = np.random.default_rng(seed).integers(0, case["ctx"] + 1, b)
    new = np.full(b, case["tokens"])
    if case["tokens"] > 1 and b > 1:
        new = np.random.default_rng(case["tokens"]).integers(max(1, case["tokens"] // 2), case["tokens"] + 1, b)
    return lens, new


def _append_inputs(case, seed):
    """K/V rows of the new tokens in batch order, a slot each, and the cache they go to."""
    g = _gen(seed)
    bs = case["bs"]
    lens, new = _append_lens(case, seed)
    first = lens // bs
    blocks = -(-new // bs) + 1  # only the blocks that may be written belong to this cache
    total = int(blocks.sum())
    pool, scales = _cache(g, total, case)
    perm = _perm(g, total).long()
    t = int(new.sum())
    k, v = (_normals(g, (t, case["hkv"], case["d"]), case["dtype"]).permute(1, 0, 2) for _ in range(2))
    base = np.concatenate([[0], np.cumsum(blocks)])[:-1]
    starts = np.concatenate([[0], np.cumsum(new)])
    seq = np.repeat(np.arange(case["batch"]), new)
    pos = lens[seq] + np.arange(t) - starts[:-1][seq]
    at = _ints(base[seq] + pos // bs - first[seq], torch.int64)
    slots = perm[at] * bs + _ints(pos % bs, torch.int64)
    return dict(k=k, v=v, pool=pool, scales=scales, slots=slots, starts=_ints(starts, torch.int64))


def _shard_lens(case, seed):
    """Tokens of every sequence in every shard [shards][batch]; one shard without a ring."""
    n, b = max(1, case["domains"]), case["batch"]
    r = np.random.default_rng(seed)
    ctx = r.integers(max(1, case["ctx"] // 2), case["ctx"] + 1, b)
    ctx[0] = case["ctx"]
    weights = np.array([4, 3, 2, 1][:n], dtype=np.float64)
    lens = np.floor(ctx[None, :] * (weights / weights.sum())[:, None]).astype(np.int64)
    lens[0] += ctx - lens.sum(0)
    return lens


def _decode_inputs(case, seed):
    g = _gen(seed)
    b, bs = case["batch"], case["bs"]
    lens = _shard_lens(case, seed)
    blocks = [max(1, -(-int(x.max()) // bs)) for x in lens]
    total = b * sum(blocks)
    q = _normals(g, (b, case["hq"], case["d"]), case["dtype"])
    pool, scales = _cache(g, total, case)
    perm = _perm(g, total)
    cuts = np.concatenate([[0], np.cumsum(blocks)]) * b
    shards = [(perm[cuts[i]: cuts[i + 1]].view(b, blocks[i]), _ints(lens[i]), int(lens[i].max())) for i in range(len(blocks))]
    return dict(q=q, pool=pool, scales=scales, shards=shards, t0=3 if case["domains"] == 0 else 0)


def _gather_inputs(case, seed):
    g = _gen(seed)
    end = case["skip"] + case["tokens"]
    blocks = -(-end // case["bs"])
    pool, scales = _cache(g, blocks + 2, case)
    return dict(pool=pool, scales=scales, table=_perm(g, blocks + 2)[:blocks], t0=case["skip"], t1=end)


def _prefill_inputs(case, seed):
    g = _gen(seed)
    chunks = [int(c) for c in case["chunks"].split(",")]
    s = sum(chunks)
    blocks = -(-s // case["bs"])
    q = _normals(g, (s, case["hq"], case["d"]), case["dtype"]).permute(1, 0, 2)
    pool, scales = _cache(g, blocks, case)
    return dict(q=q, pool=pool, scales=scales, table=_perm(g, blocks), chunks=chunks)


INPUTS = {"plan": _plan_inputs, "append": _append_inputs, "decode": _decode_inputs, "gather": _gather_inputs,
          "prefill": _prefill_inputs}


def _package():
    return importlib.import_module("hetero-cp-ringattn_amd")


def prepare(case, seed):
    st = dict(INPUTS[case["kind"]](case, seed), case=case)
    empty = lambda *shape, dtype: torch.empty(shape, dtype=dtype, device=DEVICE)  # noqa: E731
    if case["kind"] == "plan":
        b, cap = case["batch"], st["capacity"]
        st["out"] = dict(slots=empty(cap, dtype=torch.int64), positions=empty(cap, dtype=torch.int64),
                         token_starts=empty(b + 1, dtype=torch.int32), seq_lens_out=empty(b, dtype=torch.int32),
                         free_count_out=empty(1, dtype=torch.int32))
        if own:
            st["ws"] = empty(max(1, _package().kv_plan_workspace_size(b)), dtype=torch.uint8)
    elif case["kind"] == "decode":
        f = torch.float32
        b, hq, d = st["q"].shape
        st["o"] = empty(b, hq, d, dtype=f if case["domains"] == 0 else st["q"].dtype)
        st["lse"] = empty(b, hq, dtype=f)
        if own:
            H = _package()
            tables, _, longest = st["shards"][0]
            n = (H.kv8_decode_workspace_size(st["q"], st["pool"], tables, st["t0"], longest) if case["domains"] == 0 else
                 H.kv8_decode_ring_workspace_size(st["q"], st["pool"], st["shards"]))
            st["ws"] = empty(max(1, n), dtype=torch.uint8)
    elif case["kind"] == "gather":
        shape = (case["hkv"], case["tokens"], case["d"])
        st["k"], st["v"] = (empty(*shape, dtype=TORCH_DTYPE[case["dtype"]]) for _ in range(2))
    elif case["kind"] == "prefill":
        q = st["q"]
        st["o"] = empty(*q.shape, dtype=q.dtype)
        st["lse"] = empty(*q.shape[:2], dtype=torch.float32)
        if own:
            n = _package().replay_workspace_size(q.dtype, case["hq"], case["hkv"], case["d"], st["chunks"], paged=True)
            st["ws"] = empty(max(1, n), dtype=torch.uint8)
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
    H = _package()
    if kind == "plan":
        H.kv_plan_step(st["seq_lens"], st["new_lens"], st["tables"], st["free"], st["free_count"], st["case"]["bs"],
                       workspace=st["ws"], **st["out"])
        return dict(st["out"], tables=st["tables"], free=st["free"])
    if kind == "append":
        H.kv8_append(st["pool"], st["scales"], st["k"], st["v"], st["slots"])
        return st["pool"], st["scales"]
    if kind == "decode":
        if st["case"]["domains"] == 0:
            tables, lens, longest = st["shards"][0]
            return H.kv8_decode_partial(st["q"], st["pool"], st["scales"], tables, st["t0"], longest, seq_lens=lens,
                                        workspace=st["ws"], o=st["o"], lse=st["lse"])
        return H.kv8_decode_ring_replay(st["q"], st["pool"], st["scales"], st["shards"], 0, out=st["o"],
                                        lse_out=st["lse"], workspace=st["ws"])
    if kind == "gather":
        return H.kv8_gather(st["pool"], st["scales"], st["table"], 0, st["t0"], st["t1"], k_out=st["k"], v_out=st["v"])
    return H.kv8_ring_attention_replay_paged(st["q"], st["pool"], st["scales"], st["table"], st["chunks"], out=st["o"],
                                             lse_out=st["lse"], workspace=st["ws"])


def _plain_plan(st):
    bs, out = st["case"]["bs"], st["out"]
    lens, new, tables, free = st["seq_lens"].long(), st["new_lens"].long(), st["tables"], st["free"]
    count = st["free_count"].long()
    b, width = tables.shape
    cap = st["capacity"]
    gone = new < 0
    add = new.clamp(min=0)
    ends = torch.cumsum(add, 0)
    used = (lens + bs - 1) // bs
    fits = ~gone & ((lens + add + bs - 1) // bs <= width) & (ends <= cap)
    need = torch.where(fits, (lens + add + bs - 1) // bs - used, 0)
    back = torch.where(gone, used, 0)
    back_ends, need_ends = torch.cumsum(back, 0), torch.cumsum(need, 0)
    # the stack once the ended sequences' blocks lie on it (one place more, for what is not pushed)
    col = torch.arange(width, device=DEVICE)
    at = torch.where(gone[:, None] & (col[None, :] < used[:, None]), count + (back_ends - back)[:, None] + col[None, :],
                     free.numel())
    stack = torch.cat([free, free[:1]])
    stack[at.reshape(-1)] = tables.reshape(-1)
    stack = stack[:-1]
    top = count + back_ends[-1:]
    served = fits & ((need == 0) | (need_ends <= top))
    taken = torch.where(served, need, 0)
    left = top - taken.sum()
    # new table entries, from the top of the stack
    fresh = served[:, None] & (col[None, :] >= used[:, None]) & (col[None, :] < (used + need)[:, None])
    pick = (top - 1 - (need_ends - need)[:, None] - (col[None, :] - used[:, None])).clamp(0, free.numel() - 1)
    tables.copy_(torch.where(fresh, stack[pick], tables))
    place = torch.arange(free.numel(), device=DEVICE)
    free.copy_(torch.where((place >= count) & (place < left), stack, free))
    # every token's sequence, position and slot
    i = torch.arange(cap, device=DEVICE)
    seq = torch.searchsorted(ends, i, right=True)
    inside = seq < b
    seq = seq.clamp(max=b - 1)
    pos = torch.where(inside, lens[seq] + i - (ends - add)[seq], 0)
    blk = tables[seq, (pos // bs).clamp(max=width - 1)].long()
    out["slots"].copy_(torch.where(inside & served[seq], blk * bs + pos % bs, -1))
    out["positions"].copy_(pos)
    out["token_starts"][1:] = ends
    out["token_starts"][:1] = 0
    out["seq_lens_out"].copy_(torch.where(gone, 0, torch.where(served, lens + add, lens)))
    out["free_count_out"].copy_(left)
    return dict(out, tables=tables, free=free)


def _power_scale(amax, fmt):
    """The smallest power of two (2^-100 at least) under which amax is within the format."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1)
    bits, top = (9, 448.0 / 512.0) if fmt == "e4m3" else (7, 127.0 / 128.0)
    e = torch.where(amax > 0, e - bits + (m > top).to(e.dtype), -100).clamp(min=-100)
    return _power(e)


def _encode(x, fmt):
    return x.to(torch.float8_e4m3fn) if fmt == "e4m3" else torch.round(x).to(torch.int8)


def _plain_append(st):
    case = st["case"]
    fmt, bs, pool, scales, slots = case["fmt"], case["bs"], st["pool"], st["scales"], st["slots"]
    _, nb, _, h, d = pool.shape
    x = torch.stack([st["k"], st["v"]]).float().permute(0, 2, 1, 3)  # [2, T, Hkv, D]
    blk, first = slots // bs, slots[st["starts"][:-1]]
    amax = torch.zeros(2, nb, h, device=DEVICE).index_reduce_(1, blk, x.abs().amax(3), "amax")
    # the first block of a sequence may hold earlier rows: its scale never falls, they are rounded again where it grows
    fb, fa = first // bs, first % bs
    old = torch.where((fa > 0)[None, :, None], scales[:, fb], 0.0)
    need = _power_scale(amax, fmt)
    need[:, fb] = torch.maximum(need[:, fb], old)
    before = torch.arange(bs, device=DEVICE)[None, :] < fa[:, None]  # [B, bs]
    held = pool[:, fb].float() * (old / need[:, fb])[:, :, None, :, None]
    codes = pool.view(torch.uint8)
    codes[:, fb] = torch.where(before[None, :, :, None, None], _encode(held, fmt).view(torch.uint8), codes[:, fb])
    scales[:, blk] = need[:, blk]
    codes.view(2, nb * bs, h, d)[:, slots] = _encode(x / need[:, blk][..., None], fmt).view(torch.uint8)
    return pool, scales


def _rows(st, table, plane):
    """The cached rows of the tables' blocks in fp32: [..., blocks * bs, Hkv, D]."""
    at = table.long()
    codes, scales = st["pool"][plane].view(torch.uint8)[at], st["scales"][plane][at]
    x = codes.view(st["pool"].dtype).float() * scales[..., None, :, None]
    return x.reshape(*table.shape[:-1], -1, *x.shape[-2:])


def _softmax_rows(s, v):
    """(softmax(s) @ v, log-sum-exp) over the last axis; a row without a key gives 0 and -inf."""
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0), (m + torch.log(total)).squeeze(-1)


def _plain_decode(st):
    case = st["case"]
    b, hq, d = st["q"].shape
    hkv = case["hkv"]
    k, v = (torch.cat([_rows(st, t, plane) for t, _, _ in st["shards"]], 1) for plane in range(2))  # [B, n, Hkv, D]
    seen = torch.cat([(torch.arange(t.shape[1] * case["bs"], device=DEVICE)[None, :] < n[:, None])
                      for t, n, _ in st["shards"]], 1)
    seen[:, : st["t0"]] = False
    q = st["q"].float().view(b, hkv, hq // hkv, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(d)
    s = torch.where(seen[:, None, None, :], s, -math.inf)
    o, lse = _softmax_rows(s, v.permute(0, 2, 1, 3).contiguous())
    st["o"].copy_(o.reshape(b, hq, d))
    st["lse"].copy_(lse.reshape(b, hq))
    return st["o"], st["lse"]


def _plain_gather(st):
    st["k"].copy_(_rows(st, st["table"], 0)[st["t0"]: st["t1"]].permute(1, 0, 2))
    st["v"].copy_(_rows(st, st["table"], 1)[st["t0"]: st["t1"]].permute(1, 0, 2))
    return st["k"], st["v"]


def _plain_prefill(st):
    case, q = st["case"], st["q"].float()
    hq, n, d = q.shape
    hkv = case["hkv"]
    k, v = (_rows(st, st["table"], plane)[:n] for plane in range(2))
    s = torch.matmul(q.reshape(hkv, -1, d), k.permute(1, 2, 0).contiguous()).view(hkv, hq // hkv, n, n) / math.sqrt(d)
    i = torch.arange(n, device=DEVICE)
    s = torch.where(i[None, :] <= i[:, None], s, -math.inf)
    o, lse = _softmax_rows(s, v.permute(1, 0, 2).contiguous()[:, None])
    st["o"].copy_(o.reshape(hq, n, d))
    st["lse"].copy_(lse.reshape(hq, n))
    return st["o"], st["lse"]


PLAIN = {"plan": _plain_plan, "append": _plain_append, "decode": _plain_decode, "gather": _plain_gather,
         "prefill": _plain_prefill}


# ---------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "plan":
        lens, new = _plan_lens(case, 0)
        add = np.maximum(new, 0)
        bs = case["bs"]
        blocks = int((-(-(lens + add) // bs) - -(-lens // bs)).sum()) + int((-(-lens // bs))[new < 0].sum())
        # lengths in and out, a table or stack entry read and written per block that moves, slot and position of a token
        return {"bytes": 16 * case["batch"] + 8 * blocks + 16 * (case["batch"] + case["prefills"] * case["chunk"]), "flops": 0}
    h, d, bs = case["hkv"], case["d"], case["bs"]
    es = 4 if case["dtype"] == "f32" else 2
    if kind == "append":
        t = int(_append_lens(case, 0)[1].sum())
        return {"bytes": 2 * t * h * d * (es + 1) + 8 * t + 8 * h * -(-t // bs), "flops": 2 * t * h * d}
    if kind == "decode":
        t, hq = int(_shard_lens(case, 0).sum()), case["hq"]
        out = 4 if case["domains"] == 0 else es
        return {"bytes": 2 * t * h * d + 8 * h * -(-t // bs) + case["batch"] * hq * (d * (es + out) + 4), "flops": 4 * t * hq * d}
    if kind == "gather":
        t = case["tokens"]
        return {"bytes": 2 * t * h * d * (es + 1) + 8 * h * -(-t // bs), "flops": 2 * t * h * d}
    s, hq = sum(int(c) for c in case["chunks"].split(",")), case["hq"]
    return {"bytes": 2 * s * h * d + 8 * h * -(-s // bs) + s * hq * (2 * d * es + 4), "flops": 2 * d * hq * s * (s + 1)}


# ---------------------------------------------------------------------------------
# 64-bit results
# ---------------------------------------------------------------------------------
def _attend64(q, k, v, visible):
    """One KV head in fp64: q [n, D], k / v [m, D], visible [n, m] or [m]."""
    s = torch.mm(q.double(), k.t().contiguous()) / math.sqrt(q.shape[1])
    s = s.masked_fill(~visible.expand_as(s), -math.inf)
    lse = torch.logsumexp(s, 1)
    w = torch.exp(s - lse[:, None]).nan_to_num_(0.0)  # a row without a key: all weights 0
    return torch.mm(w, v), lse


def _values64(pool, scales, plane, blocks):
    """Rows of a list of blocks as fp64 values [blocks * bs, Hkv, D]."""
    at = blocks.long()
    c = pool[plane].view(torch.uint8)[at].view(pool.dtype).double() if pool.dtype == torch.int8 else \
        pool[plane].view(torch.uint8)[at].view(pool.dtype).float().double()
    return (c * scales[plane][at].double().view(len(at), 1, -1, 1)).flatten(0, 1)


def _round64(x, fmt):
    """The format's nearest value (ties to even) of fp64 values within its range."""
    if fmt == "int8":
        return torch.round(x)
    e = torch.frexp(x)[1].clamp(min=-5)  # |x| in [2^(e-1), 2^e): steps of 2^(e-4), 2^-9 below 2^-6
    step = _power(e - 4, torch.float64)
    return torch.round(x / step) * step


def _exact_append(case, st):
    fmt, bs = case["fmt"], case["bs"]
    pool, scales = st["pool"], st["scales"]
    nb, h, d = pool.shape[1], pool.shape[3], pool.shape[4]
    val = pool.float().double() if fmt == "e4m3" else pool.double()
    sc = scales.double()
    slots = st["slots"].cpu().numpy()
    starts = np.flatnonzero(np.concatenate([[True], (np.diff(slots) != 1) | (slots[1:] % bs == 0)]))
    for i, n in zip(starts, np.diff(np.concatenate([starts, [len(slots)]]))):
        blk, a = divmod(int(slots[i]), bs)
        for plane, src in enumerate((st["k"], st["v"])):
            x = src[:, i: i + n].permute(1, 0, 2).double()
            top = x.abs().amax((0, 2))
            lg = torch.ceil(torch.log2(top / LARGEST[fmt])).clamp(min=-100)
            lg = torch.where(LARGEST[fmt] * _power(lg, torch.float64) < top, lg + 1, lg)  # log2's own rounding
            lg = torch.where(LARGEST[fmt] * _power(lg - 1, torch.float64) >= top, lg - 1, lg).clamp(min=-100)
            s = _power(lg, torch.float64)
            if a > 0:
                s = torch.maximum(s, sc[plane, blk])
                val[plane, blk, :a] = _round64(val[plane, blk, :a] * (sc[plane, blk] / s)[None, :, None], fmt)
            val[plane, blk, a: a + n] = _round64(x / s[None, :, None], fmt)
            sc[plane, blk] = s
    return val, sc


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    st = INPUTS[case["kind"]](case, seed)
    pool, scales = st["pool"], st["scales"]
    if case["kind"] == "append":
        if case["tokens"] * case["batch"] > 20000:
            return None
        val, sc = _exact_append(case, st)
        return (val if case["fmt"] == "e4m3" else None), sc
    if case["kind"] == "gather":
        return tuple(_values64(pool, scales, i, st["table"])[st["t0"]: st["t1"]].permute(1, 0, 2) for i in range(2))
    rep = case["hq"] // case["hkv"]
    if case["kind"] == "prefill":
        hq, n, d = st["q"].shape
        k, v = (_values64(pool, scales, i, st["table"])[:n] for i in range(2))
        i = torch.arange(n, device=DEVICE)
        got = [_attend64(st["q"][h], k[:, h // rep].contiguous(), v[:, h // rep].contiguous(), i[None, :] <= i[:, None])
               for h in range(hq)]
        return torch.stack([o for o, _ in got]), torch.stack([l for _, l in got])
    outs, lses = [], []
    lens = _shard_lens(case, seed)
    for b in range(case["batch"]):
        k, v = (torch.cat([_values64(pool, scales, i, t[b])[: int(n[b])] for (t, _, _), n in zip(st["shards"], lens)])
                for i in range(2))
        seen = torch.arange(k.shape[0], device=DEVICE) >= st["t0"]
        got = [_attend64(st["q"][b, h * rep: (h + 1) * rep], k[:, h].contiguous(), v[:, h].contiguous(), seen)
               for h in range(case["hkv"])]
        outs.append(torch.cat([o for o, _ in got]))
        lses.append(torch.cat([l for _, l in got]))
    return torch.stack(outs), torch.stack(lses)
