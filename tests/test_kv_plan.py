"""The step plan of a paged cache (block tables, slots, positions, free-block stack) against
a plain restatement on the host, one sequence at a time.  Every output is a whole number
and has to be equal."""
import ctypes

import numpy as np
import pytest
import torch

import hcp_ring_amd as H

I32 = torch.int32


def plan_reference(lens, new, tables, free, count, bs, capacity):
    """The plan sequence by sequence: (slots, positions, starts, lens, count, tables, free)."""
    lens, new, tables, free = (np.array(x, dtype=np.int64) for x in (lens, new, tables, free))
    b, width = tables.shape
    out_lens, before = lens.copy(), free[:count].copy()
    stack = list(before)
    for i in range(b):
        if new[i] < 0:
            stack += list(tables[i, : -(-lens[i] // bs)])
            out_lens[i] = 0
    starts = np.concatenate([[0], np.cumsum(np.maximum(new, 0))])
    slots, positions = np.full(capacity, -1, np.int64), np.zeros(capacity, np.int64)
    asked, top, taken = 0, len(stack), 0
    new_tables = tables.copy()
    for i in range(b):
        if new[i] < 0:
            continue
        used, blocks = -(-lens[i] // bs), -(-(lens[i] + new[i]) // bs)
        served = blocks <= width and starts[i + 1] <= capacity
        if served:
            need = blocks - used
            asked += need
            served = need == 0 or asked <= top
            if served:
                for j in range(need):
                    new_tables[i, used + j] = stack[top - 1 - taken - j]
                taken += need
                out_lens[i] += new[i]
        for t in range(new[i]):
            at = starts[i] + t
            if at < capacity:
                positions[at] = lens[i] + t
                if served:
                    slots[at] = new_tables[i, positions[at] // bs] * bs + positions[at] % bs
    left = top - taken
    new_free = free.copy()
    for at in range(count, left):
        new_free[at] = stack[at]
    return slots, positions, starts, out_lens, left, new_tables, new_free


def plan_inputs(seed, batch, bs, ctx, spare, new, ended=0, width=None):
    r = np.random.default_rng(seed)
    lens = r.integers(0, ctx + 1, batch)
    used = -(-lens // bs)
    width = width or int(-(-(ctx + max(int(max(new)), 0)) // bs)) + 1
    ids = r.permutation(int(used.sum()) + spare + 5)
    tables = np.full((batch, width), -1, np.int64)
    cur = 0
    for i in range(batch):
        tables[i, : used[i]] = ids[cur: cur + used[i]]
        cur += used[i]
    free = np.full(len(ids), -1, np.int64)
    free[:spare] = ids[cur: cur + spare]
    new = np.resize(np.array(new), batch)
    new[r.permutation(batch)[:ended]] = -1
    return lens, new, tables, free, spare


def call(lens, new, tables, free, count, bs, capacity, in_place=False):
    d = lambda x: torch.tensor(np.asarray(x), dtype=I32, device="cuda")  # noqa: E731
    t = [d(lens), d(new), d(tables), d(free), d([count])]
    kw = dict(seq_lens_out=t[0], free_count_out=t[4]) if in_place else {}
    slots, pos, starts, out_lens, left = H.kv_plan_step(*t, bs, capacity, **kw)
    return [x.cpu().numpy() for x in (slots, pos, starts, out_lens)] + [int(left)] + [t[2].cpu().numpy(), t[3].cpu().numpy()]


NAMES = ("slots", "positions", "token_starts", "seq_lens_out", "free_count_out", "block_tables", "free_blocks")


def check(args, bs, capacity, in_place=False):
    want = plan_reference(*args, bs, capacity)
    got = call(*args, bs, capacity, in_place)
    for name, g, w in zip(NAMES, got, want):
        assert np.array_equal(g, w), name
    return want


CASES = [
    # seed, batch, bs, ctx, spare, new lengths (repeated over the batch), ended, capacity beyond the tokens
    (1, 1, 16, 0, 4, [1], 0, 0),               # one token of an empty sequence
    (2, 1, 16, 40, 0, [0], 0, 3),              # nothing to add, nothing free
    (3, 5, 16, 200, 20, [1], 0, 0),            # a decode step
    (4, 7, 16, 31, 9, [17, 1, 0, 33], 2, 4),   # zero, one and many tokens, two ended
    (5, 9, 1, 12, 30, [1, 5], 3, 0),           # blocks of one token
    (6, 6, 48, 500, 11, [100, 1], 1, 2),       # blocks of no power of two
    (7, 64, 16, 300, 12, [40], 4, 0),          # too few blocks: a prefix is served, full blocks need none
    (8, 300, 32, 700, 500, [1, 1, 1, 77], 11, 5),
    (9, 1025, 16, 90, 4000, [3, 1], 40, 0),    # more sequences than the scan's workgroup has threads
    (10, 2500, 16, 40, 1500, [1, 2, 0, 31], 200, 9),
    (11, 3, 16, 5000, 900, [9000, 4000, 1], 0, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[str(c[0]) for c in CASES])
def test_plan_matches_the_host(gpu, case):
    seed, batch, bs, ctx, spare, new, ended, more = case
    args = plan_inputs(seed, batch, bs, ctx, spare, new, ended)
    capacity = int(np.maximum(args[1], 0).sum()) + more
    H.fetch_device_errors()
    check(args, bs, capacity)
    check(args, bs, capacity, in_place=True)
    assert H.fetch_device_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("batch,every,more", [(700, 97, 3000), (1024, 1024, 2100), (3000, 601, 0), (4000, 3, 500), (70000, 9000, 1)])
def test_plan_of_mostly_idle_sequences(gpu, batch, every, more):
    # many sequences between two tokens that are neighbours, and at either end; tokens end inside,
    # at and before the capacity
    args = list(plan_inputs(30, batch, 16, 60, 300, [0]))
    args[1][::every] = np.resize([5, 300, 1], len(args[1][::every]))
    args[1][batch // 2] = 17
    check(args, 16, int(args[1].sum()) + more)
    check(args, 16, int(args[1].sum()) - 20, in_place=True)


@pytest.mark.gpu
def test_plan_refuses_what_does_not_fit(gpu):
    # too few places in the token list, and rows too short for the new tokens: those
    # sequences keep their length and row, the others are served
    args = plan_inputs(20, 40, 16, 100, 300, [5, 60], 3)
    total = int(np.maximum(args[1], 0).sum())
    want = check(args, 16, total - 70)
    assert (want[3] == args[0]).any()
    args = plan_inputs(21, 40, 16, 100, 300, [5, 60], 3, width=7)
    want = check(args, 16, total)
    assert (want[3] == args[0]).any() and (want[3] > args[0]).any()


@pytest.mark.gpu
def test_plan_steps_of_a_serving_loop(gpu):
    # many steps in place, sequences ending and their places taken by new prompts: no block is
    # ever held twice and none is lost
    bs, batch, width, total = 16, 24, 12, 150
    r = np.random.default_rng(3)
    d = lambda x: torch.tensor(np.asarray(x), dtype=I32, device="cuda")  # noqa: E731
    lens, tables = d(np.zeros(batch)), d(np.full((batch, width), -1))
    free, count = d(r.permutation(total)), d([total])
    ws = torch.empty(H.kv_plan_workspace_size(batch), dtype=torch.uint8, device="cuda")
    for step in range(60):
        host = lens.cpu().numpy()
        new = np.where(host == 0, r.integers(0, 50, batch), 1)
        new[(r.random(batch) < 0.05) & (host > 0)] = -1
        args = (host, new, tables.cpu().numpy(), free.cpu().numpy(), int(count))
        cap = int(np.maximum(new, 0).sum()) + 1
        slots, pos, starts, _, _ = H.kv_plan_step(lens, d(new), tables, free, count, bs, cap, seq_lens_out=lens,
                                                  free_count_out=count, workspace=ws)
        want = plan_reference(*args, bs, cap)
        for name, g, w in zip(NAMES, (slots, pos, starts, lens, count, tables, free), want):
            assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1)), (step, name)
        held = [want[5][i, : -(-want[3][i] // bs)] for i in range(batch)]
        everything = np.concatenate(held + [want[6][: want[4]]])
        assert sorted(everything.tolist()) == list(range(total)), step


@pytest.mark.gpu
def test_plan_replays_in_a_graph(gpu):
    # captured once, replayed as the lengths change on the device: every replay equals the host
    bs, batch = 16, 10
    args = plan_inputs(30, batch, bs, 60, 80, [1], 0)
    d = lambda x: torch.tensor(np.asarray(x), dtype=I32, device="cuda")  # noqa: E731
    lens, new, tables, free, count = [d(x) for x in args[:4]] + [d([args[4]])]
    slots = torch.empty(batch * 4, dtype=torch.int64, device="cuda")
    pos = torch.empty_like(slots)
    starts = torch.empty(batch + 1, dtype=I32, device="cuda")
    ws = torch.empty(H.kv_plan_workspace_size(batch), dtype=torch.uint8, device="cuda")
    go = lambda: H.kv_plan_step(lens, new, tables, free, count, bs, slots=slots, positions=pos,  # noqa: E731
                                token_starts=starts, seq_lens_out=lens, free_count_out=count, workspace=ws)
    keep = [x.clone() for x in (lens, tables, free, count)]
    go()  # warm-up outside the capture
    torch.cuda.synchronize()
    for x, k in zip((lens, tables, free, count), keep):
        x.copy_(k)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        go()
    r = np.random.default_rng(1)
    for step in range(6):
        add = r.integers(-1, 5, batch)
        new.copy_(d(add))
        args = [x.cpu().numpy() for x in (lens, new, tables, free)] + [int(count)]
        want = plan_reference(*args, bs, batch * 4)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for name, got, w in zip(NAMES, (slots, pos, starts, lens, count, tables, free), want):
            assert np.array_equal(got.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1)), (step, name)


@pytest.mark.gpu
def test_plan_flags_what_it_cannot_follow(gpu):
    # a negative length, a length beyond its row, a bad table entry, blocks given back twice:
    # flags, slots of -1, everything else as it was
    d = lambda x: torch.tensor(np.asarray(x), dtype=I32, device="cuda")  # noqa: E731

    def go(lens, new, tables, free, count, cap=4):
        H.fetch_device_errors()
        out = H.kv_plan_step(d(lens), d(new), d(tables), d(free), d([count]), 16, cap)
        return [x.cpu().tolist() for x in out], H.fetch_device_errors()

    rows = [[0, 1], [2, 3]]
    out, flags = go([-5, 17], [1, 1], rows, [9, 8, 7, 6, 5, 4, 0, 0, 0, 0], 6)
    assert flags == 8 and out[0] == [-1, 3 * 16 + 1, -1, -1] and out[3] == [-5, 18] and out[1][1] == 17
    out, flags = go([33, 17], [-1, 1], rows, [9, 8, 7, 6, 5, 4, 0, 0, 0, 0], 6)
    assert flags == 8 and out[0] == [3 * 16 + 1, -1, -1, -1] and out[3] == [33, 18] and out[4] == [6]
    out, flags = go([17, 17], [1, 1], [[0, -1], [2, 77]], [9, 8, 7, 6, 5, 4, 0, 0, 0, 0], 6)
    assert flags == 1 and out[0] == [-1, -1, -1, -1]
    out, flags = go([32, 17], [-1, 1], rows, [3, 2, 1], 2)
    assert flags == 9 and out[4] == [3] and out[3] == [0, 18]  # bit 0 too: block 3 of 3 in the second row
    out, flags = go([32, 16], [0, 1], rows, [3, 2, 1], -4)
    assert flags == 8 and out[4] == [0] and out[0][0] == -1


def test_plan_refusals():
    lib = H.lib()
    p = 256  # a pointer that is never followed: every call below is refused on the host

    def go(batch=2, bs=16, nb=8, seq=p, new=p, tables=p, stride=4, n=4, free=p, count=p, cap=3, starts=p, slots=p, pos=p,
           lens_out=p, count_out=p, ws=p, ws_bytes=1 << 20):
        return lib.hcp_kv_plan_step(batch, bs, nb, seq, new, tables, stride, n, free, count, cap, starts, slots, pos,
                                    lens_out, count_out, ws, ws_bytes, None)

    for bad in (dict(batch=0), dict(batch=-1), dict(bs=0), dict(nb=0), dict(nb=1 << 31), dict(cap=-1), dict(cap=1 << 31),
                dict(n=0), dict(stride=3), dict(seq=None), dict(new=None), dict(tables=None), dict(free=None),
                dict(count=None), dict(starts=None), dict(slots=None), dict(pos=None), dict(lens_out=None),
                dict(count_out=None), dict(ws=None), dict(ws_bytes=10), dict(ws=264)):
        assert go(**bad) == -6, bad
        assert H.last_error().startswith("hcp_kv_plan_step:"), bad
    assert lib.hcp_kv_plan_workspace_size(0) == 0 and lib.hcp_kv_plan_workspace_size(-3) == 0
    sizes = [lib.hcp_kv_plan_workspace_size(b) for b in (1, 2, 100, 1000, 5000)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    null = [0 if t in (ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t) else None for t in lib.hcp_kv_plan_step.argtypes]
    assert lib.hcp_kv_plan_step(*null) == -6


def test_plan_python_refusals():
    z = lambda n, dt=I32: torch.zeros(n, dtype=dt)  # noqa: E731
    with pytest.raises(ValueError, match="capacity"):
        H.kv_plan_step(z(2), z(2), z((2, 3)), z(8), z(1), 16)
    with pytest.raises(ValueError, match="new_lens"):
        H.kv_plan_step(z(2), z(3), z((2, 3)), z(8), z(1), 16, 4)
    with pytest.raises(ValueError, match="slots"):
        H.kv_plan_step(z(2), z(2), z((2, 3)), z(8), z(1), 16, slots=z(4))
    with pytest.raises(ValueError, match="block_tables"):
        H.kv_plan_step(z(2), z(2), z((3, 2)).t(), z(8), z(1), 16, 4)
    with pytest.raises(ValueError, match="GPU"):
        H.kv_plan_step(z(2), z(2), z((2, 3)), z(8), z(1), 16, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [3, 1100])
@pytest.mark.parametrize("bad", [-1, 40, 1 << 30])
def test_plan_flags_a_bad_entry_that_an_ended_sequence_gives_back(gpu, batch, bad):
    # one of many blocks that go on the stack, first, second or far along a row; taken again at once, too
    for at in (0, 1, 7):
        lens, new = np.zeros(batch, np.int64), np.zeros(batch, np.int64)
        tables = np.full((batch, 10), -1)
        tables[1] = np.arange(10, 20)
        lens[1], new[1] = 150, -1
        tables[1, at] = bad
        args = (lens, new, tables, np.concatenate([np.arange(10), np.full(30, -1)]), 10)
        H.fetch_device_errors()
        got = call(*args, 16, 1)
        assert H.fetch_device_errors() == 1
        for name, g, w in zip(NAMES, got, plan_reference(*args, 16, 1)):
            assert np.array_equal(g, w), name
        tables[1, at] = 10 + at
        call(*args[:2], tables, *args[3:], 16, 1)
        assert H.fetch_device_errors() == 0
    lens[2], new[2] = 0, 16 * 3  # takes the stack's top: places 9, 8 and 7 of the ended row
    tables[1, 8] = bad
    got = call(lens, new, tables, *args[3:], 16, 48)
    assert H.fetch_device_errors() == 1 and (got[0][16:32] == -1).all() and (got[0][:16] >= 0).all()


def test_plan_refuses_a_capacity_that_sums_stop_at():
    # token offsets are whole numbers of 32 bits that stop at 2^31 - 1: of a list that long none would be past the end
    p = 256
    args = lambda cap: (2, 16, 8, p, p, p, 4, 4, p, p, cap, p, p, p, p, p, p, 10, None)  # noqa: E731
    assert H.lib().hcp_kv_plan_step(*args((1 << 31) - 1)) == -6 and "capacity" in H.last_error()
    assert H.lib().hcp_kv_plan_step(*args((1 << 31) - 2)) == -6 and "workspace" in H.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [3, 1100])
def test_plan_of_more_tokens_than_32_bits_hold(gpu, batch):
    # lengths whose sum passes 2^31 and 2^32: who lies past the capacity is not served, the others are
    lens, new = np.zeros(batch, np.int64), np.zeros(batch, np.int64)
    tables = np.full((batch, 4), -1)
    new[:3] = [20, (1 << 31) - 1, 1]
    if batch > 3:
        new[3:6] = (1 << 31) - 1
        new[batch - 1] = 1
    out = call(lens, new, tables, np.arange(10), 10, 16, 100)
    slots, pos, starts, out_lens, left, got_tables, _ = out
    assert slots[:20].tolist() == [9 * 16 + i for i in range(16)] + [8 * 16 + i for i in range(4)]
    assert (slots[20:] == -1).all() and pos[20:].tolist() == list(range(80))
    assert out_lens[0] == 20 and not out_lens[1:].any() and left == 8 and (got_tables[1:] == -1).all()
    assert starts.tolist() == np.minimum(np.concatenate([[0], np.cumsum(new)]), (1 << 31) - 1).tolist()
