"""Sharing, copying, freeing and moving the blocks of a paged cache (no reference
counterpart; the reference's caches are dense and complete,
kv_cache/new_kvint8.cu:83-84).

The oracles restate the rules of include/kvdecode.h row by row on the host. All
results are whole numbers or copies, so everything is compared for equality."""
import ctypes

import numpy as np
import pytest

import kvdecode as kvd

DEV = "cuda:0"
EINVAL = kvd.CUDA_ERROR_INVALID_VALUE


# --------------------------------------------------------------------- oracles
def fork_oracle(parents, lens, table, free, count, bs):
    """kvd_paged_fork_launch; returns (table, lens, free, count, copies [(src, dst, tokens)], status)."""
    B, MB = table.shape
    NB = len(free)
    lens = np.clip(lens, 0, MB * bs)
    held = -(-lens // bs)
    table_out, free = table.copy(), free.copy()
    status = 0
    good = lambda i: 0 <= i < NB  # noqa: E731
    goes_on = {int(p) for p in parents if 0 <= p < B}
    kept, ended = set(), set()
    for b in range(B):
        for i in table[b, : held[b]]:
            if good(i):
                (kept if b in goes_on else ended).add(int(i))
            else:
                status |= kvd.KVD_STATUS_BAD_BLOCK
    count = min(max(0, int(count)), NB)
    for i in sorted(ended - kept):
        if count < NB:
            free[count] = i
            count += 1
        else:
            status |= kvd.KVD_STATUS_BAD_BLOCK
    lens_out, copies, taken, refused = np.zeros_like(lens), [], {}, False
    for p in goes_on:
        rows = [b for b in range(B) if parents[b] == p]
        taken[p] = p if p in rows else rows[0]
    for b in range(B):
        p = int(parents[b])
        if not 0 <= p < B:
            continue
        row, tail = table[p, : held[p]].copy(), int(lens[p]) % bs
        if tail and taken[p] != b and good(row[-1]):
            refused = refused or count == 0
            if refused:
                status |= kvd.KVD_STATUS_NO_BLOCKS
                continue
            count -= 1
            if good(free[count]):
                copies.append((int(row[-1]), int(free[count]), tail))
            else:
                status |= kvd.KVD_STATUS_BAD_BLOCK
            row[-1] = free[count]
        table_out[b, : held[p]] = row
        lens_out[b] = lens[p]
    return table_out, lens_out, free, count, copies, status


def compact_oracle(lens, table, free, count, bs):
    """kvd_paged_compact_launch; returns (table, free, count, used, moves [(src, dst)], status)."""
    B, MB = table.shape
    NB = len(free)
    held = -(-np.clip(lens, 0, MB * bs) // bs)
    status = 0
    good = lambda i: 0 <= i < NB  # noqa: E731
    use = set()
    for b in range(B):
        for i in table[b, : held[b]]:
            if good(i):
                use.add(int(i))
            else:
                status |= kvd.KVD_STATUS_BAD_BLOCK
    given = [int(i) for i in free[: min(max(0, int(count)), NB)]]
    if any(not good(i) for i in given):
        status |= kvd.KVD_STATUS_BAD_BLOCK
    spare = {i for i in given if good(i)} - use
    both = sorted(use | spare)
    low, rest = set(both[: len(use)]), both[len(use):]
    moves = list(zip(sorted(use - low), sorted(low - use)))
    to = dict(moves)
    table_out, free_out = table.copy(), free.copy()
    for b in range(B):
        table_out[b, : held[b]] = [to.get(int(i), i) for i in table[b, : held[b]]]
    free_out[: len(rest)] = rest[::-1]
    return table_out, free_out, len(rest), max(low) + 1 if low else 0, moves, status


# ------------------------------------------------------------------- tensors
def make_pools(NB, H, bs, D, layout, seed, offset=0, pad=0):
    """Pools with every code drawn; `offset` bytes off their allocation, `pad` unused dims behind each row."""
    import torch

    gen = torch.Generator(device=DEV).manual_seed(seed)
    shape = (NB, H, bs, D + pad) if layout == "bhtd" else (NB, bs, H, D + pad)
    n = int(np.prod(shape))
    codes = [torch.randint(-128, 128, (n + offset,), dtype=torch.int8, device=DEV, generator=gen)[offset:].view(shape)[..., :D]
             for _ in range(2)]
    scales = [torch.rand((NB, H, bs), device=DEV, generator=gen) for _ in range(2)]
    bounds = torch.randint(-128, 128, (NB, H, 2, D), dtype=torch.int8, device=DEV, generator=gen)
    return [*codes, *scales, bounds, torch.rand((NB, H), device=DEV, generator=gen)]


def snapshot(pools):
    return [None if t is None else t.cpu().numpy().copy() for t in pools]


def apply_copies(before, copies, layout, bs):
    """The pools after copies (src, dst, tokens); sources are never destinations."""
    out = [None if a is None else a.copy() for a in before]
    for src, dst, n in copies:
        for x in range(2):
            at = (slice(None), slice(0, n)) if layout == "bhtd" else (slice(0, n),)
            out[x][(dst, *at)] = before[x][(src, *at)]
            out[2 + x][dst, :, :n] = before[2 + x][src, :, :n]
        for x in (4, 5):
            if out[x] is not None:
                out[x][dst] = before[x][src]
    return out


def same(pools, want):
    for got, ref in zip(pools, want):
        if ref is not None:
            np.testing.assert_array_equal(got.cpu().numpy().view(np.uint8 if ref.itemsize == 1 else np.uint32),
                                          ref.view(np.uint8 if ref.itemsize == 1 else np.uint32))


def dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).to(DEV)


def random_rows(rng, B, MB, bs, NB, lens, share=0.0, taken=()):
    """A table whose rows hold blocks of their own, or (share) the first blocks of the row before; and the ids left."""
    ids = [i for i in rng.permutation(NB) if i not in taken]
    table = rng.integers(-5, NB + 5, size=(B, MB)).astype(np.int32)  # entries behind a row's blocks are anything
    at = 0
    for b in range(B):
        n = -(-int(np.clip(lens[b], 0, MB * bs)) // bs)
        first = 0
        if b and rng.random() < share:
            first = min(n, -(-int(np.clip(lens[b - 1], 0, MB * bs)) // bs) - 1)
            first = int(rng.integers(0, max(0, first) + 1))
            table[b, :first] = table[b - 1, :first]
        table[b, first:n] = ids[at: at + n - first]
        at += n - first
    return table, np.array(ids[at:], np.int32)


def run_fork(parents, lens, table, free, count, bs, pools, layout, in_place, ws=None, stream=None):
    import torch

    B, MB = table.shape
    t = {"lens": dev(lens), "table": dev(table), "free": dev(free), "count": dev([count])}
    out = {} if in_place else {"seq_lens_out": torch.full((B,), -7, dtype=torch.int32, device=DEV),
                               "block_table_out": t["table"].clone(),
                               "free_count_out": torch.full((1,), -7, dtype=torch.int32, device=DEV)}
    got_table, got_lens = kvd.paged_fork(dev(parents), t["lens"], t["table"], t["free"], t["count"], *pools[:4],
                                         bounds=pools[4], bound_scale=pools[5], layout=layout, workspace=ws,
                                         stream=stream, **out)
    if in_place:
        assert got_table is t["table"] and got_lens is t["lens"]
    else:
        assert got_table is out["block_table_out"]
        np.testing.assert_array_equal(t["table"].cpu().numpy(), table)  # inputs stay
        np.testing.assert_array_equal(t["lens"].cpu().numpy(), lens)
    return got_table, got_lens, t["free"], t["count"] if in_place else out["free_count_out"]


def check_fork(parents, lens, table, free, count, bs, pools, layout, in_place, ws=None):
    before = snapshot(pools)
    want = fork_oracle(np.asarray(parents), np.asarray(lens), table, free, count, bs)
    got = run_fork(parents, lens, table, free, count, bs, pools, layout, in_place, ws)
    for g, w in zip(got, want[:4]):
        np.testing.assert_array_equal(g.cpu().numpy().reshape(-1), np.asarray(w, np.int32).reshape(-1))
    same(pools, apply_copies(before, want[4], layout, bs))
    assert kvd.device_status() == want[5]
    return want


# ------------------------------------------------------------------- fork, GPU
@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("B,MB,bs,H,D,layout,bounds", [
    (1, 1, 1, 1, 1, "bhtd", False),
    (2, 3, 16, 2, 128, "bthd", True),
    (7, 5, 8, 3, 64, "bhtd", True),
    (33, 300, 4, 1, 20, "bthd", False),   # table rows of more than one stretch, 4-byte codes
    (64, 9, 5, 2, 7, "bhtd", True),       # odd block size, single bytes
    (700, 4, 16, 1, 96, "bhtd", False),   # more rows than threads
])
def test_fork_matches_rule(B, MB, bs, H, D, layout, bounds, in_place):
    rng = np.random.default_rng(B * 100 + bs)
    lens = rng.integers(0, MB * bs + 1, size=B)
    lens[rng.random(B) < 0.2] = 0
    lens[rng.random(B) < 0.2] //= bs
    lens[rng.random(B) < 0.3] //= bs * bs
    lens = np.where(rng.random(B) < 0.3, lens // bs * bs, lens)  # nothing to copy
    need = int((-(-lens // bs)).sum())
    NB = need + B + 11
    table, left = random_rows(rng, B, MB, bs, NB, lens, share=0.5)
    parents = rng.integers(-1, B, size=B)
    parents[rng.random(B) < 0.1] = B + 3
    free = np.full(NB, -1, np.int32)
    count = min(len(left), B)
    free[:count] = left[:count]
    pools = make_pools(NB, H, bs, D, layout, B)
    if not bounds:
        pools[4] = pools[5] = None
    check_fork(parents, lens, table, free, count, bs, pools, layout, in_place)


@pytest.mark.gpu
@pytest.mark.parametrize("spare", [0, 1, 3])
def test_fork_refuses_copies_when_the_stack_is_empty(spare):
    lens = np.array([5, 0, 0, 0, 0, 9])
    table = np.full((6, 4), -1, np.int32)
    table[0, :2], table[5, :3] = [3, 8], [1, 4, 6]
    free = np.full(12, -1, np.int32)
    free[:3] = [0, 10, 7]
    want = check_fork([0, 0, 0, 0, 0, -1], lens, table, free, spare, 4, make_pools(12, 2, 4, 16, "bhtd", 1), "bhtd", True)
    # row 5's three blocks go on the stack first: copies for as many rows as there are blocks
    assert (want[1] == 0).sum() == 1 + max(0, 4 - (3 + spare))


@pytest.mark.gpu
def test_fork_all_rows_end_and_all_stay():
    rng = np.random.default_rng(3)
    lens = np.array([40, 0, 17, 64])
    table, left = random_rows(rng, 4, 4, 16, 20, lens)
    free = np.full(20, -1, np.int32)
    free[: len(left)] = left
    pools = make_pools(20, 2, 16, 32, "bthd", 2)
    want = check_fork([-1] * 4, lens, table, free, len(left), 16, pools, "bthd", True)
    assert want[3] == 20
    want = check_fork([0, 1, 2, 3], lens, table, free, len(left), 16, pools, "bthd", True)
    assert want[4] == [] and want[3] == len(left)


@pytest.mark.gpu
def test_fork_with_ids_outside_the_pool():
    lens = np.array([20, 33, 20])
    table = np.array([[2, 99], [-3, 5], [7, 1]], np.int32)
    table = np.concatenate([table, np.full((3, 1), 4, np.int32)], axis=1)
    free = np.full(10, -1, np.int32)
    free[:2] = [12, 9]  # one bad id on the free list too
    pools = make_pools(10, 1, 16, 16, "bhtd", 4)
    want = check_fork([0, 0, 2], lens, table, free, 2, 16, pools, "bhtd", True)
    assert want[5] & kvd.KVD_STATUS_BAD_BLOCK
    check_fork([2, 2, 2], lens, table, np.array([12] + [-1] * 9, np.int32), 1, 16, pools, "bhtd", False)


@pytest.mark.gpu
def test_fork_of_a_full_list_stops_at_its_end():
    # a free list that also names blocks of a row: their second entry has no room
    lens = np.array([32, 16])
    table = np.array([[0, 1], [2, 3]], np.int32)
    free = np.arange(4, dtype=np.int32)
    want = check_fork([-1, 1], lens, table, free, 4, 16, make_pools(4, 1, 16, 16, "bhtd", 5), "bhtd", True)
    assert want[5] == kvd.KVD_STATUS_BAD_BLOCK and want[3] == 4


@pytest.mark.gpu
@pytest.mark.parametrize("offset,pad", [(0, 16), (4, 0), (1, 3)])
def test_fork_of_pools_off_alignment(offset, pad):
    rng = np.random.default_rng(offset)
    lens = np.array([21, 0, 50, 3])
    table, left = random_rows(rng, 4, 4, 16, 30, lens)
    free = np.full(30, -1, np.int32)
    free[: len(left)] = left
    for layout in ("bhtd", "bthd"):
        pools = make_pools(30, 3, 16, 32, layout, 6, offset, pad)
        check_fork([2, 0, 2, 2], lens, table, free, len(left), 16, pools, layout, True)


@pytest.mark.gpu
def test_fork_steps_in_one_graph_and_on_two_streams():
    """Beam steps captured once and replayed: each replay continues from the state that the last one left."""
    import torch

    rng = np.random.default_rng(8)
    B, MB, bs, NB = 12, 6, 8, 120
    lens = rng.integers(1, MB * bs, size=B)
    table, left = random_rows(rng, B, MB, bs, NB, lens)
    free = np.full(NB, -1, np.int32)
    free[: len(left)] = left
    parents = np.array([0, 0, 0, 5, 4, 4, 6, 6, 8, -1, 9, 11])
    pools = make_pools(NB, 2, bs, 32, "bhtd", 7)
    host = snapshot(pools)
    t = [dev(lens), dev(table), dev(free), dev([len(left)])]
    d_parents = dev(parents)
    ws = torch.zeros(kvd.paged_fork_workspace_size(t[1], t[2]), dtype=torch.uint8, device=DEV)
    call = lambda: kvd.paged_fork(d_parents, *t, *pools[:4], bounds=pools[4], bound_scale=pools[5], workspace=ws)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    state = (table, lens, free, len(left))
    for _ in range(3):
        graph.replay()
        tb, ln, fr, ct, copies, status = fork_oracle(parents, state[1], state[0], state[2], state[3], bs)
        host = apply_copies(host, copies, "bhtd", bs)
        state = (tb, ln, fr, ct)
        for g, w in zip(t, (ln, tb, fr, [ct])):
            np.testing.assert_array_equal(g.cpu().numpy(), np.asarray(w, np.int32))
        same(pools, host)
    assert int(ws.view(torch.int32)[0]) == 0 and kvd.device_status() in (0, kvd.KVD_STATUS_NO_BLOCKS)
    # another stream than the current one, scratch made by the call
    with torch.cuda.stream(side):
        pass
    side.wait_stream(torch.cuda.current_stream())
    kvd.paged_fork(d_parents, *t, *pools[:4], bounds=pools[4], bound_scale=pools[5], stream=side)
    side.synchronize()
    tb, ln, fr, ct, copies, _ = fork_oracle(parents, state[1], state[0], state[2], state[3], bs)
    for g, w in zip(t, (ln, tb, fr, [ct])):
        np.testing.assert_array_equal(g.cpu().numpy(), np.asarray(w, np.int32))
    same(pools, apply_copies(host, copies, "bhtd", bs))
    kvd.device_status()


# ---------------------------------------------------------------- compact, GPU
def check_compact(lens, table, free, count, bs, pools, layout, in_place, ws=None):
    import torch

    before = snapshot(pools)
    want = compact_oracle(np.asarray(lens), table, free, count, bs)
    t = [dev(lens), dev(table), dev(free), dev([count])]
    out = {} if in_place else {"block_table_out": t[1].clone(), "free_blocks_out": t[2].clone(),
                               "used": torch.full((1,), -7, dtype=torch.int32, device=DEV)}
    used = kvd.paged_compact(*t, *pools[:4], bounds=pools[4], bound_scale=pools[5], layout=layout, workspace=ws, **out)
    got_table, got_free = (t[1], t[2]) if in_place else (out["block_table_out"], out["free_blocks_out"])
    for g, w in zip((got_table, got_free, t[3], used), want[:4]):
        np.testing.assert_array_equal(g.cpu().numpy().reshape(-1), np.asarray(w, np.int32).reshape(-1))
    same(pools, apply_copies(before, [(s, d, bs) for s, d in want[4]], layout, bs))
    assert kvd.device_status() == want[5]
    if not in_place:
        np.testing.assert_array_equal(t[1].cpu().numpy(), table)
        np.testing.assert_array_equal(t[2].cpu().numpy(), free)
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("B,MB,bs,NB,H,D,layout,bounds", [
    (1, 1, 1, 1, 1, 1, "bhtd", False),
    (3, 4, 16, 31, 2, 128, "bthd", True),
    (5, 40, 8, 400, 1, 64, "bhtd", True),
    (17, 300, 3, 9001, 1, 12, "bthd", False),
    (40, 30, 7, 1311, 2, 5, "bhtd", True),
])
def test_compact_matches_rule(B, MB, bs, NB, H, D, layout, bounds, in_place):
    for fill in (0.0, 0.4, 1.0):
        rng = np.random.default_rng(int(B + 10 * fill))
        most = min(NB // B, MB) * bs
        lens = (rng.integers(0, most + 1, size=B) * fill).astype(np.int64)
        table, left = random_rows(rng, B, MB, bs, NB, lens, share=0.4)
        free = np.full(NB, -9, np.int32)
        count = len(left) - (len(left) // 5 if fill == 0.4 else 0)  # some blocks belong to others
        free[:count] = left[:count]
        pools = make_pools(NB, H, bs, D, layout, B)
        if not bounds:
            pools[4] = pools[5] = None
        check_compact(lens, table, free, count, bs, pools, layout, in_place)


@pytest.mark.gpu
def test_compact_with_bad_ids_and_twice():
    import torch

    lens = np.array([48, 20])
    table = np.array([[18, 55, 3], [-2, 11, 11]], np.int32)
    free = np.array([0, 1, 1, 40, -3, 18] + [-1] * 14, np.int32)  # twice the same, outside the pool, in use
    pools = make_pools(20, 2, 16, 32, "bhtd", 9)
    want = check_compact(lens, table, free, 6, 16, pools, "bhtd", False)
    assert want[5] == kvd.KVD_STATUS_BAD_BLOCK
    # a second call finds nothing to move; one scratch for both
    rng = np.random.default_rng(1)
    lens = rng.integers(1, 60, size=6)
    table, left = random_rows(rng, 6, 4, 16, 60, lens)
    free = np.full(60, -1, np.int32)
    free[: len(left)] = left
    pools = make_pools(60, 1, 16, 32, "bthd", 9)
    ws = torch.zeros(kvd.paged_compact_workspace_size(dev(table), dev(free)), dtype=torch.uint8, device=DEV)
    first = check_compact(lens, table, free, len(left), 16, pools, "bthd", True, ws)
    assert first[3] == int((-(-lens // 16)).sum()) and first[4]
    second = check_compact(lens, first[0], first[1], first[2], 16, pools, "bthd", True, ws)
    assert second[4] == [] and second[3] == first[3]


@pytest.mark.gpu
def test_compact_in_a_graph():
    import torch

    rng = np.random.default_rng(2)
    lens = rng.integers(1, 100, size=9)
    table, left = random_rows(rng, 9, 7, 16, 200, lens)
    free = np.full(200, -1, np.int32)
    free[: len(left)] = left
    pools = make_pools(200, 2, 16, 64, "bhtd", 3)
    host = snapshot(pools)
    t = [dev(lens), dev(table), dev(free), dev([len(left)])]
    used = dev([0])
    ws = torch.zeros(kvd.paged_compact_workspace_size(t[1], t[2]), dtype=torch.uint8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kvd.paged_compact(*t, *pools[:4], bounds=pools[4], bound_scale=pools[5], used=used, workspace=ws)
    state = (table, free, len(left))
    for _ in range(2):
        tb, fr, ct, us, moves, _ = compact_oracle(lens, state[0], state[1], state[2], 16)
        graph.replay()
        host = apply_copies(host, [(s, d, 16) for s, d in moves], "bhtd", 16)
        state = (tb, fr, ct)
        for g, w in zip((t[1], t[2], t[3], used), (tb, fr, [ct], [us])):
            np.testing.assert_array_equal(g.cpu().numpy(), np.asarray(w, np.int32))
        same(pools, host)
    assert kvd.device_status() == 0


@pytest.mark.gpu
def test_blocks_past_32_bits():
    """Pools of more than 2^32 codes: copies and moves at both ends."""
    import torch

    NB, H, bs, D = 34000, 8, 128, 128
    pools = [torch.zeros((NB, H, bs, D), dtype=torch.int8, device=DEV) for _ in range(2)]
    pools += [torch.zeros((NB, H, bs), device=DEV) for _ in range(2)]
    assert pools[0].numel() > 1 << 32
    last = NB - 1
    gen = torch.Generator(device=DEV).manual_seed(1)
    marks = []
    for t in pools[:2]:
        t[last] = torch.randint(-128, 128, (H, bs, D), dtype=torch.int8, device=DEV, generator=gen)
        marks.append(t[last].clone())
    for t in pools[2:]:
        t[last] = torch.rand((H, bs), device=DEV, generator=gen)
        marks.append(t[last].clone())
    lens, table, free, count = dev([100, 0]), dev([[last], [5]]), dev([last - 1, 0] + [-1] * (NB - 2)), dev([1])
    kvd.paged_fork(dev([0, 0]), lens, table, free, count, *pools)
    assert table.tolist() == [[last], [last - 1]] and lens.tolist() == [100, 100] and int(count) == 0
    for t, m in zip(pools, marks):
        assert torch.equal(t[last - 1, :, :100], m[:, :100]) and not t[last - 1, :, 100:].any()
    count.fill_(2)
    free[:2] = dev([7, 3])
    used = kvd.paged_compact(lens, table, free, count, *pools)
    assert table.tolist() == [[7], [3]] and int(used) == 8 and free[:2].tolist() == [last, last - 1]
    for t, m in zip(pools, marks):
        assert torch.equal(t[7], m) and torch.equal(t[3, :, :100], m[:, :100])
    assert kvd.device_status() == 0


@pytest.mark.gpu
def test_fork_and_compact_share_a_workspace():
    import torch

    rng, B, MB, bs, NB = np.random.default_rng(5), 9, 40, 8, 500
    ws = torch.zeros(max(f(torch.empty((B, MB)), torch.empty(NB)) for f in (
        kvd.paged_fork_workspace_size, kvd.paged_compact_workspace_size)), dtype=torch.uint8, device=DEV)
    pools = make_pools(NB, 2, bs, 64, "bhtd", 6)
    lens = rng.integers(0, MB * bs + 1, size=B)
    table, left = random_rows(rng, B, MB, bs, NB, lens, share=0.4)
    free, count = np.full(NB, -1, np.int32), len(left)
    free[:count] = left
    for step in range(3):  # every step takes over what the one before left
        table, lens, free, count, *_ = check_fork(rng.integers(-1, B, size=B), lens, table, free, count, bs, pools, "bhtd",
                                                  True, ws)
        table, free, count, *_ = check_compact(lens, table, free, count, bs, pools, "bhtd", True, ws)


@pytest.mark.gpu
def test_pools_of_two_layers_share_a_table():
    import torch

    rng, B, MB, bs, NB = np.random.default_rng(8), 6, 12, 16, 90
    layers = [make_pools(NB, 2, bs, 32, "bhtd", s) for s in (1, 2)]
    lens = rng.integers(1, MB * bs + 1, size=B)
    table, left = random_rows(rng, B, MB, bs, NB, lens)
    free, count = np.full(NB, -1, np.int32), len(left)
    free[:count] = left
    parents = rng.integers(0, B, size=B)
    fork = fork_oracle(parents, lens, table, free, count, bs)
    move = compact_oracle(fork[1], *fork[:1], fork[2], fork[3], bs)
    before = [snapshot(p) for p in layers]
    t = [dev(lens), dev(table), dev(free), dev([count])]
    other = [torch.empty_like(x) for x in t]
    for i, pools in enumerate(layers):  # the last one updates what they share
        own = {} if i else dict(seq_lens_out=other[0], block_table_out=other[1], free_count_out=other[3])
        kvd.paged_fork(dev(parents), *t, *pools[:4], bounds=pools[4], bound_scale=pools[5], **own)
    for x, w in zip((t[1], t[0], t[2], t[3]), fork):
        np.testing.assert_array_equal(x.cpu().numpy().reshape(-1), np.asarray(w, np.int32).reshape(-1))
    for i, pools in enumerate(layers):
        own = {} if i else dict(block_table_out=other[1], free_blocks_out=other[2])
        kvd.paged_compact(t[0], t[1], t[2], t[3] if i else t[3].clone(), *pools[:4], bounds=pools[4], bound_scale=pools[5], **own)
    for x, w in zip((t[1], t[2], t[3]), move):
        np.testing.assert_array_equal(x.cpu().numpy().reshape(-1), np.asarray(w, np.int32).reshape(-1))
    for pools, was in zip(layers, before):
        same(pools, apply_copies(apply_copies(was, fork[4], "bhtd", bs), [(s, d, bs) for s, d in move[4]], "bhtd", bs))
    assert kvd.device_status() == 0


# ------------------------------------------------------------------------ CPU
def pages_desc(**kw):
    d = kvd.PagesDesc(4, 2, 64, 16, 100, 8, 8, 8, 2 * 16 * 64, 16 * 64, 64, 32, 16)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [dict(batch=0), dict(batch=8193), dict(num_kv_heads=0), dict(head_dim=0), dict(block_size=0),
                                dict(num_blocks=0), dict(num_blocks=(1 << 30) + 1), dict(max_blocks_per_seq=0),
                                dict(block_table_stride=7), dict(block_table_out_stride=7),
                                dict(block_size=1, max_blocks_per_seq=(1 << 30) + 1, block_table_stride=1 << 31,
                                     block_table_out_stride=1 << 31),
                                dict(max_blocks_per_seq=1 << 28, block_table_stride=1 << 28, block_table_out_stride=1 << 28),
                                dict(block_size=1 << 24, head_dim=64, max_blocks_per_seq=2)])
def test_bad_descriptors_are_refused(kw):
    L, d = kvd.lib(), pages_desc(**kw)
    assert L.kvd_paged_fork_workspace_size(ctypes.byref(d)) == 0
    assert L.kvd_paged_compact_workspace_size(ctypes.byref(d)) == 0
    assert L.kvd_paged_fork_launch(ctypes.byref(d), *[256 * i for i in range(1, 16)], 4096, 1 << 40, None) == EINVAL
    assert L.kvd_paged_compact_launch(ctypes.byref(d), *[256 * i for i in range(1, 15)], 4096, 1 << 40, None) == EINVAL


def test_bad_arguments_are_refused():
    L, d = kvd.lib(), pages_desc()
    # d, parents, lens, table, free, count, K, V, ks, vs, bounds, bound_scale, lens_out, table_out, count_out, ws, bytes
    fork = [ctypes.byref(d), *[256 * i for i in range(1, 16)], L.kvd_paged_fork_workspace_size(ctypes.byref(d)), None]
    for i in list(range(0, 16)):
        assert L.kvd_paged_fork_launch(*fork[:i], None, *fork[i + 1:]) == EINVAL, i
    assert L.kvd_paged_fork_launch(*fork[:16], fork[16] - 1, None) == EINVAL
    assert L.kvd_paged_fork_launch(*fork[:15], 4098, *fork[16:]) == EINVAL
    other = pages_desc(block_table_out_stride=9)  # in place, the rows lie where they lay
    assert L.kvd_paged_fork_launch(ctypes.byref(other), *fork[1:13], fork[3], *fork[14:]) == EINVAL
    assert L.kvd_paged_fork_launch(*fork[:12], fork[1], *fork[13:]) == EINVAL  # lengths written over the parents
    compact = [ctypes.byref(d), *[256 * i for i in range(1, 15)], L.kvd_paged_compact_workspace_size(ctypes.byref(d)), None]
    for i in list(range(0, 15)):
        assert L.kvd_paged_compact_launch(*compact[:i], None, *compact[i + 1:]) == EINVAL, i
    assert L.kvd_paged_compact_launch(*compact[:15], compact[15] - 1, None) == EINVAL
    assert L.kvd_paged_compact_launch(*compact[:14], 4098, *compact[15:]) == EINVAL
    assert L.kvd_paged_compact_launch(ctypes.byref(other), *compact[1:11], compact[2], *compact[12:]) == EINVAL


def test_tensors_of_wrong_shapes_are_refused():
    import torch

    i32 = torch.int32
    pools = [torch.zeros((10, 2, 16, 32), dtype=torch.int8) for _ in range(2)] + [torch.zeros((10, 2, 16)) for _ in range(2)]
    lens, table, free, count = (torch.zeros(s, dtype=i32) for s in ((4,), (4, 3), (10,), (1,)))
    parents = torch.zeros(4, dtype=i32)
    calls = [lambda **k: kvd.paged_fork(k.get("parents", parents), k.get("lens", lens), k.get("table", table),
                                        k.get("free", free), k.get("count", count), *pools, **k.get("more", {})),
             lambda **k: kvd.paged_compact(k.get("lens", lens), k.get("table", table), k.get("free", free),
                                           k.get("count", count), *pools, **k.get("more", {}))]
    for call in calls:
        for bad in (dict(lens=lens.long()), dict(table=torch.zeros((5, 3), dtype=i32)), dict(free=free[:9]),
                    dict(count=torch.zeros(2, dtype=i32)), dict(more=dict(bounds=torch.zeros((10, 2, 2, 32), dtype=torch.int8))),
                    dict(more=dict(block_table_out=torch.zeros((4, 2), dtype=i32))), dict(more=dict(layout="tbhd"))):
            with pytest.raises(ValueError):
                call(**bad)
        with pytest.raises(ValueError, match="current CUDA device"):
            call()
    with pytest.raises(ValueError):
        calls[0](parents=parents[:3])
    with pytest.raises(ValueError):
        calls[1](more=dict(free_blocks_out=free[:9]))
