"""Paged serving steps: block tables and slot maps, slot writes and reads, block
selection, decode over selected blocks (no reference counterpart; the
reference's caches are dense and complete, kv_cache/new_kvint8.cu:83-84).

Oracles are plain numpy restatements of the rules in include/kvdecode.h: the
plan is run request by request, codes come from the C quantiser of the test
oracle, bounds, scores and attention are computed in 64 bits (rounded to fp32
where the rule says fp32). Plans, codes, bounds and selections are compared
exactly; attention within 2e-5 + 1e-4 |ref| (the framework's decode tolerance)
plus half a unit in the last place of a 16-bit output."""
import ctypes

import numpy as np
import pytest

import kvdecode as kvd
import pyoracle as po

DEV = "cuda:0"
EINVAL = kvd.CUDA_ERROR_INVALID_VALUE


# --------------------------------------------------------------------- oracles
def plan_oracle(lens, new, table, free, count, bs, num_slots):
    """kvd_paged_plan_launch, one request after the other; returns (table, free, count, lens, starts, slots, status)."""
    table, free, lens_out = table.copy(), free.copy(), np.zeros_like(lens)
    B, MB = table.shape
    NB = len(free)
    cap = MB * bs
    lens = np.clip(lens, 0, cap)
    stack = list(free[: min(max(0, int(count)), NB)])
    status = 0
    for b in range(B):
        if new[b] < 0:
            stack += list(table[b, : -(-int(lens[b]) // bs)])
    total, wanted, tokens = len(stack), 0, 0
    starts = [0]
    slots = np.full(num_slots, -1, np.int64)
    for b in range(B):
        n, ln = int(new[b]), int(lens[b])
        held = -(-ln // bs)
        if n < 0:
            starts.append(min(tokens, num_slots))
            continue
        lens_out[b] = ln
        first = tokens
        tokens += n
        starts.append(min(tokens, num_slots))
        if n > 0 and (ln + n > cap or tokens > num_slots):
            status |= kvd.KVD_STATUS_CACHE_FULL
            continue
        need = -(-(ln + n) // bs) - held
        wanted += need
        if need and wanted > total:
            status |= kvd.KVD_STATUS_NO_BLOCKS
            continue
        for j in range(held, held + need):
            table[b, j] = stack.pop()
        lens_out[b] = ln + n
        for i in range(n):
            blk = int(table[b, (ln + i) // bs])
            if 0 <= blk < NB:
                slots[first + i] = blk * bs + (ln + i) % bs
            else:
                status |= kvd.KVD_STATUS_BAD_BLOCK
    c0 = min(max(0, int(count)), NB)
    for i in range(c0, len(stack)):
        if i < NB:
            free[i] = stack[i]
        else:
            status |= kvd.KVD_STATUS_BAD_BLOCK
    return table, free, min(len(stack), NB), lens_out, np.array(starts, np.int32), slots, status


def bounds_oracle(codes, scales):
    """Bound codes [2][D] and step of one block's keys: codes [n][D] int8, scales [n] fp32."""
    if not np.isfinite(scales).all():
        return np.zeros((2, codes.shape[1]), np.int8), np.float32(np.nan)
    x = codes.astype(np.float32) * scales.astype(np.float32)[:, None]
    hi, lo = x.max(0), x.min(0)
    step = np.float32(max(np.abs(hi).max(), np.abs(lo).max())) / np.float32(127)
    if not step > 0:
        return np.zeros((2, codes.shape[1]), np.int8), np.float32(step)
    up = np.clip(np.ceil(hi / step), -127, 127)
    down = np.clip(np.floor(lo / step), -127, 127)
    return np.stack([up, down]).astype(np.int8), step


def select_oracle(q, bounds, step, table, lens, bs, k, first, last):
    """Selection rule in whole numbers and fp32 products; q [B,Hq,D] fp32."""
    B, Hq, D = q.shape
    NB, H = step.shape
    G, MB = Hq // H, table.shape[1]
    sel = np.full((B, H, k), -1, np.int32)
    sel_lens = np.zeros((B, H), np.int32)
    qc, qs = po.quantize_rows(q)
    for b in range(B):
        ln = int(np.clip(lens[b], 0, MB * bs))
        n = -(-ln // bs)
        for h in range(H):
            if n <= k:
                idx = np.arange(n)
                sel_lens[b, h] = ln
            else:
                ids = table[b, :n]
                good = (ids >= 0) & (ids < NB)
                bd = bounds[np.where(good, ids, 0), h].astype(np.int64)
                c = qc[b, h * G:(h + 1) * G].astype(np.int64)
                dots = np.maximum(c, 0) @ bd[:, 0].T + np.minimum(c, 0) @ bd[:, 1].T
                with np.errstate(all="ignore"):
                    v = dots.astype(np.float32) * qs[b, h * G:(h + 1) * G].astype(np.float32)[:, None]
                    v = np.where(np.isnan(v), np.inf, v).max(0).astype(np.float32)
                    s = v * step[np.where(good, ids, 0), h]
                s = np.where(np.isnan(s), np.inf, s).astype(np.float64)
                s = np.where(good, s, -np.inf)
                rank = np.zeros(n)
                rank[good] = 1
                rank[:first] = 2
                rank[n - last:] = 2
                order = sorted(range(n), key=lambda i: (-rank[i], -s[i] if rank[i] == 1 else 0.0, i))
                idx = np.sort(np.array(order[:k]))
                sel_lens[b, h] = (k - n) * bs + ln
            sel[b, h, : len(idx)] = table[b, idx]
    return sel, sel_lens


def sparse_oracle(q, Kp, Vp, ksp, vsp, sel, sel_lens, layout, scale=None):
    """Attention over the selected tokens in 64 bits."""
    B, Hq, D = q.shape
    H = sel.shape[1]
    G, bs = Hq // H, ksp.shape[2]
    out = np.zeros((B, Hq, D))
    scale = scale or 1.0 / np.sqrt(D)
    for b in range(B):
        for h in range(H):
            n = min(int(max(0, sel_lens[b, h])), sel.shape[2] * bs)
            if n == 0:
                continue
            ids = sel[b, h, : -(-n // bs)]
            rows = (lambda p: p[ids, h]) if layout == "bhtd" else (lambda p: p[ids, :, h])
            K = rows(Kp).reshape(-1, D)[:n].astype(np.float64) * ksp[ids, h].reshape(-1)[:n, None].astype(np.float64)
            V = rows(Vp).reshape(-1, D)[:n].astype(np.float64) * vsp[ids, h].reshape(-1)[:n, None].astype(np.float64)
            s = q[b, h * G:(h + 1) * G].astype(np.float64) @ K.T * scale
            p = np.exp(s - s.max(1, keepdims=True))
            out[b, h * G:(h + 1) * G] = (p / p.sum(1, keepdims=True)) @ V
    return out


# ------------------------------------------------------------- inputs
def plan_inputs(seed, B, bs, MB, spare, ends=0, prompts=0, prompt_len=100):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, MB * bs * 3 // 4 + 1, B).astype(np.int32)
    new = rng.integers(0, 3, B).astype(np.int32)
    who = rng.permutation(B)
    new[who[:ends]] = -1
    new[who[ends: ends + prompts]] = rng.integers(1, prompt_len + 1, len(who[ends: ends + prompts]))
    held = -(-lens // bs)
    NB = int(held.sum()) + spare + 1
    ids = rng.permutation(NB).astype(np.int32)
    table = np.full((B, MB), -7, np.int32)
    at = 0
    for b in range(B):
        table[b, : held[b]] = ids[at: at + held[b]]
        at += held[b]
    free = np.full(NB, -9, np.int32)
    free[:spare] = ids[at: at + spare]
    return lens, new, table, free, spare


def pools(seed, NB, H, bs, D, layout):
    rng = np.random.default_rng(seed)
    shape = (NB, H, bs, D) if layout == "bhtd" else (NB, bs, H, D)
    Kp, Vp = (rng.integers(-127, 128, size=shape, dtype=np.int8) for _ in range(2))
    ksp, vsp = (rng.uniform(0.005, 0.03, size=(NB, H, bs)).astype(np.float32) for _ in range(2))
    return Kp, Vp, ksp, vsp


def select_inputs(seed, B, H, G, D, bs, MB, lens):
    rng = np.random.default_rng(seed)
    NB = B * MB + 3
    table = rng.permutation(NB)[: B * MB].reshape(B, MB).astype(np.int32)
    c = rng.integers(-60, 61, (NB, H, 1, D))
    w = rng.integers(0, 61, (NB, H, 1, D))
    bounds = np.concatenate([c + w, c - w], axis=2).astype(np.int8)
    step = rng.uniform(0.01, 0.03, (NB, H)).astype(np.float32)
    q = rng.standard_normal((B, H * G, D)).astype(np.float32)
    return q, bounds, step, table, np.asarray(lens, np.int32)


# ------------------------------------------------------------------ CPU tests
def test_plan_oracle_by_hand():
    """Three requests, blocks of 4: one ends, one grows into a new block, one is refused."""
    lens = np.array([5, 4, 6], np.int32)
    new = np.array([-1, 2, 9], np.int32)
    table = np.array([[3, 1, -1, -1], [0, -1, -1, -1], [2, 4, -1, -1]], np.int32)
    free = np.array([5, -1, -1, -1, -1, -1], np.int32)
    t, f, c, ln, st, sl, status = plan_oracle(lens, new, table, free, 1, 4, 11)
    # the stack is 5, 3, 1 (top): request 1 takes 1; request 2 needs 2 more: 3 and 5 are there
    assert t[1, 1] == 1 and list(t[2, 2:4]) == [3, 5] and c == 0 and status == 0
    assert list(ln) == [0, 6, 15] and list(st) == [0, 0, 2, 11]
    assert list(sl) == [4, 5, 18, 19, 12, 13, 14, 15, 20, 21, 22]
    t, f, c, ln, st, sl, status = plan_oracle(lens, new, table, free, 0, 4, 11)
    assert status == kvd.KVD_STATUS_NO_BLOCKS and list(ln) == [0, 6, 6] and c == 1 and f[0] == 3
    assert (sl[2:] == -1).all()


def test_bounds_hold_every_key():
    """The bound codes times the step enclose each dequantised key, up to the fp32 rounding of the step."""
    rng = np.random.default_rng(2)
    codes = rng.integers(-127, 128, (16, 64), dtype=np.int8)
    scales = rng.uniform(1e-3, 2, 16).astype(np.float32)
    bd, step = bounds_oracle(codes, scales)
    x = codes.astype(np.float64) * scales.astype(np.float64)[:, None]
    tol = 127 * float(step) * 2.0 ** -22  # a quotient and the step are each rounded once
    assert (bd[0] * float(step) >= x.max(0) - tol).all() and (bd[1] * float(step) <= x.min(0) + tol).all()


def test_symbols_and_refusals():
    L = kvd.lib()
    d = kvd.PagedPlanDesc(4, 16, 8, 4, 10, 4)
    ok = [256] * 10
    assert L.kvd_paged_plan_workspace_size(ctypes.byref(d)) == 16
    assert L.kvd_paged_plan_launch(None, *ok, 16, None) == EINVAL
    for i in range(10):
        bad = list(ok)
        bad[i] = None
        assert L.kvd_paged_plan_launch(ctypes.byref(d), *bad, 16, None) == EINVAL, i
    assert L.kvd_paged_plan_launch(ctypes.byref(d), *ok, 15, None) == EINVAL  # workspace too small
    for bad in [(0, 16, 8, 4, 10, 4), (8193, 16, 8, 4, 10, 4), (4, 0, 8, 4, 10, 4), (4, 16, 0, 4, 10, 4),
                (4, 16, 8, 0, 10, 4), (4, 16, 8, 4, -1, 4), (4, 16, 8, 4, 10, 3), (4, 1 << 16, 8, 1 << 16, 10, 1 << 16)]:
        d = kvd.PagedPlanDesc(*bad)
        assert L.kvd_paged_plan_workspace_size(ctypes.byref(d)) == 0
        assert L.kvd_paged_plan_launch(ctypes.byref(d), *ok, 16, None) == EINVAL

    rows = (4, 2, 64, 16, 8, 0, 128, 64, 2048, 1024, 64, 32, 16)
    d = kvd.PagedRowsDesc(*rows)
    for i in range(7):
        bad = [256] * 9
        bad[i] = None
        assert L.kvd_paged_write_launch(ctypes.byref(d), *bad, None) == EINVAL, i
        bad = [256] * 7
        bad[i] = None
        assert L.kvd_paged_read_launch(ctypes.byref(d), *bad, None) == EINVAL, i
    assert L.kvd_paged_write_launch(ctypes.byref(d), *[256] * 7, 256, None, None) == EINVAL  # bounds without scales
    assert L.kvd_paged_write_launch(ctypes.byref(d), *[256] * 7, None, 256, None) == EINVAL
    for at, value in [(0, -1), (1, 0), (2, 0), (2, 513), (3, 0), (4, 0), (5, 1), (5, 2 | 4), (5, 32)]:
        bad = list(rows)
        bad[at] = value
        d = kvd.PagedRowsDesc(*bad)
        assert L.kvd_paged_write_launch(ctypes.byref(d), *[256] * 9, None) == EINVAL, (at, value)
        assert L.kvd_paged_read_launch(ctypes.byref(d), *[256] * 7, None) == EINVAL, (at, value)
    d = kvd.PagedRowsDesc(0, *rows[1:])
    assert L.kvd_paged_write_launch(ctypes.byref(d), *[None] * 9, None) == 0  # nothing to do

    sel = (2, 8, 2, 64, 16, 40, 20, 8, 1, 2, 0, 256, 256, 20, 512, 64)
    d = kvd.BlockSelectDesc(*sel)
    assert L.kvd_block_select_workspace_size(ctypes.byref(d)) == 2 * 2 * 20 * 4
    for i in range(6):
        bad = [256] * 6
        bad[i] = None
        assert L.kvd_block_select_launch(ctypes.byref(d), *bad, 320, None) == EINVAL, i
    assert L.kvd_block_select_launch(ctypes.byref(d), *[256] * 6, 319, None) == EINVAL  # workspace too small
    for at, value in [(0, 0), (1, 0), (1, 7), (2, 0), (3, 0), (3, 513), (4, 0), (5, 0), (6, 0), (6, 1 << 28), (7, 0),
                      (7, 2), (8, -1), (8, 7), (9, 0), (10, 1), (10, 6), (11, None), (12, None), (13, 19)]:
        bad = list(sel)
        bad[at] = value
        d = kvd.BlockSelectDesc(*bad)
        assert L.kvd_block_select_workspace_size(ctypes.byref(d)) == 0 or at in (11, 12)
        assert L.kvd_block_select_launch(ctypes.byref(d), *[256] * 6, 1 << 30, None) == EINVAL, (at, value)

    sp = dict(batch=2, num_q_heads=8, num_kv_heads=2, head_dim=128, block_size=16, num_blocks=64, max_blocks_per_seq=8,
              seq_lens=256, block_table=256, block_table_stride=8, o_stride_h=128)
    assert L.kvd_sparse_decode_launch(None, *[256] * 7, 0, None) == EINVAL
    d = kvd.PagedDesc(**sp)
    for i in range(6):
        bad = [256] * 7
        bad[i] = None
        assert L.kvd_sparse_decode_launch(ctypes.byref(d), *bad, 0, None) == EINVAL, i
    for key, value in [("batch", 0), ("num_q_heads", 7), ("block_table_stride", 7), ("flags", 64), ("flags", 1 | 8),
                       ("flags", 1), ("seq_lens", None)]:
        d = kvd.PagedDesc(**{**sp, key: value})
        assert L.kvd_sparse_decode_launch(ctypes.byref(d), *[256] * 7, 0, None) == EINVAL, (key, value)
    d = kvd.PagedDesc(**{**sp, "flags": kvd.KVD_FLAG_QK_INT8})
    assert L.kvd_sparse_decode_launch(ctypes.byref(d), *[256] * 7, 0, None) == 801  # cudaErrorNotSupported


def test_long_budgets_are_refused():
    """A selection's tokens are counted in 32 bits: budgets above 2^30 tokens do not reach a kernel."""
    L = kvd.lib()
    sp = dict(batch=1, num_q_heads=1, num_kv_heads=1, head_dim=80, block_size=1 << 14, num_blocks=64,
              seq_lens=256, block_table=256, block_table_stride=1 << 17, o_stride_h=80)
    d = kvd.PagedDesc(**sp, max_blocks_per_seq=1 << 16)
    assert L.kvd_sparse_workspace_size(ctypes.byref(d)) > 0  # 2^30 tokens
    for blocks in ((1 << 16) + 1, (1 << 17) - 1):
        d = kvd.PagedDesc(**sp, max_blocks_per_seq=blocks)
        assert L.kvd_sparse_workspace_size(ctypes.byref(d)) == 0
        assert L.kvd_sparse_decode_launch(ctypes.byref(d), *[256] * 7, 1 << 40, None) == EINVAL


def test_python_refusals():
    import torch

    i32 = torch.int32
    z = torch.zeros
    lens, table, free = z(2, dtype=i32), z((2, 4), dtype=i32), z(8, dtype=i32)
    with pytest.raises(ValueError):
        kvd.paged_plan(lens, z(3, dtype=i32), table, free, z(1, dtype=i32), 4, z(4, dtype=torch.int64))
    with pytest.raises(ValueError):
        kvd.paged_plan(lens, lens, table, free, z(1, dtype=i32), 4, z(4, dtype=i32))
    k, pool, sc = z((3, 2, 64)), z((5, 2, 8, 64), dtype=torch.int8), z((5, 2, 8))
    slots = z(3, dtype=torch.int64)
    with pytest.raises(ValueError):
        kvd.paged_write(k[:2], k[:2], slots, pool, pool, sc, sc)
    with pytest.raises(ValueError):
        kvd.paged_write(k.double(), k.double(), slots, pool, pool, sc, sc)
    with pytest.raises(ValueError):
        kvd.paged_write(k, k, slots, pool, pool, sc, sc, bounds=z((5, 2, 2, 64), dtype=torch.int8))
    with pytest.raises(ValueError):
        kvd.paged_read(slots, pool, pool, sc[:, :, :4], sc[:, :, :4])
    bounds, step = z((5, 2, 2, 64), dtype=torch.int8), z((5, 2))
    with pytest.raises(ValueError):
        kvd.block_select(z((2, 3, 64)), bounds, step, table, lens, 8, 4)
    with pytest.raises(ValueError):
        kvd.block_select(z((2, 4, 64)), bounds, step, table.long(), lens, 8, 4)
    with pytest.raises(ValueError):
        kvd.sparse_decode(z((2, 4, 64)), pool, pool, sc, sc, z((2, 2, 3), dtype=i32), z((2,), dtype=i32))
    with pytest.raises(ValueError):
        kvd.sparse_decode(z((2, 4, 64)), pool, pool, sc, sc, z((2, 2, 3), dtype=i32), z((2, 2), dtype=i32),
                          out=z((2, 4, 32)))


# ------------------------------------------------------------------ GPU tests
def _dev(*arrays):
    import torch

    return [torch.from_numpy(np.ascontiguousarray(a)).to(DEV) for a in arrays]


def _run_plan(lens, new, table, free, count, bs, num_slots, in_place=True, ws=None):
    import torch

    tl, tn, tt, tf = _dev(lens, new, table, free)
    tc = torch.tensor([count], dtype=torch.int32, device=DEV)
    slots = torch.full((num_slots,), 77, dtype=torch.int64, device=DEV)
    kw = {} if in_place else dict(seq_lens_out=torch.empty_like(tl), free_count_out=torch.empty_like(tc))
    _, starts = kvd.paged_plan(tl, tn, tt, tf, tc, bs, slots, workspace=ws, **kw)
    status = kvd.device_status()
    lo, co = kw.get("seq_lens_out", tl), kw.get("free_count_out", tc)
    if not in_place:
        assert np.array_equal(tl.cpu().numpy(), lens) and int(tc) == count
    return tt.cpu().numpy(), tf.cpu().numpy(), int(co), lo.cpu().numpy(), starts.cpu().numpy(), slots.cpu().numpy(), status


def _same_plan(got, want):
    for a, b, what in zip(got, want, ("table", "free", "count", "lens", "starts", "slots", "status")):
        assert np.array_equal(a, b), what


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("B,bs,MB,spare,ends,prompts,plen,extra", [
    (1, 16, 4, 3, 0, 0, 1, 0), (1, 1, 1, 0, 1, 0, 1, 2), (7, 3, 9, 2, 2, 2, 11, 0), (33, 16, 20, 40, 5, 6, 130, 3),
    (256, 64, 16, 100, 0, 0, 1, 0), (257, 8, 40, 300, 30, 40, 90, 0), (1500, 16, 30, 900, 100, 60, 300, 17),
    (64, 16, 600, 4000, 0, 8, 7000, 0), (5, 16, 8, 0, 5, 0, 1, 0)])
def test_plan_matches_the_oracle(B, bs, MB, spare, ends, prompts, plen, extra, in_place):
    args = plan_inputs(B * 7 + bs, B, bs, MB, spare, ends, prompts, plen)
    num_slots = int(np.maximum(args[1], 0).sum()) + extra
    _same_plan(_run_plan(*args, bs, num_slots, in_place), plan_oracle(*args, bs, num_slots))


@pytest.mark.gpu
def test_plan_refusals_and_odd_inputs():
    """Too few blocks, rows and slots; lengths below zero and past the table; sums past 32 bits; bad ids."""
    import torch

    lens, new, table, free, count = plan_inputs(5, 40, 16, 12, 30, 3, 10, 200)
    for num_slots in (0, 5, 200, 3000):
        _same_plan(_run_plan(lens, new, table, free, count, 16, num_slots), plan_oracle(lens, new, table, free, count, 16, num_slots))
    for c in (-3, 0, 2, 10 ** 6):
        _same_plan(_run_plan(lens, new, table, free, c, 16, 900), plan_oracle(lens, new, table, free, c, 16, 900))
    odd = lens.copy()
    odd[3], odd[4], odd[5] = -5, 10 ** 6, 12 * 16
    _same_plan(_run_plan(odd, new, table, free, count, 16, 3000), plan_oracle(odd, new, table, free, count, 16, 3000))
    big = new.copy()
    big[7:12] = 2 ** 31 - 1
    _same_plan(_run_plan(lens, big, table, free, count, 16, 3000), plan_oracle(lens, big, table, free, count, 16, 3000))
    broken, listed = table.copy(), free.copy()
    broken[:, 0] = 10 ** 6
    listed[20:30] = -4
    _same_plan(_run_plan(lens, new, broken, listed, count, 16, 3000), plan_oracle(lens, new, broken, listed, count, 16, 3000))
    # the workspace is left as it was: one buffer serves calls of different sizes
    ws = torch.zeros(16, dtype=torch.uint8, device=DEV)
    for num_slots in (3000, 20000, 1):
        _same_plan(_run_plan(lens, new, table, free, count, 16, num_slots, ws=ws),
                   plan_oracle(lens, new, table, free, count, 16, num_slots))
    assert int(ws.sum()) == 0


def _quantise(x):
    c, s = po.quantize_rows(np.ascontiguousarray(x, np.float32))
    return c, s


def _write_case(seed, T, H, D, bs, layout, starts, dtype):
    """Tokens of len(starts) requests laid over random blocks, each from its own offset."""
    import torch

    rng = np.random.default_rng(seed)
    parts = np.diff(np.sort(np.concatenate([[0, T], rng.integers(0, T + 1, len(starts) - 1)])))
    NB = T // bs + 2 * len(starts) + 2
    ids, at, slots = rng.permutation(NB), 0, []
    for n, o in zip(parts, starts):
        pos = o + np.arange(n)
        m = -(-(o + int(n)) // bs) if n else 0
        blk = ids[at: at + m]
        at += m
        slots.append(blk[pos // bs] * bs + pos % bs)
    slots = np.concatenate(slots).astype(np.int64)
    Kp, Vp, ksp, vsp = pools(seed + 1, NB, H, bs, D, layout)
    k, v = (torch.from_numpy((rng.standard_normal((T, H, D)) * np.exp(rng.standard_normal((T, H, 1)))).astype(np.float32)).to(dtype)
            for _ in range(2))
    return slots, NB, Kp, Vp, ksp, vsp, k, v


def _write_oracle(slots, NB, Kp, Vp, ksp, vsp, k, v, bs, layout):
    Kp, Vp, ksp, vsp = Kp.copy(), Vp.copy(), ksp.copy(), vsp.copy()
    H, D = k.shape[1:]
    bounds, step = np.full((NB, H, 2, D), 55, np.int8), np.full((NB, H), 0.5, np.float32)
    last = {}
    (kc, kss), (vc, vss) = _quantise(k), _quantise(v)
    for t, s in enumerate(slots):
        if s < 0 or s >= NB * bs:
            continue
        blk, o = divmod(int(s), bs)
        last[blk] = o
        at = (blk, slice(None), o) if layout == "bhtd" else (blk, o)
        Kp[at], Vp[at] = kc[t], vc[t]
        ksp[blk, :, o], vsp[blk, :, o] = kss[t], vss[t]
    for blk, o in last.items():
        for h in range(H):
            rows = Kp[blk, h, : o + 1] if layout == "bhtd" else Kp[blk, : o + 1, h]
            bounds[blk, h], step[blk, h] = bounds_oracle(rows, ksp[blk, h, : o + 1])
    return Kp, Vp, ksp, vsp, bounds, step


def _bits(a):
    return a.view(np.uint32) if a.dtype == np.float32 else a


def _same_bits(got, want, what):
    a, b = got.cpu().numpy(), want
    if b.dtype == np.float32:
        assert np.array_equal(np.isnan(a), np.isnan(b)), what
        a, b = np.where(np.isnan(a), 0, a).astype(np.float32), np.where(np.isnan(b), 0, b).astype(np.float32)
    assert np.array_equal(_bits(a), _bits(b)), what


def _check_write(case, bs, layout):
    import torch

    slots, NB, Kp, Vp, ksp, vsp, k, v = case
    want = _write_oracle(slots, NB, Kp, Vp, ksp, vsp, k.float().numpy(), v.float().numpy(), bs, layout)
    tK, tV, tks, tvs, ts = _dev(Kp, Vp, ksp, vsp, slots)
    H, D = k.shape[1:]
    bounds = torch.full((NB, H, 2, D), 55, dtype=torch.int8, device=DEV)
    step = torch.full((NB, H), 0.5, device=DEV)
    tk, tv = k.to(DEV), v.to(DEV)
    kvd.paged_write(tk, tv, ts, tK, tV, tks, tvs, bounds=bounds, bound_scale=step, layout=layout)
    for got, w, what in zip((tK, tV, tks, tvs, bounds, step), want, ("K", "V", "ks", "vs", "bounds", "step")):
        _same_bits(got, w, what)
    # without bounds: the same rows
    tK2, tV2, tks2, tvs2 = _dev(Kp, Vp, ksp, vsp)
    kvd.paged_write(tk, tv, ts, tK2, tV2, tks2, tvs2, layout=layout)
    assert torch.equal(tK2, tK) and torch.equal(tV2, tV) and torch.equal(tks2, tks) and torch.equal(tvs2, tvs)
    # read back
    ko, vo = kvd.paged_read(ts, tK, tV, tks, tvs, k_out=torch.empty_like(tk), v_out=torch.empty_like(tv), layout=layout)
    ok = (slots >= 0) & (slots < NB * bs)
    for got, pool, sc in ((ko, want[0], want[2]), (vo, want[1], want[3])):
        s = np.where(ok, slots, 0)
        rows = pool[s // bs, :, s % bs] if layout == "bhtd" else pool[s // bs, s % bs]
        with np.errstate(invalid="ignore"):  # code 0 at an infinite scale stands for NaN
            value = rows.astype(np.float32) * sc[s // bs, :, s % bs][..., None]
        ref = torch.from_numpy(np.where(ok[:, None, None], value, np.float32(0))).to(k.dtype)
        assert torch.allclose(got.cpu(), ref, rtol=0, atol=0, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["bhtd", "bthd"])
@pytest.mark.parametrize("T,H,D,bs,starts,dtype", [
    (1, 1, 128, 16, [0], "float32"), (1, 8, 128, 16, [15], "bfloat16"), (5, 2, 64, 4, [3, 0], "float16"),
    (40, 3, 128, 16, [7, 0, 15], "float32"), (300, 2, 256, 64, [63, 1], "bfloat16"), (700, 4, 128, 128, [5, 0, 127], "float16"),
    (64, 2, 80, 8, [1, 2, 3], "float32"), (33, 1, 7, 16, [0], "bfloat16"), (50, 2, 512, 32, [31], "float32"),
    (600, 1, 128, 512, [300, 0], "float32"), (2000, 8, 128, 16, [3] * 9, "bfloat16"), (257, 2, 128, 1, [0, 0], "float32")])
def test_write_and_read_match_the_oracle(T, H, D, bs, starts, dtype, layout):
    import torch

    _check_write(_write_case(T + D, T, H, D, bs, layout, starts, getattr(torch, dtype)), bs, layout)
    assert kvd.device_status() == 0


@pytest.mark.gpu
def test_write_skips_and_odd_rows():
    """Slots of -1 and outside the pool; zero rows, subnormals, infinities and NaN; ties of the rounding."""
    import torch

    slots, NB, Kp, Vp, ksp, vsp, k, v = _write_case(3, 90, 2, 128, 16, "bhtd", [4, 0, 9], torch.float32)
    slots[10:13] = -1
    slots[60] = NB * 16 + 5
    slots[61] = -2
    k[0] = 0
    k[1] = 1e-40
    k[2, 0, 5] = float("inf")
    k[3, 1, 7] = float("nan")
    k[4] = float("nan")
    k[5, 0] = torch.arange(128) - 63.5  # amax 64.5: quotients at and near halves
    k[6, 1] = torch.arange(128) * 1.0
    k[7, 0] = torch.where(torch.arange(128) % 2 == 0, 127.0, 0.5) * 2.0 ** -130
    k[8, 0] = 3e38
    v[0] = -0.0
    _check_write((slots, NB, Kp, Vp, ksp, vsp, k, v), 16, "bhtd")
    assert kvd.device_status() == kvd.KVD_STATUS_BAD_BLOCK
    assert kvd.device_status() == 0


def _quotient_rows(dtype, rng):
    """Rows of 128 whose first value is the largest: every significand of the maximum (a sample of float32's), with
    values of every exponent at which a code can be other than 0, and around the halves between codes."""
    bits = {"bfloat16": 7, "float16": 10, "float32": 23}[dtype]
    sigs = 1 << bits
    top = np.arange(sigs) if sigs <= 1024 else rng.integers(0, sigs, 2000)
    rows = []
    for e in range(10):
        for base in ((-50, 0, 50) if dtype != "float16" else (4,)):
            val = np.sort(rng.choice(sigs, size=127, replace=False)) if sigs <= 1024 else rng.integers(0, sigs, (len(top), 127))
            val = np.broadcast_to(val, (len(top), 127))
            x = np.ldexp(1.0 + val / sigs, base - e)
            lead = np.ldexp(1.0 + top / sigs, base)[:, None]
            rows.append(np.concatenate([lead, np.minimum(x, lead)], 1))
    if dtype == "float32":  # within three units in the last place of a half
        lead = rows[0][:, :1].astype(np.float32)
        half = (lead / np.float32(127.0)).astype(np.float64) * (np.arange(127) + 0.5)
        near = half.astype(np.float32).view(np.int32) + rng.integers(-3, 4, half.shape, dtype=np.int32)
        rows.append(np.concatenate([lead, np.minimum(near.view(np.float32), lead)], 1))
    x = np.concatenate(rows).astype(np.float32)
    return x * np.where(rng.random(x.shape) < 0.5, -1, 1).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_write_quotients_are_the_divisions(dtype):
    """Codes and scales equal the IEEE division's bit for bit, also where a quotient lies on or beside a half."""
    import torch

    x = _quotient_rows(dtype, np.random.default_rng(11))
    x = x[: x.shape[0] // 16 * 16]
    k = torch.from_numpy(x).to(getattr(torch, dtype))
    assert torch.equal(k.float(), torch.from_numpy(x))  # all representable
    k = k[:, None]
    v = k.flip(0).contiguous()
    NB = x.shape[0] // 16
    slots = torch.arange(x.shape[0], dtype=torch.int64)
    tk, tv, ts = k.to(DEV), v.to(DEV), slots.to(DEV)
    K, V = (torch.full((NB, 1, 16, 128), 77, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((NB, 1, 16), -1.0, device=DEV) for _ in range(2))
    kvd.paged_write(tk, tv, ts, K, V, ks, vs)
    codes, scales = po.quantize_rows(x)
    _same_bits(K.reshape(-1, 128), codes, "K")
    _same_bits(ks.reshape(-1), scales, "ks")
    _same_bits(V.reshape(-1, 128), codes[::-1].copy(), "V")
    _same_bits(vs.reshape(-1), scales[::-1].copy(), "vs")


@pytest.mark.gpu
def test_write_strided_rows_and_streams():
    """Rows that are a part of a wider tensor (vector and scalar access), on a stream that is not the default."""
    import torch

    for cut, D in ((slice(0, 128), 128), (slice(1, 129), 128)):
        slots, NB, Kp, Vp, ksp, vsp, k, v = _write_case(9, 70, 2, D, 16, "bthd", [2, 0], torch.bfloat16)
        wide = torch.zeros((70, 2, 2, 160), dtype=torch.bfloat16, device=DEV)
        wide[:, 0, :, cut], wide[:, 1, :, cut] = k.to(DEV), v.to(DEV)
        want = _write_oracle(slots, NB, Kp, Vp, ksp, vsp, k.float().numpy(), v.float().numpy(), 16, "bthd")
        tK, tV, tks, tvs, ts = _dev(Kp, Vp, ksp, vsp, slots)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        kvd.paged_write(wide[:, 0, :, cut], wide[:, 1, :, cut], ts, tK, tV, tks, tvs, layout="bthd", stream=side)
        torch.cuda.current_stream().wait_stream(side)
        for got, w, what in zip((tK, tV, tks, tvs), want, ("K", "V", "ks", "vs")):
            _same_bits(got, w, what)


def _check_select(q, bounds, step, table, lens, bs, k, first, last, dtype="float32"):
    import torch

    tq = torch.from_numpy(q).to(getattr(torch, dtype))
    with np.errstate(all="ignore"):
        want = select_oracle(tq.float().numpy(), bounds, step, table, lens, bs, k, first, last)
    tb, ts, tt, tl = _dev(bounds, step, table, lens)
    sel, sl = kvd.block_select(tq.to(DEV), tb, ts, tt, tl, bs, k, first, last)
    assert np.array_equal(sl.cpu().numpy(), want[1])
    assert np.array_equal(sel.cpu().numpy(), want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,G,D,bs,MB,k,first,last,dtype", [
    (1, 1, 1, 128, 16, 40, 5, 1, 2, "float32"), (3, 2, 8, 128, 16, 100, 16, 1, 2, "bfloat16"),
    (2, 8, 4, 64, 32, 300, 40, 0, 1, "float16"), (2, 2, 16, 128, 64, 77, 30, 3, 5, "float32"),
    (1, 2, 5, 96, 8, 513, 64, 1, 1, "float32"), (2, 1, 3, 192, 8, 260, 9, 4, 5, "float32"),
    (2, 2, 2, 256, 16, 64, 20, 1, 2, "bfloat16"), (2, 2, 2, 80, 16, 64, 20, 1, 2, "float32"),
    (1, 1, 20, 128, 4, 2000, 256, 1, 2, "float32"), (1, 1, 1, 7, 1, 50, 3, 0, 1, "float32"),
    (400, 1, 1, 128, 16, 33, 8, 1, 2, "float32"), (1, 2, 8, 128, 16, 5000, 300, 1, 2, "bfloat16"),
    (1, 1, 2, 512, 16, 40, 8, 1, 2, "float32"), (1, 1, 1, 128, 1, 40000, 17, 2, 2, "float32")])
def test_select_matches_the_oracle(B, H, G, D, bs, MB, k, first, last, dtype):
    rng = np.random.default_rng(MB)
    lens = rng.integers(0, MB * bs + 1, B)
    lens[0] = MB * bs
    if B > 2:
        lens[1], lens[2] = 0, 1
    _check_select(*select_inputs(MB + k, B, H, G, D, bs, MB, lens), bs, k, first, last, dtype)
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("MB", [60, 3000])
def test_select_ties_and_odd_values(MB):
    """Equal scores go to the lower index; NaN and infinite scores; zero queries; block ids outside the pool;
    lengths below zero, past the table, at and next to block edges and the budget."""
    B, H, G, D, bs, k = 4, 2, 4, 128, 16, 12
    q, bounds, step, table, lens = select_inputs(1, B, H, G, D, bs, MB, [MB * bs, 999999, (k + 1) * bs, MB * bs - 15])
    same = np.broadcast_to(bounds[:1], bounds.shape).copy()
    _check_select(q, same, np.full_like(step, 0.02), table, lens, bs, k, 1, 2)  # all blocks tie
    few = same.copy()
    few[::7] = bounds[1]
    _check_select(q, few, np.full_like(step, 0.02), table, lens, bs, k, 1, 2)
    odd = step.copy()
    odd[::5] = np.nan
    odd[1::17] = np.inf
    odd[2::3] = 0
    _check_select(q, bounds, odd, table, lens, bs, k, 1, 2)
    qq = q.copy()
    qq[0] = 0
    qq[1, 0, 3] = np.inf
    qq[2, :, 5] = np.nan
    qq[3] = 1e-42
    _check_select(qq, bounds, odd, table, lens, bs, k, 1, 2)
    _check_select(qq, bounds, step, table, np.array([-4, k * bs, k * bs + 1, k * bs - 1], np.int32), bs, k, 1, 2)
    assert kvd.device_status() == 0
    bad = table.copy()
    bad[:, ::3] = -1
    bad[:, 1::9] = 10 ** 8
    _check_select(q, bounds, step, bad, lens, bs, k, 1, 2)
    assert kvd.device_status() == kvd.KVD_STATUS_BAD_BLOCK


@pytest.mark.gpu
@pytest.mark.parametrize("MB", [3000, 6000])
def test_select_crowds_at_the_threshold(MB):
    """A crowd of 100 to 600 blocks with scores next to one another, and the budget ends in it."""
    crowds = [100, 255, 256, 257, 300, 400, 511, 512, 513, 600]
    rng = np.random.default_rng(MB)
    B, bs = len(crowds), 16
    q, bounds, step, table, lens = select_inputs(2, B, 1, 2, 128, bs, MB, [MB * bs] * B)
    same = np.broadcast_to(bounds[:1], bounds.shape).copy()
    for b, m in enumerate(crowds):
        mine = rng.uniform(0.0, 50.0, MB)
        where = rng.permutation(np.arange(1, MB - 2))
        mine[where[:m]] = rng.uniform(100.0, 100.2, m)
        mine[where[m]] = 200.0
        step[table[b], 0] = mine
    for k in (3 + 1 + 7, 3 + 1 + 60, 3 + 1 + 99):
        _check_select(q, same, step, table, lens, bs, k, 1, 2)
    assert kvd.device_status() == 0


def _check_sparse(seed, B, H, G, D, bs, k, lens, layout, qtype="float32", otype="float32", spare=5, partial=False, ws=None):
    import torch

    rng = np.random.default_rng(seed)
    NB = B * H * k + spare
    Kp, Vp, ksp, vsp = pools(seed, NB, H, bs, D, layout)
    sel = rng.permutation(NB)[: B * H * k].reshape(B, H, k).astype(np.int32)
    lens = np.asarray(lens, np.int32).reshape(B, H)
    for b in range(B):  # what lies past a row's tokens is garbage in a live pool
        for h in range(H):
            n = min(max(0, int(lens[b, h])), k * bs)
            for j in range(n // bs, k):
                o = max(0, n - j * bs)
                ksp[sel[b, h, j], h, o:] = np.nan
                vsp[sel[b, h, j], h, o:] = np.inf
            sel[b, h, -(-n // bs):] = -1
    q = torch.from_numpy(rng.standard_normal((B, H * G, D)).astype(np.float32)).to(getattr(torch, qtype))
    ref = sparse_oracle(q.float().numpy(), Kp, Vp, ksp, vsp, sel, lens, layout)
    tK, tV, tks, tvs, tsel, tl = _dev(Kp, Vp, ksp, vsp, sel, lens)
    out = torch.full((B, H * G, D + 4 if partial else D), float("nan"), dtype=getattr(torch, otype), device=DEV)
    kvd.sparse_decode(q.to(DEV), tK, tV, tks, tvs, tsel, tl, out=out, layout=layout, partial=partial, workspace=ws)
    got = out.float().cpu().numpy().astype(np.float64)
    if partial:
        rec = got
        with np.errstate(all="ignore"):
            got = np.where(rec[..., 1:2] > 0, rec[..., 4:] / rec[..., 1:2], 0.0)
    half = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[otype]  # 8 and 11 significant bits
    tol = 2e-5 + (1e-4 + half) * np.abs(ref)
    assert np.isfinite(got).all()
    assert (np.abs(got - ref) <= tol).all(), np.abs(got - ref).max()
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["bhtd", "bthd"])
@pytest.mark.parametrize("B,H,G,D,bs,k,qt,ot", [
    (1, 1, 1, 128, 16, 3, "float32", "float32"), (2, 8, 8, 128, 16, 20, "bfloat16", "bfloat16"),
    (3, 2, 4, 128, 8, 33, "float32", "float32"), (1, 2, 16, 128, 64, 40, "float16", "float16"),
    (2, 3, 2, 128, 128, 5, "float32", "float32"), (1, 4, 1, 128, 256, 9, "bfloat16", "float32"),
    (5, 4, 1, 128, 32, 6, "float32", "float16"), (2, 2, 3, 128, 16, 12, "float32", "float32"),
    (2, 2, 8, 64, 16, 12, "bfloat16", "bfloat16"), (1, 2, 2, 80, 24, 7, "float32", "float32"),
    (1, 1, 5, 256, 1, 70, "float32", "float32"), (1, 8, 8, 128, 64, 200, "float32", "float32")])
def test_sparse_decode_matches_the_oracle(B, H, G, D, bs, k, qt, ot, layout):
    rng = np.random.default_rng(k)
    lens = rng.integers(1, k * bs + 1, B * H)
    lens[0] = k * bs
    _check_sparse(k + D, B, H, G, D, bs, k, lens, layout, qt, ot)


@pytest.mark.gpu
@pytest.mark.parametrize("D,G,bs,k", [(128, 8, 16, 12), (128, 1, 128, 3), (64, 2, 16, 12), (128, 4, 8, 300)])
def test_sparse_decode_lengths(D, G, bs, k):
    """Rows without tokens give zeros; one token; lengths at and next to block and tile edges, below zero and past
    the budget; a single block."""
    lens = [0, 1, bs - 1, bs, bs + 1, 127, 128, 129, k * bs, k * bs - 1, -3, 10 ** 6]
    _check_sparse(4, 6, 2, G, D, bs, k, lens, "bhtd")
    _check_sparse(5, 6, 2, G, D, bs, k, [0] * 12, "bhtd")
    _check_sparse(6, 1, 2, G, D, bs, 1, [1, bs], "bthd")
    _check_sparse(7, 6, 2, G, D, bs, k, lens, "bthd", partial=True)


@pytest.mark.gpu
@pytest.mark.parametrize("G", [3, 5, 6, 7, 9, 12, 16, 20, 33])
@pytest.mark.parametrize("D,bs,k", [(128, 16, 20), (64, 16, 20)])
def test_sparse_decode_groups(D, bs, k, G):
    """Groups of query heads that are no power of two or above the kernels' forms, whole and split rows, records."""
    _check_sparse(G, 2, 3, G, D, bs, k, [k * bs, 1, 77, 130, 200, k * bs - 3], "bthd", "bfloat16", "float32")
    _check_sparse(G + 1, 1, 2, G, D, 64, 40, [2560, 2500], "bhtd", "float32", "float32", partial=True)


@pytest.mark.gpu
@pytest.mark.parametrize("G", [1, 2, 3, 4])
@pytest.mark.parametrize("B,k", [(2, 60), (2, 90), (4, 130)])
def test_sparse_decode_either_side_of_little_work(B, k, G):
    """Budgets at which small groups change from one kernel to the other."""
    rng = np.random.default_rng(k)
    lens = rng.integers(0, k * 16 + 1, (B, 8))
    lens[0, :4] = 0, 1, k * 16, k * 16 - 15
    _check_sparse(k + G, B, 8, G, 128, 16, k, lens, "bhtd")


@pytest.mark.gpu
def test_sparse_decode_small_workspace_and_bad_ids():
    """Less scratch means fewer splits, not other results; a block id outside the pool is not read."""
    import torch

    for n in (1, 5000, 40000):
        _check_sparse(8, 1, 2, 8, 128, 64, 60, [3840, 3000], "bhtd", ws=torch.empty(n, dtype=torch.uint8, device=DEV))
    Kp, Vp, ksp, vsp = pools(1, 9, 2, 16, 128, "bhtd")
    sel = np.array([[[0, 1, 10 ** 8], [-5, 3, 4]]], np.int32)
    tK, tV, tks, tvs, tsel, tl = _dev(Kp, Vp, ksp, vsp, sel, np.full((1, 2), 48, np.int32))
    out = kvd.sparse_decode(torch.zeros((1, 4, 128), device=DEV), tK, tV, tks, tvs, tsel, tl)
    assert torch.isfinite(out).all()
    assert kvd.device_status() == kvd.KVD_STATUS_BAD_BLOCK


@pytest.mark.gpu
def test_full_selection_is_the_paged_decode():
    """A budget that covers the cache gives the paged decode's output (same tiles; sums may be split elsewhere)."""
    import torch

    B, H, G, D, bs, MB = 3, 2, 4, 128, 16, 20
    rng = np.random.default_rng(3)
    Kp, Vp, ksp, vsp = pools(2, B * MB, H, bs, D, "bhtd")
    table = rng.permutation(B * MB).reshape(B, MB).astype(np.int32)
    lens = np.array([320, 33, 0], np.int32)
    q = torch.randn((B, H * G, D), device=DEV)
    tK, tV, tks, tvs, tt, tl = _dev(Kp, Vp, ksp, vsp, table, lens)
    bounds, step = torch.zeros((B * MB, H, 2, D), dtype=torch.int8, device=DEV), torch.ones((B * MB, H), device=DEV)
    sel, sl = kvd.block_select(q, bounds, step, tt, tl, bs, MB)
    got = kvd.sparse_decode(q, tK, tV, tks, tvs, sel, sl).cpu().numpy()
    ref = kvd.paged_decode(q, tK, tV, tks, tvs, tt, tl).cpu().numpy()
    bad, max_abs, _ = po.check(got, ref.astype(np.float64), 2e-5, 1e-4)
    assert bad == 0, max_abs


@pytest.mark.gpu
def test_step_in_a_cuda_graph():
    """Plan, write, select and decode of one token for every request, captured once and replayed: each replay
    goes on from the state that the one before left, and the last one's output meets the oracle."""
    import torch

    B, H, G, D, bs, MB, k = 3, 2, 4, 128, 16, 12, 4
    NB = B * MB
    i32 = torch.int32
    lens = torch.tensor([0, 15, 100], dtype=i32, device=DEV)
    table = torch.full((B, MB), -1, dtype=i32, device=DEV)
    free = torch.arange(NB, dtype=i32, device=DEV)
    count = torch.tensor([NB], dtype=i32, device=DEV)
    Kp, Vp = (torch.zeros((NB, H, bs, D), dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros((NB, H, bs), device=DEV) for _ in range(2))
    bounds, step = torch.zeros((NB, H, 2, D), dtype=torch.int8, device=DEV), torch.zeros((NB, H), device=DEV)
    # the prompts, through the same calls
    prompt = lens.clone()
    lens.zero_()
    total = int(prompt.sum())
    slots = torch.empty(total, dtype=torch.int64, device=DEV)
    kvd.paged_plan(lens, prompt, table, free, count, bs, slots)
    kvd.paged_write(*(torch.randn((total, H, D), device=DEV) for _ in range(2)), slots, Kp, Vp, ks, vs, bounds, step)
    one = torch.ones(B, dtype=i32, device=DEV)
    slot = torch.empty(B, dtype=torch.int64, device=DEV)
    starts = torch.empty(B + 1, dtype=i32, device=DEV)
    ws = torch.zeros(16, dtype=torch.uint8, device=DEV)
    kn, vn, q = (torch.randn((B, n, D), device=DEV) for n in (H, H, H * G))
    out = torch.empty_like(q)
    sel, sl = torch.empty((B, H, k), dtype=i32, device=DEV), torch.empty((B, H), dtype=i32, device=DEV)
    scratch = torch.empty(kvd.sparse_workspace_size(q, Kp, sel) + 16, dtype=torch.uint8, device=DEV)

    def one_step():
        kvd.paged_plan(lens, one, table, free, count, bs, slot, starts, workspace=ws)
        kvd.paged_write(kn, vn, slot, Kp, Vp, ks, vs, bounds, step)
        kvd.block_select(q, bounds, step, table, lens, bs, k, sel_table=sel, sel_lens=sl)
        kvd.sparse_decode(q, Kp, Vp, ks, vs, sel, sl, out=out, workspace=scratch)

    one_step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one_step()
    for i in range(40):
        for t in (kn, vn, q):
            t.normal_()
        graph.replay()
    torch.cuda.synchronize()
    assert list(lens.cpu()) == [41, 56, 141] and int(count) == NB - 3 - 4 - 9
    held = [int(x) for b, n in enumerate((3, 4, 9)) for x in table[b, :n]]
    assert len(set(held)) == 16
    cpu = lambda t: t.cpu().numpy()  # noqa: E731
    want = select_oracle(cpu(q), cpu(bounds), cpu(step), cpu(table), cpu(lens), bs, k, 1, 2)
    assert np.array_equal(cpu(sel), want[0]) and np.array_equal(cpu(sl), want[1])
    for blk, n in ((int(table[2, 8]), 141 - 128), (int(table[0, 0]), 16)):
        bd, st = bounds_oracle(cpu(Kp)[blk, 1, :n], cpu(ks)[blk, 1, :n])
        assert np.array_equal(cpu(bounds)[blk, 1], bd) and cpu(step)[blk, 1] == st
    ref = sparse_oracle(cpu(q), cpu(Kp), cpu(Vp), cpu(ks), cpu(vs), *want, "bhtd")
    bad, max_abs, _ = po.check(cpu(out), ref, 2e-5, 1e-4)
    assert bad == 0, max_abs
    assert kvd.device_status() == 0
