"""Paged serving steps at sizes where every CTA goes round its pipeline many times and takes several pieces of work
(no reference counterpart). Rules and tolerances are those of test_blocks.py, whose oracles are used where they are
quick enough; the selection's is restated with matrix products in 64-bit floats, which hold its whole numbers exactly."""
import numpy as np
import pytest

import kvdecode as kvd
import pyoracle as po
from test_blocks import (DEV, _check_write, _dev, _run_plan, _same_plan, _write_case, plan_inputs, plan_oracle, pools,
                         select_inputs, select_oracle, sparse_oracle)


def long_select_oracle(q, bounds, step, table, lens, bs, k, first, last):
    """select_oracle for long rows: sums by 64-bit float products (exact below 2^53), one sort a row."""
    B, Hq, _ = q.shape
    NB, H = step.shape
    G, MB = Hq // H, table.shape[1]
    sel, sel_lens = np.full((B, H, k), -1, np.int32), np.zeros((B, H), np.int32)
    qc, qs = po.quantize_rows(q)
    for b in range(B):
        ln = int(np.clip(lens[b], 0, MB * bs))
        n = -(-ln // bs)
        ids = table[b, :n]
        good = (ids >= 0) & (ids < NB)
        at = np.where(good, ids, 0)
        for h in range(H):
            idx, sel_lens[b, h] = np.arange(n), ln
            if n > k:
                c = qc[b, h * G:(h + 1) * G].astype(np.float64)
                bd = bounds[at, h].astype(np.float64)
                dots = np.maximum(c, 0) @ bd[:, 0].T + np.minimum(c, 0) @ bd[:, 1].T
                with np.errstate(all="ignore"):
                    v = dots.astype(np.float32) * qs[b, h * G:(h + 1) * G].astype(np.float32)[:, None]
                    s = np.where(np.isnan(v), np.float32(np.inf), v).max(0) * step[at, h]
                s = np.where(np.isnan(s), np.inf, s).astype(np.float64)
                rank = good.astype(np.int64)
                rank[:first] = 2
                rank[n - last:] = 2
                idx = np.sort(np.lexsort((np.arange(n), np.where(rank == 1, -s, 0.0), -rank))[:k])
                sel_lens[b, h] = (k - n) * bs + ln
            sel[b, h, : len(idx)] = ids[idx]
    return sel, sel_lens


@pytest.mark.parametrize("seed", range(3))
def test_long_select_oracle_is_the_oracle(seed):
    B, H, G, D, bs, MB, k = 4, 2, 3, 64, 16, 40, 9
    lens = [MB * bs, (k + 1) * bs - 5, k * bs, 0]
    q, bounds, step, table, lens = select_inputs(seed, B, H, G, D, bs, MB, lens)
    step[::7], step[1::9] = np.nan, 0.02
    bounds[1::9] = bounds[1]
    table[0, 3:9] = -1, 10 ** 8, -2, 5, -1, 10 ** 8
    for k, first, last in ((9, 1, 2), (37, 0, 1), (9, 4, 5)):
        args = (q, bounds, step, table, lens, bs, k, first, last)
        for a, b in zip(long_select_oracle(*args), select_oracle(*args)):
            assert np.array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("G", [8, 20])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_select_rounds_of_the_score_pipeline(D, G):
    """About 20 tiles of 128 blocks a CTA: the ring of stages and that of the steps go round, CTAs pass from row to row
    (a new query each time), and rows without blocks, within the budget or one above it lie between."""
    H, bs, MB, k, NB = 8, 16, 9000, 50, 12000
    lens = np.array([MB * bs, 0, MB * bs - 7, k * bs, 5, 5000 * bs + 1, (k + 1) * bs, 129 * bs, MB * bs, 7000 * bs - 15, 0,
                     6001 * bs, 128 * bs, 3], np.int32)
    B = len(lens)
    rng = np.random.default_rng(D + G)
    c = rng.integers(-60, 61, (NB, H, 1, D), dtype=np.int8)
    w = rng.integers(0, 61, (NB, H, 1, D), dtype=np.int8)
    bounds = np.concatenate([c + w, c - w], axis=2)
    step = rng.uniform(0.01, 0.03, (NB, H)).astype(np.float32)
    table = np.stack([rng.permutation(NB)[:MB] for _ in range(B)]).astype(np.int32)
    q = rng.standard_normal((B, H * G, D)).astype(np.float32)
    want = long_select_oracle(q, bounds, step, table, lens, bs, k, 1, 2)
    tq, tb, ts, tt, tl = _dev(q, bounds, step, table, lens)
    for _ in range(3):
        sel, sl = kvd.block_select(tq, tb, ts, tt, tl, bs, k)
        assert np.array_equal(sl.cpu().numpy(), want[1])
        assert np.array_equal(sel.cpu().numpy(), want[0])
    assert kvd.device_status() == 0


def _check_sparse_rows(seed, B, H, G, D, bs, k, layout, ws=None):
    """Many rows: head h of request b attends to blocks of a permutation of the head's own; lengths of all kinds, rows
    without tokens among them; scales past a row's tokens are NaN and infinite."""
    import torch

    rng = np.random.default_rng(seed)
    NB = B * k + 3
    Kp, Vp, ksp, vsp = pools(seed, NB, H, bs, D, layout)
    lens = rng.integers(0, k * bs + 1, (B, H)).astype(np.int32)
    lens[rng.random((B, H)) < 0.3] = k * bs
    lens[::3, 1::2] = 0
    lens[1, 0], lens[2, 0] = 1, k * bs - 1
    sel = np.stack([rng.permutation(NB)[: B * k].reshape(B, k) for _ in range(H)], axis=1).astype(np.int32)
    for b in range(B):
        for h in range(H):
            n = int(lens[b, h])
            if n < k * bs:
                ksp[sel[b, h, n // bs], h, n % bs:] = np.nan
                vsp[sel[b, h, n // bs], h, n % bs:] = np.inf
            sel[b, h, -(-n // bs):] = -1
    q = rng.standard_normal((B, H * G, D)).astype(np.float32)
    ref = sparse_oracle(q, Kp, Vp, ksp, vsp, sel, lens, layout)
    tq, tK, tV, tks, tvs, tsel, tl = _dev(q, Kp, Vp, ksp, vsp, sel, lens)
    out = torch.full((B, H * G, D), float("nan"), device=DEV)
    kvd.sparse_decode(tq, tK, tV, tks, tvs, tsel, tl, out=out, layout=layout, workspace=ws)
    bad, max_abs, _ = po.check(out.cpu().numpy(), ref, 2e-5, 1e-4)
    assert bad == 0, max_abs
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("G,layout", [(8, "bhtd"), (3, "bthd"), (12, "bhtd"), (1, "bthd"), (2, "bhtd"), (20, "bthd")])
def test_sparse_decode_several_rows_a_cta(G, layout):
    """640 and more work rows of up to five tiles over 296 CTAs of the tensor-core kernel, whole and padded groups."""
    _check_sparse_rows(G, 80, 8, G, 128, 16, 40, layout)


@pytest.mark.gpu
@pytest.mark.parametrize("G", [1, 2, 5, 8, 12])
@pytest.mark.parametrize("D,bs,B", [(64, 16, 80), (256, 16, 70), (128, 24, 80), (64, 7, 150)])
def test_sparse_decode_many_chunks_a_split(D, bs, B, G):
    """The CUDA-core kernel with enough rows that a split is many chunks of 64 tokens, and without scratch, where one
    CTA takes a whole row of them."""
    import torch

    _check_sparse_rows(G, B, 8, G, D, bs, 640 // bs, "bhtd")
    _check_sparse_rows(G + 1, 3, 2, G, D, bs, 1500 // bs, "bthd", ws=torch.empty(1, dtype=torch.uint8, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("D,G,bs", [(80, 2, 24), (96, 5, 16)])
def test_sparse_decode_long_rows_of_other_head_dims(D, G, bs):
    import torch

    _check_sparse_rows(G, 20, 4, G, D, bs, 1500 // bs, "bthd")
    _check_sparse_rows(G, 3, 2, G, D, bs, 1500 // bs, "bhtd", ws=torch.empty(1, dtype=torch.uint8, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,D,bs,requests,dtype,layout", [
    (20011, 2, 128, 64, 1500, "bfloat16", "bhtd"), (20011, 2, 64, 128, 1200, "float32", "bthd"),
    (20000, 2, 256, 64, 40, "float32", "bhtd"), (24000, 2, 128, 128, 9, "bfloat16", "bthd"),
    (20000, 2, 256, 128, 900, "float16", "bhtd"), (21000, 2, 128, 64, 700, "float32", "bthd"),
    (8100, 2, 80, 64, 700, "float32", "bhtd"), (12000, 2, 96, 128, 30, "bfloat16", "bthd"),
    (40000, 2, 128, 16, 3000, "bfloat16", "bthd"), (40000, 2, 64, 32, 20, "float16", "bhtd")])
def test_write_several_runs_a_cta(T, H, D, bs, requests, dtype, layout):
    """Tiles of more than one token: CTAs write several runs, runs go on from one tile into the next, and refused
    stretches, single skipped tokens and a slot outside the pool lie within and between them."""
    import torch

    rng = np.random.default_rng(T + D)
    starts = rng.integers(0, bs, requests).tolist()
    slots, NB, *rest = _write_case(T + D, T, H, D, bs, layout, starts, getattr(torch, dtype))
    slots[T // 7: T // 7 + 2500] = -1
    slots[T // 2: T // 2 + 130] = -1
    slots[T // 3: T // 3 + 1500: 97] = -1
    slots[T - 700] = NB * bs + 1
    _check_write((slots, NB, *rest), bs, layout)
    assert kvd.device_status() == kvd.KVD_STATUS_BAD_BLOCK


@pytest.mark.gpu
@pytest.mark.parametrize("B,num_slots", [(4097, 30000), (8192, 200000)])
def test_plan_of_the_largest_batches(B, num_slots):
    args = plan_inputs(B, B, 16, 9, B, B // 9, B // 5, 40)
    _same_plan(_run_plan(*args, 16, num_slots), plan_oracle(*args, 16, num_slots))


def _high_and_low(NB, n, seed):
    """n block ids, the first and the last ones of the pool among them, in random order."""
    rng = np.random.default_rng(seed)
    ids = np.concatenate([np.arange(n // 2), NB - 1 - np.arange(n - n // 2)])
    return rng.permutation(ids)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["bhtd", "bthd"])
@pytest.mark.parametrize("NB,H,bs,D", [(70000, 8, 64, 128), (140000, 8, 64, 64), (2200000, 8, 1, 128), (90000, 8, 80, 80)])
def test_pools_past_32_bits(NB, H, bs, D, layout):
    """Pools, or bounds, of more than 2^32 bytes: rows written, read, scored and attended to in their first and last
    blocks are, bit for bit, those of a small pool that holds the same blocks."""
    import torch

    n, B, G, k = 40, 2, 4, 9
    g = torch.Generator(device=DEV).manual_seed(1)
    ids = torch.from_numpy(_high_and_low(NB, n, NB)).to(DEV)
    shape = lambda blocks: (blocks, H, bs, D) if layout == "bhtd" else (blocks, bs, H, D)  # noqa: E731

    def made(blocks):
        K, V = (torch.zeros(shape(blocks), dtype=torch.int8, device=DEV) for _ in range(2))
        ks, vs = (torch.zeros((blocks, H, bs), device=DEV) for _ in range(2))
        return [K, V, ks, vs], [torch.zeros((blocks, H, 2, D), dtype=torch.int8, device=DEV),
                                torch.zeros((blocks, H), device=DEV)]

    big, small = made(NB), made(n)
    assert max(t.nbytes for t in (*big[0], *big[1])) > 1 << 32
    T = n * bs - bs // 3
    k_new, v_new = (torch.randn((T, H, D), device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((B, H * G, D), device=DEV, generator=g)
    lens = torch.tensor([n // 2 * bs, T - n // 2 * bs], dtype=torch.int32, device=DEV)
    got = []
    for (pool, bound), blocks in ((big, ids), (small, torch.arange(n, device=DEV))):
        slots = (blocks[:, None] * bs + torch.arange(bs, device=DEV)).reshape(-1)[:T].contiguous()
        kvd.paged_write(k_new, v_new, slots, *pool, *bound, layout=layout)
        rows = kvd.paged_read(slots, *pool, layout=layout)
        table = blocks.view(B, n // B).to(torch.int32)
        sel, sl = kvd.block_select(q, *bound, table, lens, bs, k)
        out = kvd.sparse_decode(q, *pool, sel, sl, layout=layout)
        got.append([*rows, out, sl] + [t[blocks] for t in (*pool, *bound)] + [sel])
    for a, b in zip(got[0][:-1], got[1][:-1]):
        assert torch.equal(a, b)
    assert torch.equal(got[0][-1], ids[got[1][-1].long()].to(torch.int32))
    assert got[0][0].abs().max() > 1 and kvd.device_status() == 0


@pytest.mark.gpu
def test_slots_past_32_bits():
    """More than 2^31 slots: blocks of a slot are found by 64-bit division; rows of 4 values in the last blocks."""
    import torch

    bs, D, n = 64, 4, 30
    NB = (1 << 25) + 100
    K, V = (torch.zeros((NB, 1, bs, D), dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros((NB, 1, bs), device=DEV) for _ in range(2))
    ids = torch.from_numpy(_high_and_low(NB, n, 3)).to(DEV)
    slots = (ids[:, None] * bs + torch.arange(bs, device=DEV)).reshape(-1)[: n * bs - 5].contiguous()
    assert int(slots.max()) >= 1 << 31
    slots[100:120] = -1
    slots[500] = NB * bs
    x, y = (torch.randn((len(slots), 1, D), device=DEV) for _ in range(2))
    kvd.paged_write(x, y, slots, K, V, ks, vs)
    ok = ((slots >= 0) & (slots < NB * bs)).cpu().numpy()
    at = slots[torch.from_numpy(ok).to(DEV)]
    for rows, pool, scales in ((x, K, ks), (y, V, vs)):
        codes, sc = po.quantize_rows(rows.cpu().numpy()[ok])
        assert np.array_equal(pool[at // bs, 0, at % bs].cpu().numpy(), codes[:, 0])
        assert np.array_equal(scales[at // bs, 0, at % bs].cpu().numpy(), sc[:, 0])
    got, _ = kvd.paged_read(slots, K, V, ks, vs)
    codes, sc = po.quantize_rows(x.cpu().numpy())
    assert np.array_equal(got.cpu().numpy(), np.where(ok[:, None, None], codes.astype(np.float32) * sc[..., None], np.float32(0)))
    assert kvd.device_status() == kvd.KVD_STATUS_BAD_BLOCK
