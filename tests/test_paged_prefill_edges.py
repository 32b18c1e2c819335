"""Attention of packed new tokens over a paged INT8 cache: inputs at which single steps of the kernels can go wrong.

Inputs, oracle and tolerances are those of test_paged_prefill.py; where a test needs another bound it derives it."""
import ctypes
import re
from pathlib import Path

import numpy as np
import pytest

import kvdecode as kvd
from test_paged_prefill import DEV, TYPES, check, close, make_case, oracle, prefill, prefill_desc

CSRC = Path(__file__).resolve().parents[1] / "cuda-operators_b200" / "csrc"


def tokens(s, b=0):
    """(blocks, offsets) of request b's tokens, in their order."""
    import torch

    t = torch.arange(int(s["len"][b]), device=DEV)
    return s["table"][b].long()[t // s["bs"]], t % s["bs"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,every", [("float32", 128, 1024), ("float16", 256, 8192), ("bfloat16", 256, 8192)])
@pytest.mark.parametrize("what", ["scores", "values"])
@pytest.mark.parametrize("times", [1, 2])
def test_references_that_move_where_sums_are_put_aside(dtype, n, every, what, times):
    # Sums in parts: a warpgroup puts its sums aside after some of its tiles, and starts again from zero. Here the
    # scores rise by 10 in base 2, or value scales by 2^10, at just those tiles (every so many tokens), so that sums are
    # put aside and scaled in the same step. What was put aside is 0.25 to 20 percent of what comes after it, and all
    # values are above zero: a sum that counts twice, or not at all, is off by more than the tolerance.
    import torch

    H = torch.cuda.get_device_properties(0).multi_processor_count  # a unit of work a CTA: rows are not split
    ln = times * every + 400
    s = make_case(1, [n], [ln], H, 1, 64, 64, dtype, seed=31)
    s["V"] = s["V"].abs()
    s["K"][..., 0] = 0
    blk, off = tokens(s)
    level = torch.arange(ln, device=DEV) // every
    if what == "scores":
        s["q"] *= 0.02
        s["q"][:, :, 0] = 8.0
        s["ks"].fill_(10 * np.log(2) / 60)  # 8 x 60 level ks / sqrt(64) = 10 ln 2 level
        s["K"][blk, :, off, 0] = (60 * level).to(torch.int8).unsqueeze(-1)
    else:
        s["vs"][blk, :, off] *= (2.0 ** (10 * level.float())).unsqueeze(-1)
    close(prefill(s, causal=False), s, oracle(s, causal=False))
    assert kvd.device_status() == 0


def test_kernels_wait_for_the_one_before_them():
    # Every kernel that is launched with the programmatic attribute waits for its predecessor, whatever its arguments
    # say, before it lets the next one begin and before it looks at memory that others write; or, where a class of
    # requests follows another, it acquires the stamp that the plan released, and waits where it does not find it.
    begins = (CSRC / "kvd_chunk.cuh").read_text().split("void class_begins")[1].split("\n}\n")[0]
    at = [begins.find(x) for x in ("ld.acquire.gpu.global.u64", "stamp == p.stamp", "__syncthreads();",
                                   "if (!s_ready) grid_dependency_wait();", "} else {\n        grid_dependency_wait();", "\n    allow_dependents();")]
    assert at[0] >= 0 and at == sorted(at)
    assert "st.release.gpu.global.u64" in (CSRC / "kvd_chunk.cu").read_text()
    found = 0
    for name in ("kvd_chunk.cu", "kvd_chunk_few.cu", "kvd_chunk_tile.cu", "kvd_pages.cu"):
        source = (CSRC / name).read_text()
        for part in source.split("__global__")[1:]:
            body = part[part.index("{\n"): part.index("\n}\n")]
            wait, allow = body.find("\n    grid_dependency_wait();"), body.find("\n    allow_dependents();")
            if wait < 0:
                wait, allow = body.find("\n    class_begins(p);"), len(body)
                assert body.endswith("\n    class_ends(p);")
            assert 0 <= wait < allow, (name, part[:100])
            assert not re.search(r"\bp\.(head|first|rec|starts|seq_lens|table|lens|parents|Q|K|V|ks|vs|bits_a|free_in)\b", body[:wait])
            found += 1
    assert found >= 9


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_plans_of_calls_that_follow_each_other(dtype):
    # Requests of every class in each call, two calls in turn with other lengths and rows, in one graph with one
    # workspace, and replays with other lengths: a kernel that read the plan of a call before would take other units.
    # What says that a plan is there is gone when the call has ended.
    import torch

    n = [[1, 8, 30, 1, 120, 2, 50, 1] * 4, [50, 1, 1, 9, 2, 140, 1, 20] * 4]
    cases = [make_case(32, x, np.asarray(x) + 300 * (1 + i), 8, 4, 128, 16, dtype, seed=40 + i) for i, x in enumerate(n)]
    wants = [oracle(s) for s in cases]
    outs = [torch.empty_like(s["q"]) for s in cases]
    ws = torch.full((max(kvd.paged_prefill_workspace_size(s["q"], s["K"], s["table"]) for s in cases),), 255,
                    dtype=torch.uint8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for _ in range(3):
            for s, o in zip(cases, outs):
                o.fill_(float("nan"))
                prefill(s, out=o, workspace=ws)
    for _ in range(4):
        graph.replay()
        for s, o, w in zip(cases, outs, wants):
            close(o, s, w)
        assert int(ws[:8].view(torch.int64)) == 0
        for s in cases:
            s["lens"].sub_(17)
            s["len"] = s["len"] - 17
        wants = [oracle(s) for s in cases]
    for s, w in zip(cases, wants):  # calls outside of graphs
        close(prefill(s, workspace=ws), s, w)
        assert int(ws[:8].view(torch.int64)) == 0
    assert kvd.device_status() == 0


FEW = [(128, 4, 2), (128, 4, 10), (64, 1, 7), (64, 2, 21)]  # dims, heads a KV head, rows: 8 to 42 rows a KV head


def hidden_scales(D, G, n, dtype, value, ln):
    """Whose last tokens' value scales are far above what the rows in front of them see. "steps": each new token's is
    four times the one before it, so every row has a largest of its own."""
    s = make_case(1, [n], [ln], 2, G, D, 16, dtype, seed=51)
    blk, off = tokens(s)
    if value == "steps":
        s["vs"] *= 1e-6
        for i in range(n):
            s["vs"][blk[ln - n + i], :, off[ln - n + i]] *= 4.0 ** min(i + 1, 8 if dtype == "float16" else 40)
    else:
        s["vs"][blk[-1], :, off[-1]] = value
    return s


def check_hidden_scales(D, G, n, dtype, value, ln=None):
    # Causal rows: what a row gets does not depend on value scales of tokens behind it. A small weight is off by 2^-25 of
    # a reference that is at least 2^6 of the largest value scale that the row sees, times a code of at most 127: 2^-31
    # of 127 times that scale a token, in every dim, also where the code of the token with that scale is 0. So the
    # largest |v| of the tolerance is 127 times the largest scale in sight.
    import torch

    s = hidden_scales(D, G, n, dtype, value, ln or max(203, n + 33))
    out, mean, _, size = oracle(s)
    blk, off = tokens(s)
    sees = 127.0 * s["vs"][blk, :, off].double().cummax(0).values[-n:].repeat_interleave(G, 1)
    want = out, mean, sees.unsqueeze(-1).expand_as(out), size
    got = prefill(s)
    s["n"], s["starts_host"] = np.array([n - 1]), np.array([0, n - 1])  # every row but the last: the large ones are hidden
    close(got, s, want)
    if dtype != "float16" or value == "steps":  # the last row's fit the output
        close(got, {**s, "n": np.array([n]), "starts_host": np.array([0, n])}, want)
    s["n"], s["starts_host"] = np.array([n]), np.array([0, n])
    close(prefill(s, out_dtype=torch.float32), s, want)
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G,n", FEW)
@pytest.mark.parametrize("value", ["steps", 1e10, 1e20, 1e36])
def test_value_scales_of_hidden_tokens_with_few_rows(D, G, n, dtype, value):
    check_hidden_scales(D, G, n, dtype, value)


MANY = [(128, 4, 40), (128, 1, 300), (64, 1, 130), (64, 8, 70)]  # 130 to 560 rows a KV head


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G,n", MANY)
@pytest.mark.parametrize("value", ["steps", 1e10, 1e20, 1e36])
def test_value_scales_of_hidden_tokens_with_many_rows(D, G, n, dtype, value):
    check_hidden_scales(D, G, n, dtype, value)


def sizes(rows, **kw):
    L = kvd.lib()
    return [int(L.kvd_paged_prefill_workspace_size(ctypes.byref(prefill_desc(num_rows=t, **kw)))) for t in rows]


SHAPES = [(8, 8, 8, 257, 128), (128, 1, 8, 257, 128), (1, 2, 1, 600, 64), (300, 8, 4, 600, 128), (64, 16, 1, 94, 64),
          (4, 2, 64, 300, 128), (2, 1, 100, 300, 64), (40, 1, 7, 3, 128)]


def check_sizes(B, H, G, MB, D, flags):
    # scratch for a loop's largest step serves every smaller one
    rows = [*range(0, 700), *range(700, 70000, 331)]
    got = sizes(rows, batch=B, num_q_heads=H * G, num_kv_heads=H, max_blocks_per_seq=MB, block_table_stride=MB, head_dim=D,
                flags=flags)
    assert got[0] > 0 and all(x <= y for x, y in zip(got, got[1:]))


@pytest.mark.parametrize("B,H,G,MB,D", SHAPES)
@pytest.mark.parametrize("flags", [0, kvd.KVD_FLAG_Q_BF16 | kvd.KVD_FLAG_OUT_BF16])
def test_workspace_does_not_shrink_with_more_rows(B, H, G, MB, D, flags):
    check_sizes(B, H, G, MB, D, flags)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,G,MB,D", SHAPES)
def test_workspace_does_not_shrink_with_more_rows_on_the_gpu(B, H, G, MB, D):
    check_sizes(B, H, G, MB, D, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_one_workspace_serves_chunks_and_then_single_tokens(dtype):
    import torch

    chunk = make_case(8, [16, 1, 1, 1, 1, 1, 1, 1], [4000, 900, 17, 300, 1, 2222, 64, 4100], 8, 8, 128, 16, dtype, seed=63)
    one = make_case(8, [1] * 8, [4001, 901, 18, 301, 2, 2223, 65, 4100], 8, 8, 128, 16, dtype, seed=64)
    chunk["table"] = torch.nn.functional.pad(chunk["table"], (0, one["table"].shape[1] - chunk["table"].shape[1]))
    size = kvd.paged_prefill_workspace_size(chunk["q"], chunk["K"], chunk["table"])
    ws = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
    for s in (chunk, one, chunk):
        close(prefill(s, workspace=ws), s, oracle(s))
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G,n,ln", [(128, 4, 2, 9001), (128, 4, 40, 9001), (64, 1, 300, 20011), (128, 1, 1000, 3000)])
@pytest.mark.parametrize("value", ["steps", 1e20])
def test_value_scales_of_hidden_tokens_of_long_rows(D, G, n, ln, dtype, value):
    # tokens in stretches, some of which no row sees as a whole
    check_hidden_scales(D, G, n, dtype, value, ln)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 32])
def test_many_small_weights_beside_a_large_one(dtype, n):
    # 2^20 tokens of weight 2^-25.5 beside one of weight 1, all values the same: the small weights are 2.2 percent of
    # their sum, and the output is the value. As one fp16 term a weight is off by half a step (2^-11 of it) or, below the
    # smallest normal fp16, by 2^-25 of a reference that is at least 2^6 of the large weight: 2^20 tokens x 2^-31, 2^-11.
    # (The same for the scale of bf16's values and its product with the code, and half a step of the output.) Nearly all entries of the table name
    # one block, so that the pool is small; a unit of work a CTA: rows of 32 tokens are not split.
    import torch

    H, bs, D, G = torch.cuda.get_device_properties(0).multi_processor_count, 128, 64, 8
    MB = (1 << 20) // bs
    K, V = (torch.zeros((2, H, bs, D), dtype=torch.int8, device=DEV) for _ in range(2))
    V.fill_(64)
    K[0, :, 0, 0] = 100
    ks = torch.full((2, H, bs), 25.5 * np.log(2) / 100, device=DEV)  # 8 x 100 ks / sqrt(64) = 25.5 ln 2
    vs = torch.full((2, H, bs), 0.01, device=DEV)
    table = torch.ones((1, MB), dtype=torch.int32, device=DEV)
    table[0, 0] = 0
    q = torch.zeros((n, H * G, D), dtype=getattr(torch, dtype), device=DEV)
    q[..., 0] = 8.0
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = kvd.paged_prefill(q, K, V, ks, vs, table, i32([1 << 20]), i32([0, n]), causal=False, out_dtype=q.dtype).double()
    want = 64 * float(vs[0, 0, 0])
    eps = torch.finfo(q.dtype).eps / 2
    tol = 1e-4 + 2.0 ** -11 + (0.0 if dtype == "float32" else eps + 3 * 2.0 ** -11)
    assert float((got / want - 1).abs().max()) <= tol
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G,n", [(128, 4, 1), (128, 4, 10), (64, 1, 7), (128, 4, 40), (64, 1, 300), (96, 2, 6)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_value_scales_that_are_not_finite(D, G, n, dtype, value):
    # a row that sees such a token is NaN in every dim, also where its code is 0 or the weight vanishes; others are as ever
    import torch

    for small in (False, True):
        s = make_case(2, [n, 3], [703, 90], 2, G, D, 16, dtype, seed=61)
        want = oracle(s)
        blk, off = tokens(s)
        at = 703 - n // 2 - 1  # the rows from n - 1 - n // 2 on see it
        s["vs"][blk[at], 1, off[at]] = value
        s["V"][blk[at], 1, off[at], :9] = 0
        if small:
            s["ks"][blk[at], 1, off[at]] = 0.0  # score 0, where other tokens of its rows have hundreds
            s["q"] *= 40.0
            want = None
        got = prefill(s)
        assert torch.isnan(got[n - 1 - n // 2: n, G:]).all()
        rest = got.clone()
        rest[n - 1 - n // 2: n, G:] = 0.0
        assert torch.isfinite(rest).all()
        if want is not None:
            out = want[0].clone()
            out[n - 1 - n // 2: n, G:] = 0.0
            close(rest, s, (out, *want[1:]))
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [2, 20, 200])
def test_rows_and_scales_near_the_smallest_number(dtype, n):
    # query rows of 1e-34 with a softmax scale of 1e-9: all scores vanish, and the weights of what a row sees are equal
    s = make_case(1, [n], [n + 150], 2, 2, 128, 16, dtype, seed=62)
    s["q"] *= 1e-34
    check(s, scale=1e-9)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,layout", [(257, "bhtd"), (384, "bthd"), (511, "bhtd"), (512, "bhtd")])
def test_wide_heads(dtype, D, layout):
    # more dims than the CUDA-core kernel has threads, three and four times
    check(make_case(3, [1, 9, 5], [70, 9, 130], 2, 2, D, 16, dtype, layout, seed=71, extra=2), causal=True)
    check(make_case(2, [3, 1], [2, 200], 1, 3, D, 7, dtype, layout, seed=72), causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G,n", [(128, 4, 2), (128, 4, 11), (64, 1, 300), (128, 8, 70), (96, 1, 5)])
def test_codes_of_minus_128(dtype, D, G, n):
    # the lowest code, which the quantiser does not make and the layout allows
    s = make_case(2, [n, 1], [n + 290, 40], 2, G, D, 16, dtype, seed=73)
    for x in ("K", "V"):
        s[x][:, :, ::3] = -128
        s[x][..., 5] = -128
    check(s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_more_requests_than_the_plan_keeps(dtype):
    # over 1,024 requests the plan looks lengths up again instead of keeping them; some have no rows, some no tokens
    rng = np.random.default_rng(74)
    n = rng.integers(0, 4, size=2500)
    n[::500] = 90
    lens = np.maximum(0, n + rng.integers(-2, 60, size=2500))
    lens[7] = 9000
    check(make_case(2500, n, lens, 1, 2, 64, 16, dtype, seed=74))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_what_a_request_gets_beside_others(dtype):
    # The plan splits tokens by the work of the whole call, so a row's bits depend on the other requests; its value does not.
    s = make_case(6, [40, 1, 300, 2, 9, 64], [4000, 9000, 1300, 64, 700, 64], 2, 4, 128, 16, dtype, seed=75)
    want = oracle(s)
    for b in range(6):
        one = {**s, "n": s["n"][b:b + 1], "len": s["len"][b:b + 1], "starts_host": s["starts_host"][b:b + 2],
               "table": s["table"][b:b + 1], "lens": s["lens"][b:b + 1], "starts": s["starts"][b:b + 2].contiguous()}
        close(prefill(one), one, want)
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G,n", [(128, 4, 2), (128, 4, 80), (64, 1, 11), (64, 2, 200)])
def test_value_scales_over_eight_powers_of_ten(dtype, D, G, n):
    s = make_case(2, [n, n], [1500, 333], 1, G, D, 16, dtype, seed=76, v_spread=1e4)
    check(s)
    s["ks"].zero_()  # equal weights
    check(s)
