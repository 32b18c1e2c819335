"""Attention of packed new tokens over a paged INT8 cache (no reference
counterpart: the reference's prefill attention, attention/, is fp32 with no KV
cache).

The oracle computes the formula of include/kvdecode.h in 64 bits. Tolerances,
per element, against it:

* 2e-5 + 1e-4 |ref|, the framework's own for fp32 sums over the INT8 cache;
* a 16-bit output adds half a step of its type: eps / 2 relative (and half the
  smallest step of fp16, 2^-25);
* where the output has 16 bits the weights enter the sum of values as fp16, each
  off by half a step: fp16 keeps 10 bits behind the leading one, so steps are at
  most 2^-10 of a value and half a step 2^-11. Over a row that is at most
  2^-11 sum_j p_j |v_j| / sum_j p_j. A weight below the smallest normal fp16 is off by 2^-25 of a
  reference that is at least 2^-8 of the row's largest: 2^-17 of the largest
  |v| a token, at most, counted as 2^-17 max |v| in all;
* where the output is bf16 a value's scale and its product with the code enter as
  fp16 too: two more half steps, 3 2^-11 sum_j p_j |v_j| with the weights' (whose
  products with each other, below 2^-20, the first term covers);
* 32-bit outputs have two fp16 terms of a weight, whose steps end at 2^-24: half of
  that, 2^-25, of a reference that is at least 2^6 of the largest value scale, is
  2^-31 of the largest |v| a token, however small the weight: 2^-31 len max |v|.
  (It shows where a token that outweighs all others has a code of 0 and values are
  far above 1, so that 2e-5 is nothing);
* the scores: with A = max_j sum_d |q_d k_jd| ks_j scale, rounding the queries to
  two fp16 terms (22 bits) moves a score by at most 2^-22 A, and each of the 16
  fp32 sums of 16 dims (8, times 2 terms) by half a step of at most 2^-24 A:
  together 1.25 2^-20 A. A change of d in the scores moves the output by at most
  d sum_j p_j |v_j - out| <= 2 d sum_j p_j |v_j| to first order, so
  2.5 2^-20 A sum_j p_j |v_j|: far below the first term where scores are of
  ordinary size (A is about 7 in most tests here).
"""
import ctypes

import numpy as np
import pytest

import kvdecode as kvd

DEV = "cuda:0"
EINVAL = kvd.CUDA_ERROR_INVALID_VALUE
TYPES = ("float32", "bfloat16", "float16")


# ---------------------------------------------------------------------- inputs
def make_case(B, n, lens, H, G, D, bs, dtype, layout="bhtd", seed=0, extra=0, front=0, k_spread=1.0, v_spread=1.0):
    """Rows, pools and tables on the GPU: n[b] rows and lens[b] tokens of request b."""
    import torch

    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    n, lens = np.asarray(n), np.asarray(lens)
    held = -(-lens // bs)
    MB = max(1, int(held.max())) + 1
    NB = int(held.sum()) + 3
    ids = rng.permutation(NB)
    table = rng.integers(-1000, 2 * NB + 1000, size=(B, MB)).astype(np.int32)  # behind a request's blocks: anything
    at = 0
    for b in range(B):
        table[b, : held[b]] = ids[at: at + held[b]]
        at += held[b]
    shape = (NB, H, bs, D) if layout == "bhtd" else (NB, bs, H, D)
    s = {"n": n, "len": lens, "bs": bs, "layout": layout, "G": G, "table_host": table}
    s["K"], s["V"] = (torch.randint(-127, 128, shape, dtype=torch.int8, device=DEV, generator=gen) for _ in range(2))
    spread = lambda x: torch.exp(np.log(x) * (2 * torch.rand((NB, H, bs), device=DEV, generator=gen) - 1))  # noqa: E731
    s["ks"], s["vs"] = 0.012 * spread(k_spread), 0.01 * spread(v_spread)
    starts = front + np.concatenate([[0], np.cumsum(n)])
    T = int(starts[-1]) + extra
    s["q"] = torch.randn((T, H * G, D), device=DEV, generator=gen).to(getattr(torch, dtype))
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).to(DEV)  # noqa: E731
    s |= {"table": i32(table), "lens": i32(lens), "starts": i32(starts), "starts_host": starts}
    return s


def oracle(s, causal=True, scale=None):
    """(out, mean of |v| under the weights, largest |v|, A) in 64 bits for every row."""
    import torch

    q = s["q"].double()
    T, Hq, D = q.shape
    G, H = s["G"], Hq // s["G"]
    scale = scale or 1 / np.sqrt(D)
    out, mean, top, size = (torch.zeros((T, Hq, D), dtype=torch.float64, device=DEV) for _ in range(4))
    NB = s["ks"].shape[0]
    for b in range(len(s["n"])):
        n, ln, t0 = int(s["n"][b]), int(s["len"][b]), int(s["starts_host"][b])
        if n == 0 or ln == 0:
            continue
        ids = torch.from_numpy(s["table_host"][b, : -(-ln // s["bs"])]).to(DEV).long()
        good = (ids >= 0) & (ids < NB)
        ids = torch.where(good, ids, 0)
        for h in range(H):
            def rows(pool, sc):
                p = pool[ids, h] if s["layout"] == "bhtd" else pool[ids, :, h]
                sc = torch.where(good.view(-1, 1), sc[ids, h].double(), 0.0)
                return (p.double() * sc.unsqueeze(-1)).reshape(-1, D)[:ln]
            k, v = rows(s["K"], s["ks"]), rows(s["V"], s["vs"])
            sees = ln - n + torch.arange(n, device=DEV) + 1 if causal else torch.full((n,), ln, device=DEV)
            hidden = torch.arange(ln, device=DEV) >= sees.view(n, 1, 1)
            x = torch.einsum("igd,td->igt", q[t0: t0 + n, h * G: (h + 1) * G], k) * scale
            x = x.masked_fill(hidden, -np.inf)
            m = x.amax(-1, keepdim=True)
            e = torch.exp(x - torch.where(m == -np.inf, 0.0, m))
            e = torch.where(hidden, 0.0, e)
            p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
            at = (slice(t0, t0 + n), slice(h * G, (h + 1) * G))
            v0 = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)  # hidden values may be anything
            out[at], mean[at] = p @ v0, p @ v0.abs()
            a = torch.einsum("igd,td->igt", q[t0: t0 + n, h * G: (h + 1) * G].abs(), k.abs()) * scale
            size[at] = a.masked_fill(hidden, 0.0).amax(-1, keepdim=True)
            top[at] = torch.where(hidden.unsqueeze(-1).expand(n, 1, ln, 1), 0.0, v0.abs()).amax(2).expand(n, G, D)
    return out, mean, top, size


def close(got, s, want, dtype=None):
    import torch

    out, mean, top, size = want
    dtype = dtype or got.dtype
    tol = 2e-5 + 1e-4 * out.abs() + 2.5 * 2.0 ** -20 * size * mean
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * out.abs() + 2.0 ** -25 + 2.0 ** -17 * top
        tol = tol + (3 if dtype == torch.bfloat16 else 1) * 2.0 ** -11 * mean
    else:
        tol = tol + 2.0 ** -31 * float(s["len"].max()) * top
    rows = torch.zeros(got.shape[0], dtype=torch.bool, device=DEV)
    for b in range(len(s["n"])):
        rows[int(s["starts_host"][b]): int(s["starts_host"][b + 1])] = True
    d = (got.double() - out).abs()
    bad = ~(d <= tol) & rows.view(-1, 1, 1)
    assert not bad.any(), (int(bad.sum()), float(d[rows].max()), [int(x) for x in bad.nonzero()[0]])


def prefill(s, **kw):
    return kvd.paged_prefill(s["q"], s["K"], s["V"], s["ks"], s["vs"], s["table"], s["lens"], s["starts"],
                             layout=s["layout"], **kw)


def check(s, causal=True, out_dtype=None, scale=0.0):
    import torch

    want = oracle(s, causal, scale or None)
    out = torch.full(s["q"].shape, float("nan"), dtype=out_dtype or s["q"].dtype, device=DEV)
    for _ in range(2):
        got = prefill(s, causal=causal, out=out, softmax_scale=scale)
        assert got is out
        close(got, s, want)
        first, last = int(s["starts_host"][0]), int(s["starts_host"][-1])
        assert torch.isnan(out[:first]).all() and torch.isnan(out[last:]).all()  # left as they were
    assert kvd.device_status() == 0


# ------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,H,G,bs,layout", [
    (128, 2, 4, 16, "bhtd"), (128, 1, 8, 64, "bthd"), (128, 3, 1, 32, "bhtd"), (128, 2, 3, 16, "bthd"),
    (128, 1, 16, 128, "bhtd"), (64, 2, 1, 16, "bthd"), (64, 1, 8, 8, "bhtd"), (64, 2, 5, 7, "bhtd"),
    (128, 1, 2, 1, "bhtd"), (128, 1, 40, 24, "bthd"), (64, 1, 200, 16, "bhtd"), (96, 2, 2, 16, "bhtd"),
    (20, 1, 3, 5, "bthd"), (256, 1, 2, 16, "bhtd"), (128, 1, 4, 256, "bhtd"),
])
@pytest.mark.parametrize("causal", [True, False])
def test_matches_formula(dtype, D, H, G, bs, layout, causal):
    # no rows, no tokens, one of each, more rows than tokens, tile and block borders, odd lengths
    n = [0, 3, 1, 1, 5, 33, 64, 1, 129, 7]
    lens = [9, 0, 1, 300, 3, 33, 128, 257, 131, 500]
    s = make_case(len(n), n, lens, H, G, D, bs, dtype, layout, seed=D + G, extra=3, front=2)
    check(s, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out", [("bfloat16", "float32"), ("float16", "bfloat16"), ("float32", "float16"),
                                       ("float32", "bfloat16"), ("bfloat16", "float16"), ("float16", "float32")])
@pytest.mark.parametrize("D,G,n", [(128, 4, 150), (64, 1, 300), (128, 8, 2)])
def test_types_of_rows_and_output(dtype, out, D, G, n):
    import torch

    s = make_case(2, [n, 1], [n + 190, 77], 2, G, D, 16, dtype, seed=n)
    check(s, out_dtype=getattr(torch, out), scale=0.11)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G", [(128, 8), (64, 2)])
def test_long_contexts_and_many_requests(dtype, D, G):
    # contexts that are split over the GPU beside short ones, single tokens beside chunks
    check(make_case(3, [1, 6, 130], [9001, 20011, 15000], 2, G, D, 64, dtype, seed=5))
    rng = np.random.default_rng(6)
    n = rng.integers(0, 9, size=300)
    n[::40] = 70
    check(make_case(300, n, n + rng.integers(0, 200, size=300), 1, G, D, 16, dtype, "bthd", seed=6))
    check(make_case(1, [1300], [1300], 2, G, D, 32, dtype, seed=7))
    check(make_case(2, [700, 1], [90, 4000], 2, G, D, 32, dtype, seed=8), causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 80])
def test_scales_of_very_different_sizes(dtype, n):
    # k scales over four powers of ten in all (weights of one token), v scales over eight
    check(make_case(2, [n, n], [1500, 333], 1, 4, 128, 16, dtype, seed=9, k_spread=1e2))
    s = make_case(2, [n, n], [1500, 333], 1, 4, 128, 16, dtype, seed=10, v_spread=1e2)
    check(s)
    s["ks"].zero_()  # equal weights
    s["vs"][::2] = 0.0
    check(s)
    s["vs"].zero_()
    check(s)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("later_k,later_v", [(1.0, 1.0), (100.0, 1.0), (1.0, 1e22), (1.0, 1e-22), (100.0, 1e22)])
def test_sums_of_long_rows_when_later_tokens_weigh_more(D, later_k, later_v):
    # 32-bit outputs of long rows are summed in parts, with references that may lie far from each other
    s = make_case(18, [128] * 18, [6000 - 130 * (b % 3) for b in range(18)], 8, 1, D, 16, "float32", seed=4)
    late = s["table"].long()[:, 200:375].clamp(0, s["ks"].shape[0] - 1).flatten()  # blocks of tokens from 3,200 on
    if later_v > 1:
        s["vs"] *= 1e-11  # so that their sums stay far from fp32's end
    s["ks"][late] *= later_k
    s["vs"][late] *= later_v
    check(s)


@pytest.mark.gpu
@pytest.mark.parametrize("n,dtype,products", [(2, "float32", 64), (128, "float32", 64), (128, "float16", 512)])
def test_sums_of_long_rows_do_not_drift(n, dtype, products):
    # A product on the tensor cores cuts a sum off, at 2^-23 of it at most, always towards zero. With values above
    # zero all losses of a row have one sign: 32,768 tokens are 2,048 products of 16, or twice as many in two terms.
    # Sums in parts of at most so many products lose 2^-23 of a part each (parts are added with rounding to nearest,
    # whose error has no sign, and neither has that of fp16 weights and outputs: 2^-11 over the root of 10^6 values);
    # weights of two terms (2^-22), exponentials (2^-22) and the sum of weights are counted as 2^-20.
    import torch

    H = torch.cuda.get_device_properties(0).multi_processor_count  # a unit of work a CTA: rows are not split
    s = make_case(1, [n], [32768], H, 1, 64, 64, dtype, seed=3)
    s["V"] = s["V"].abs()
    got = prefill(s, causal=False)
    ids = s["table"][0, :512].long()
    loss = []
    for h in range(H):
        k, v = ((s[x][ids, h].double() * s[y][ids, h].double().unsqueeze(-1)).reshape(-1, 64) for x, y in (("K", "ks"), ("V", "vs")))
        want = torch.softmax(s["q"][:, h].double() @ k.T / 8, -1) @ v
        loss.append((got[:, h].double() / want - 1).mean())
    assert abs(float(torch.stack(loss).mean())) <= products * 2.0 ** -23 + 2.0 ** -20
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G,n", [(128, 8, 1), (128, 8, 40), (64, 1, 5), (64, 1, 200), (96, 1, 30)])
def test_what_a_row_does_not_see_does_not_matter(dtype, D, G, n):
    import torch

    ln, bs = 203, 16
    s = make_case(1, [n], [ln], 2, G, D, bs, dtype, seed=11)
    want = oracle(s)
    last = int(s["table_host"][0, ln // bs])
    for t, v in ((s["ks"], float("nan")), (s["vs"], float("inf"))):
        t[last, :, ln % bs:] = v  # behind the last token
    free = [i for i in range(s["ks"].shape[0]) if i not in s["table_host"][0, : -(-ln // bs)]]
    s["ks"][free], s["vs"][free] = float("inf"), float("nan")
    close(prefill(s, out_dtype=s["q"].dtype), s, want)
    if n > 1:  # the last token is hidden from all rows but its own
        s["ks"][last, :, ln % bs - 1], s["vs"][last, :, ln % bs - 1] = float("nan"), float("-inf")
        got = prefill(s, out_dtype=s["q"].dtype)
        s["n"], s["starts_host"] = np.array([n - 1]), np.array([0, n - 1])
        close(got, s, want)
        assert not torch.isfinite(got[n - 1]).any()
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_with_infinities_and_extremes(dtype):
    import torch

    s = make_case(2, [70, 3], [400, 90], 1, 4, 128, 16, dtype, seed=12)
    s["q"][5, 1, 3], s["q"][9, 0, 7], s["q"][71, 2, 0] = float("nan"), float("inf"), float("-inf")
    s["q"][20, 3] = 0.0
    s["q"][30, 2] = torch.finfo(s["q"].dtype).tiny
    s["q"][40, 1] = 0.0  # scores whole steps of 60 apart, equal ones bit for bit
    s["q"][40, 1, 5] = 6e4
    s["q"][41, 1] = s["q"][41, 1] * (2.0 ** -9)
    got = prefill(s, out_dtype=torch.float32)
    touched = torch.zeros(got.shape[:2], dtype=torch.bool, device=DEV)
    for t, h in ((5, 1), (9, 0), (71, 2)):
        assert not torch.isfinite(got[t, h]).any()
        touched[t, h] = True
        s["q"][t, h] = 0.0
    want = oracle(s)
    got = torch.where(touched.unsqueeze(-1), want[0].float(), got)
    close(got, s, want, torch.float32)


@pytest.mark.gpu
def test_one_token_of_each_request_is_a_decode():
    import torch

    n, lens = [1] * 9, [1, 16, 17, 900, 64, 5000, 31, 128, 129]
    s = make_case(9, n, lens, 2, 8, 128, 16, "bfloat16", seed=13)
    got = prefill(s, out_dtype=torch.float32)
    ref = kvd.paged_decode(s["q"], s["K"], s["V"], s["ks"], s["vs"], s["table"], s["lens"])
    # two evaluations, each within 2e-5 + 1e-4 |out| of the exact one
    assert ((got - ref).abs() <= 2 * (2e-5 + 1e-4 * ref.abs())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D,n", [(128, 1), (128, 100), (64, 40), (96, 10)])
def test_ids_outside_the_pool(D, n):
    s = make_case(2, [n, 2], [170, 60], 2, 2, D, 16, "float32", seed=14)
    s["table_host"][0, 3], s["table_host"][1, 0] = -1, s["ks"].shape[0]
    s["table"].copy_(kvd._types()[0].from_numpy(s["table_host"]))
    want = oracle(s)
    close(prefill(s), s, want)
    assert kvd.device_status() == kvd.KVD_STATUS_BAD_BLOCK


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(128, "bfloat16"), (64, "float32"), (128, "float32")])
def test_strides_and_alignment(D, dtype):
    """Rows and outputs that are parts of wider tensors, pools whose rows lie apart, bases off 16 bytes."""
    import torch

    s = make_case(3, [90, 1, 4], [290, 33, 65], 2, 4, D, 16, dtype, seed=15)
    want = oracle(s)
    T = s["q"].shape[0]
    for off, pad in ((0, 8), (8, 0), (1, 3)):
        row = (8 + pad) * (D + pad) + off
        wide = torch.zeros(T * row + 64, dtype=s["q"].dtype, device=DEV)
        q = torch.as_strided(wide, (T, 8, D), (row, D + pad, 1), off)
        q.copy_(s["q"])
        out = torch.as_strided(torch.full_like(wide, float("nan")), q.shape, q.stride(), off)
        got = kvd.paged_prefill(q, s["K"], s["V"], s["ks"], s["vs"], s["table"], s["lens"], s["starts"], out=out)
        close(got, s, want)
    for off, pad in ((16, 16), (0, 4), (3, 0)):
        pools = []
        for t in (s["K"], s["V"]):
            NB, H, bs, _ = t.shape
            flat = torch.zeros(NB * H * (bs * (D + pad)) + off, dtype=torch.int8, device=DEV)
            view = flat[off:].view(NB, H, bs, D + pad)[..., :D]
            view.copy_(t)
            pools.append(view)
        scales = []
        for t in (s["ks"], s["vs"]):
            view = torch.zeros((*t.shape[:2], t.shape[2] + 3), device=DEV)[..., 1: t.shape[2] + 1]
            view.copy_(t)
            scales.append(view)
        got = kvd.paged_prefill(s["q"], *pools, *scales, s["table"], s["lens"], s["starts"], out_dtype=s["q"].dtype)
        close(got, s, want)
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 150])
def test_caches_past_32_bits(n):
    """Blocks whose codes lie more than 2^32 bytes into the pools."""
    import torch

    NB, H, bs, D = 34000, 8, 128, 128
    s = make_case(1, [n], [700], H, 1, D, bs, "bfloat16", seed=16)
    want = oracle(s)
    K, V = (torch.zeros((NB, H, bs, D), dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros((NB, H, bs), device=DEV) for _ in range(2))
    ids = torch.tensor([NB - 1, 5, NB - 7, 33990, 12, NB - 3], dtype=torch.int32, device=DEV)
    old = s["table"][0, :6].long()
    for big, small in ((K, s["K"]), (V, s["V"]), (ks, s["ks"]), (vs, s["vs"])):
        big[ids.long()] = small[old]
    got = kvd.paged_prefill(s["q"], K, V, ks, vs, ids.view(1, -1).contiguous(), s["lens"], s["starts"], out_dtype=s["q"].dtype)
    close(got, s, want)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 100])
def test_graphs_streams_and_two_calls_at_once(n):
    import torch

    a = make_case(2, [n, 3], [n + 5000, 77], 2, 4, 128, 16, "bfloat16", seed=17)
    b = make_case(2, [n, 1], [n + 4000, 700], 2, 4, 128, 16, "bfloat16", seed=18)
    wants = [oracle(a), oracle(b)]
    outs, graphs = [torch.empty_like(x["q"]) for x in (a, b)], []
    size = max(kvd.paged_prefill_workspace_size(x["q"], x["K"], x["table"]) for x in (a, b))
    ws = torch.full((size,), 255, dtype=torch.uint8, device=DEV)  # needs no initialisation; one for both graphs
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for x, o in zip((a, b), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            prefill(x, out=o, workspace=ws)
        graphs.append(graph)
    for _ in range(2):
        for o in outs:
            o.fill_(float("nan"))
        for g in graphs:
            g.replay()
        for x, o, w in zip((a, b), outs, wants):
            close(o, x, w)
        # new lengths in the same graph
    a["lens"].sub_(9)
    a["len"] = a["len"] - 9
    graphs[0].replay()
    close(outs[0], a, oracle(a))
    # calls on two streams at once, each with scratch of its own
    torch.cuda.synchronize()
    for _ in range(3):
        got = [prefill(x, stream=st, out_dtype=torch.bfloat16) for x, st in ((a, side), (b, other), (a, other), (b, side))]
        torch.cuda.synchronize()
        for x, g, w in zip((a, b, a, b), got, (oracle(a), wants[1], oracle(a), wants[1])):
            close(g, x, w)
    assert kvd.device_status() == 0


@pytest.mark.gpu
def test_results_do_not_depend_on_other_requests_or_runs():
    import torch

    s = make_case(4, [40, 1, 300, 2], [4000, 9000, 1300, 64], 2, 8, 128, 16, "bfloat16", seed=19)
    first = prefill(s)
    for _ in range(5):
        assert torch.equal(prefill(s), first)


@pytest.mark.gpu
def test_starts_that_do_not_fit_are_clamped():
    import torch

    s = make_case(3, [5, 4, 6], [50, 40, 30], 1, 2, 64, 16, "float32", seed=20)
    want = oracle(s)
    s["starts"].copy_(torch.tensor([0, 5, 9, 400], dtype=torch.int32))
    close(prefill(s), s, want)
    out = torch.full_like(s["q"], float("nan"))
    s["starts"].copy_(torch.tensor([-3, 5, 2, 15], dtype=torch.int32))  # not ascending: any rows, none outside
    prefill(s, out=out)
    s["lens"].copy_(torch.tensor([1 << 30, -5, 30], dtype=torch.int32))
    s["table"].clamp_(0, s["ks"].shape[0] - 1)
    prefill(s, out=out)
    torch.cuda.synchronize()
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,B", [(3, 40), (200, 40)])
def test_starts_that_go_back_and_forth_stay_inside_the_workspace(T, B):
    """Every second request claims all rows: their work must not need more records than the workspace has room for."""
    import torch

    s = make_case(B, [T] * B, [9000] * B, 2, 4, 128, 16, "bfloat16", seed=21)
    q = s["q"][:T].contiguous()
    starts = torch.tensor([0, T] * (B // 2) + [0], dtype=torch.int32, device=DEV)
    size = kvd.paged_prefill_workspace_size(q, s["K"], s["table"])
    ws = torch.full((size + (64 << 20),), 171, dtype=torch.uint8, device=DEV)
    out = kvd.paged_prefill(q, s["K"], s["V"], s["ks"], s["vs"], s["table"], s["lens"], starts, workspace=ws[:size])
    torch.cuda.synchronize()
    assert bool((ws[size:] == 171).all()) and torch.isfinite(out).all()
    assert kvd.device_status() == 0


@pytest.mark.gpu
def test_no_rows():
    import torch

    s = make_case(2, [0, 0], [5, 0], 1, 1, 128, 16, "float32")
    assert prefill(s).shape == (0, 1, 128)
    s = make_case(1, [0], [50], 1, 1, 128, 16, "bfloat16", extra=4)
    out = torch.full_like(s["q"], 7.0)
    prefill(s, out=out)
    assert (out == 7.0).all()


# ------------------------------------------------------------------------ CPU
def prefill_desc(**kw):
    d = kvd.PagedPrefillDesc(2, 8, 2, 128, 10, 16, 100, 8, 1, 0, 256, 256, 256, 8, 2 * 16 * 128, 16 * 128, 128, 32, 16,
                             1024, 128, 1024, 128, 0.0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [
    dict(batch=0), dict(num_q_heads=0), dict(num_kv_heads=0), dict(num_q_heads=9), dict(head_dim=0), dict(head_dim=513),
    dict(num_rows=-1), dict(block_size=0), dict(num_blocks=0), dict(max_blocks_per_seq=0), dict(block_table_stride=7),
    dict(seq_lens=None), dict(row_starts=None), dict(block_table=None), dict(flags=1), dict(flags=2 | 4), dict(flags=8 | 16),
    dict(flags=32), dict(flags=64), dict(num_rows=1 << 28), dict(max_blocks_per_seq=1 << 27, block_table_stride=1 << 27)])
def test_bad_descriptors_are_refused(kw):
    L, d = kvd.lib(), prefill_desc(**kw)
    assert L.kvd_paged_prefill_workspace_size(ctypes.byref(d)) == 0
    assert L.kvd_paged_prefill_launch(ctypes.byref(d), *[256] * 6, 256, 1 << 40, None) == EINVAL


def test_bad_arguments_are_refused():
    L, d = kvd.lib(), prefill_desc()
    args = [256] * 6
    assert L.kvd_paged_prefill_launch(None, *args, 256, 1 << 40, None) == EINVAL
    for i in range(6):
        assert L.kvd_paged_prefill_launch(ctypes.byref(d), *args[:i], None, *args[i + 1:], 256, 1 << 40, None) == EINVAL
    assert L.kvd_paged_prefill_launch(ctypes.byref(d), *args, 264, 1 << 40, None) == EINVAL  # workspace off 16 bytes
    size = L.kvd_paged_prefill_workspace_size(ctypes.byref(d))
    if size:
        assert L.kvd_paged_prefill_launch(ctypes.byref(d), *args, 256, size - 1, None) == EINVAL
        assert L.kvd_paged_prefill_launch(ctypes.byref(d), *args, None, 0, None) == EINVAL
    assert L.kvd_paged_prefill_launch(ctypes.byref(prefill_desc(num_rows=0)), *[None] * 6, None, 0, None) == 0


def test_tensors_of_wrong_shapes_are_refused():
    import torch

    i32 = torch.int32
    q = torch.zeros((10, 8, 32))
    pools = [torch.zeros((10, 2, 16, 32), dtype=torch.int8) for _ in range(2)] + [torch.zeros((10, 2, 16)) for _ in range(2)]
    lens, table, starts = torch.zeros(4, dtype=i32), torch.zeros((4, 3), dtype=i32), torch.zeros(5, dtype=i32)
    good = dict(q=q, pools=pools, table=table, lens=lens, starts=starts)

    def call(more=None, **kw):
        a = good | kw
        kvd.paged_prefill(a["q"], *a["pools"], a["table"], a["lens"], a["starts"], **(more or {}))

    for bad in (dict(q=q.double()), dict(q=q[:, :7]), dict(q=torch.zeros((10, 8, 16))), dict(lens=lens.long()),
                dict(starts=starts[:4]), dict(table=table[:3]), dict(table=table.float()), dict(more=dict(layout="x")),
                dict(more=dict(out=q[:9])), dict(more=dict(out=q, out_dtype=torch.bfloat16)),
                dict(pools=[pools[0], pools[1], pools[2][:9], pools[3]])):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError, match="current CUDA device"):
        call()
