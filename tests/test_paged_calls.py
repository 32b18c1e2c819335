"""The bindings of the paged serving steps: streams, scratch, devices and outputs (no reference counterpart)."""
import ctypes

import pytest

import kvdecode as kvd
from test_blocks import DEV, EINVAL, _check_select, _same_plan, plan_inputs, plan_oracle, select_inputs


class _NoLaunch:
    """A library whose launches are counted and not made."""

    def __init__(self):
        self.names = []

    def __getattr__(self, name):
        if name.endswith("_size"):
            return lambda *args: 64
        return lambda *args: self.names.append(name) or 0


def _every_call():
    """(call, names of its tensors, tensors) of every paged serving step, all on the host."""
    import torch

    B, H, G, D, bs, MB, NB, T, k = 2, 2, 2, 64, 8, 4, 9, 3, 2
    i8, i32, i64 = torch.int8, torch.int32, torch.int64
    z = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype)  # noqa: E731
    pools = lambda: dict(k_pool=z(NB, H, bs, D, dtype=i8), v_pool=z(NB, H, bs, D, dtype=i8),  # noqa: E731
                         ks_pool=z(NB, H, bs), vs_pool=z(NB, H, bs))
    return [
        (lambda **t: kvd.paged_plan(block_size=bs, **t),
         dict(seq_lens=z(B, dtype=i32), new_lens=z(B, dtype=i32), block_table=z(B, MB, dtype=i32),
              free_blocks=z(NB, dtype=i32), free_count=z(1, dtype=i32), slot_map=z(T, dtype=i64),
              token_starts=z(B + 1, dtype=i32), seq_lens_out=z(B, dtype=i32), free_count_out=z(1, dtype=i32),
              workspace=z(16, dtype=torch.uint8))),
        (kvd.paged_write, dict(k_new=z(T, H, D), v_new=z(T, H, D), slot_map=z(T, dtype=i64), **pools(),
                               bounds=z(NB, H, 2, D, dtype=i8), bound_scale=z(NB, H))),
        (kvd.paged_read, dict(slot_map=z(T, dtype=i64), **pools(), k_out=z(T, H, D), v_out=z(T, H, D))),
        (lambda **t: kvd.block_select(block_size=bs, budget=k, last=1, **t),
         dict(q=z(B, H * G, D), bounds=z(NB, H, 2, D, dtype=i8), bound_scale=z(NB, H), block_table=z(B, MB, dtype=i32),
              seq_lens=z(B, dtype=i32), sel_table=z(B, H, k, dtype=i32), sel_lens=z(B, H, dtype=i32),
              workspace=z(256, dtype=torch.uint8))),
        (kvd.sparse_decode, dict(q=z(B, H * G, D), **pools(), sel_table=z(B, H, k, dtype=i32),
                                 sel_lens=z(B, H, dtype=i32), out=z(B, H * G, D), workspace=z(64, dtype=torch.uint8)))]


@pytest.mark.parametrize("which", range(5))
def test_tensors_of_another_device_are_refused(which, monkeypatch):
    """A tensor left on the host, or on another GPU than the rest, is a ValueError and nothing is launched: the
    library would take its address for one of the GPU's. Devices are pretended."""
    import torch

    call, tensors = _every_call()[which]
    lib = _NoLaunch()
    monkeypatch.setattr(kvd, "_lib", lib)
    monkeypatch.setattr(kvd, "_cuda", (None, lambda: 0), raising=False)
    with pytest.raises(ValueError):
        call(**tensors, stream=0)  # all on the host
    where = {}
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: where.get(id(t), 0))
    call(**tensors, stream=0)
    assert len(lib.names) == 1
    for name, t in tensors.items():
        for device in (-1, 1):
            where = {id(t): device}
            with pytest.raises(ValueError):
                call(**tensors, stream=0)
    assert len(lib.names) == 1


@pytest.mark.parametrize("which", range(5))
def test_tensors_of_a_gpu_that_is_not_current_are_refused(which, monkeypatch):
    """Launches go to the current device and are sized for it: tensors of another GPU are a ValueError there."""
    import torch

    call, tensors = _every_call()[which]
    lib = _NoLaunch()
    monkeypatch.setattr(kvd, "_lib", lib)
    monkeypatch.setattr(kvd, "_cuda", (None, lambda: 0), raising=False)
    for index, launches in ((0, 1), (1, 1)):
        monkeypatch.setattr(torch.Tensor, "get_device", lambda t: index)
        if index == 0:
            call(**tensors, stream=0)
        else:
            with pytest.raises(ValueError):
                call(**tensors, stream=0)
        assert len(lib.names) == launches


def test_workspaces_off_their_boundary_are_refused():
    """Workspaces hold 32-bit words: one on another boundary would be a misaligned access in the kernels. Host checks
    alone, nothing is launched."""
    L = kvd.lib()
    plan = kvd.PagedPlanDesc(4, 16, 8, 4, 10, 4)
    sparse = kvd.PagedDesc(batch=2, num_q_heads=8, num_kv_heads=2, head_dim=128, block_size=16, num_blocks=64,
                           max_blocks_per_seq=8, seq_lens=256, block_table=256, block_table_stride=8, o_stride_h=128)
    select = kvd.BlockSelectDesc(2, 8, 2, 64, 16, 40, 20, 8, 1, 2, 0, 256, 256, 20, 512, 64)
    for at in (257, 258, 259):
        assert L.kvd_paged_plan_launch(ctypes.byref(plan), *[256] * 9, at, 64, None) == EINVAL
        assert L.kvd_sparse_decode_launch(ctypes.byref(sparse), *[256] * 6, at, 1 << 20, None) == EINVAL
        assert L.kvd_block_select_launch(ctypes.byref(select), *[256] * 5, at, 1 << 20, None) == EINVAL


def test_selections_past_two_to_the_30_blocks_are_refused():
    """The kernels count blocks in 32 bits: a table of nearly 2^31 blocks of one token, or a budget of as many, would
    pass them. Such sizes do not reach a kernel; 2^30 do."""
    L = kvd.lib()

    def size(blocks, budget):
        d = kvd.BlockSelectDesc(1, 1, 1, 64, 1, 40, blocks, budget, 1, 2, 0, 256, 256, blocks, 64, 64)
        if blocks > 1 << 30 or budget > 1 << 30:
            assert L.kvd_block_select_launch(ctypes.byref(d), *[256] * 6, 1 << 62, None) == EINVAL
        return L.kvd_block_select_workspace_size(ctypes.byref(d))

    assert size(1 << 30, 8) == 4 << 30
    for blocks in ((1 << 30) + 1, (1 << 31) - 128, (1 << 31) - 1):
        assert size(blocks, 8) == 0
        size(100, blocks)


@pytest.mark.parametrize("which", [0, 3, 4])
def test_workspaces_with_gaps_are_refused(which, monkeypatch):
    """A strided view's bytes do not lie together; nothing is launched for it."""
    import torch

    call, tensors = _every_call()[which]
    lib = _NoLaunch()
    monkeypatch.setattr(kvd, "_lib", lib)
    monkeypatch.setattr(kvd, "_cuda", (None, lambda: 0), raising=False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    for gaps in (torch.zeros((512, 2), dtype=torch.uint8)[:, 0], torch.zeros(1, dtype=torch.uint8).expand(512)):
        with pytest.raises(ValueError):
            call(**{**tensors, "workspace": gaps}, stream=0)
    assert not lib.names


@pytest.mark.parametrize("given", ["k_out", "v_out"])
def test_read_makes_the_output_that_is_missing(given, monkeypatch):
    """One output given, part of a wider tensor: it is the one that the call fills and returns, and the other is made
    with its type and strides. Devices are pretended, nothing is launched."""
    import torch

    _, tensors = _every_call()[2]
    buffer = torch.empty((3, 4, 64), dtype=torch.bfloat16)[:, 1:3]
    tensors = {n: t for n, t in tensors.items() if n not in ("k_out", "v_out")}
    args = []

    class Lib:
        kvd_paged_read_launch = staticmethod(lambda *a: args.append(a) or 0)

    monkeypatch.setattr(kvd, "_lib", Lib())
    monkeypatch.setattr(kvd, "_cuda", (lambda device: 0, lambda: 0), raising=False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    out = kvd.paged_read(**tensors, **{given: buffer})
    at = 0 if given == "k_out" else 1
    assert out[at] is buffer and out[0].data_ptr() != out[1].data_ptr()
    assert out[1 - at].dtype == torch.bfloat16 and out[1 - at].stride() == buffer.stride()
    assert args[0][6:8] == (out[0].data_ptr(), out[1].data_ptr())
    with pytest.raises(ValueError):
        kvd.paged_read(**tensors, **{given: buffer}, dtype=torch.float32)
    with pytest.raises(ValueError):
        kvd.paged_read(**tensors, k_out=buffer, v_out=torch.empty_like(buffer), dtype=torch.float16)
    assert len(args) == 1


@pytest.mark.gpu
def test_read_into_one_given_output():
    """On the GPU: the given half of a fused buffer gets the rows, the other output the same as a call without any."""
    import torch

    x = _step_inputs()
    pools = (x["K"], x["V"], x["ks"], x["vs"])
    want = kvd.paged_read(x["slots"], *pools, dtype=torch.bfloat16)
    for at in (0, 1):
        wide = torch.zeros((5000, 3, 2, 64), dtype=torch.bfloat16, device=DEV)
        given = wide[:, 1]
        got = kvd.paged_read(x["slots"], *pools, **{("k_out", "v_out")[at]: given})
        assert got[at] is given and torch.equal(given, want[at]) and torch.equal(got[1 - at], want[1 - at])
        assert not wide[:, 0].any() and not wide[:, 2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("as_handle", [False, True])
def test_plan_on_a_side_stream_without_a_workspace(as_handle):
    """The workspace is zeroed on the stream that the plan runs on: work that waits on the current stream, and what
    the workspace's memory held before, change nothing. 20,000 slots are many CTAs, which count themselves in it."""
    import torch

    args = plan_inputs(3, 64, 16, 600, 4000, 2, 8, 7000)
    lens, new, table, free = (torch.from_numpy(a).to(DEV) for a in args[:4])
    count = torch.tensor([args[4]], dtype=torch.int32, device=DEV)
    slots = torch.full((20000,), 77, dtype=torch.int64, device=DEV)
    starts = torch.empty(65, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    stale = [torch.full((16,), 255, dtype=torch.uint8, device=DEV) for _ in range(64)]
    torch.cuda.synchronize()
    del stale
    torch.cuda._sleep(40_000_000)  # tens of milliseconds
    kvd.paged_plan(lens, new, table, free, count, 16, slots, starts,
                   stream=side.cuda_stream if as_handle else side)
    side.synchronize()
    torch.cuda.synchronize()
    got = (*(t.cpu().numpy() for t in (table, free)), int(count), *(t.cpu().numpy() for t in (lens, starts, slots)),
           kvd.device_status())
    _same_plan(got, plan_oracle(*args, 16, 20000))


class _Spy:
    """The library, with the arguments of every launch kept."""

    def __init__(self, lib):
        self.lib, self.args = lib, []

    def __getattr__(self, name):
        fn = getattr(self.lib, name)
        if not name.endswith("_launch"):
            return fn

        def call(*args):
            self.args.append(args)
            return fn(*args)

        return call


def _step_inputs(B=2, H=2, G=2, D=64, bs=16, MB=300):
    """Pools, bounds, tables, rows and queries of a serving step, on the GPU."""
    import torch

    g = torch.Generator(device=DEV).manual_seed(1)
    NB = B * MB
    x = dict(K=torch.randint(-127, 128, (NB, H, bs, D), dtype=torch.int8, device=DEV, generator=g),
             V=torch.randint(-127, 128, (NB, H, bs, D), dtype=torch.int8, device=DEV, generator=g),
             ks=torch.rand((NB, H, bs), device=DEV, generator=g) * 0.02,
             vs=torch.rand((NB, H, bs), device=DEV, generator=g) * 0.02,
             bounds=torch.randint(-127, 128, (NB, H, 2, D), dtype=torch.int8, device=DEV, generator=g),
             step=torch.rand((NB, H), device=DEV, generator=g),
             table=torch.randperm(NB, device=DEV, generator=g).to(torch.int32).view(B, MB),
             lens=torch.tensor([MB * bs, MB * bs - 7], dtype=torch.int32, device=DEV),
             slots=torch.randperm(NB * bs, device=DEV, generator=g)[:5000].to(torch.int64),
             q=torch.randn((B, H * G, D), device=DEV, generator=g), bs=bs)
    x["bounds"] = x["bounds"].sort(dim=2, descending=True).values.contiguous()
    return x


def _step_calls(x, stream):
    """Every call that makes scratch or outputs of its own, as (outputs, pointers of the scratch)."""
    import torch

    spy = _Spy(kvd.lib())
    kvd._lib, real = spy, kvd._lib
    try:
        grow = torch.zeros_like(x["lens"])
        count = torch.zeros(1, dtype=torch.int32, device=DEV)
        free = torch.empty(x["K"].shape[0], dtype=torch.int32, device=DEV)
        slots = torch.empty(600, dtype=torch.int64, device=DEV)
        torch.cuda.synchronize()
        _, starts = kvd.paged_plan(x["lens"], grow, x["table"], free, count, x["bs"], slots, stream=stream)
        rows = kvd.paged_read(x["slots"], x["K"], x["V"], x["ks"], x["vs"], stream=stream)
        sel, sl = kvd.block_select(x["q"], x["bounds"], x["step"], x["table"], x["lens"], x["bs"], 40, stream=stream)
        out = kvd.sparse_decode(x["q"], x["K"], x["V"], x["ks"], x["vs"], sel, sl, stream=stream)
    finally:
        kvd._lib = real
    scratch = [args[-3] for args in (spy.args[0], spy.args[2], spy.args[3])]
    torch.cuda.synchronize()
    return (starts, *rows, sel, sl, out), scratch


@pytest.mark.gpu
@pytest.mark.parametrize("as_handle", [False, True])
def test_what_a_call_makes_belongs_to_its_stream(as_handle):
    """Scratch and outputs of calls on a side stream are memory of that stream: once dropped they are not handed to
    the current stream, on which nothing waits for the call. The results are those of the current stream's calls."""
    import torch

    x = _step_inputs()
    want, _ = _step_calls(x, None)
    side = torch.cuda.Stream()
    got, scratch = _step_calls(x, side.cuda_stream if as_handle else side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    sizes = [t.nbytes for t in got] + [16, 2 * 2 * 300 * 4]
    at = {t.data_ptr() for t in got} | set(scratch)
    assert None not in at and 0 not in at
    del got, a, b
    for n in sizes:  # what the calls had is not handed out here
        again = [torch.empty(n, dtype=torch.uint8, device=DEV) for _ in range(8)]
        assert not at & {t.data_ptr() for t in again}
    side.synchronize()
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("as_handle", [False, True])
def test_scratch_of_the_dense_and_paged_calls_belongs_to_their_stream(as_handle):
    """The same of the decode, append-decode, paged decode, prefill, combine and row quantiser."""
    import torch

    B, H, G, S, D, bs = 2, 2, 4, 4096, 128, 16
    g = torch.Generator(device=DEV).manual_seed(2)
    rnd = lambda *shape: torch.randn(shape, device=DEV, generator=g)  # noqa: E731
    K, V = (torch.randint(-127, 128, (B, H, S, D), dtype=torch.int8, device=DEV, generator=g) for _ in range(2))
    ks, vs = (torch.rand((B, H, S), device=DEV, generator=g) * 0.02 for _ in range(2))
    Kp, Vp = (t.view(B, H, S // bs, bs, D).transpose(1, 2).reshape(-1, H, bs, D).contiguous() for t in (K, V))
    ksp, vsp = (t.view(B, H, S // bs, bs).transpose(1, 2).reshape(-1, H, bs).contiguous() for t in (ks, vs))
    table = torch.arange(B * S // bs, dtype=torch.int32, device=DEV).view(B, -1)
    full = torch.full((B,), S, dtype=torch.int32, device=DEV)
    q, kn, vn, qp = rnd(B, H * G, D), rnd(B, H, D), rnd(B, H, D), rnd(B, H * G, 64, D)
    parts, rows = rnd(3, 5, D + 4).abs(), rnd(7, D)

    def calls(stream):
        spy = _Spy(kvd.lib())
        kvd._lib, real = spy, kvd._lib
        try:
            lens = full - 1
            k2, v2, ks2, vs2 = K.clone(), V.clone(), ks.clone(), vs.clone()
            torch.cuda.synchronize()
            outs = [kvd.decode(q, K, V, ks, vs, stream=stream),
                    kvd.append_decode(kn, vn, q, k2, v2, ks2, vs2, lens, stream=stream),
                    kvd.prefill(qp, K, V, ks, vs, stream=stream),
                    kvd.paged_decode(q, Kp, Vp, ksp, vsp, table, full, stream=stream),
                    kvd.combine(parts, stream=stream), *kvd.quantize_rows(rows, stream=stream)]
        finally:
            kvd._lib = real
        torch.cuda.synchronize()
        return outs, [args[-3] for args in spy.args[:4]], [args[-2] for args in spy.args[:4]]  # workspaces

    want, _, _ = calls(None)
    side = torch.cuda.Stream()
    got, scratch, bytes_ = calls(side.cuda_stream if as_handle else side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    at = {t.data_ptr() for t in got} | set(scratch)
    sizes = [t.nbytes for t in got] + bytes_
    del got, a, b
    for n in sizes:
        again = [torch.empty(n, dtype=torch.uint8, device=DEV) for _ in range(8)]
        assert not at & {t.data_ptr() for t in again}
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(5))
def test_host_tensors_among_the_gpu_s_are_refused(which):
    """As above with real devices: every tensor in turn is left on the host. Refused before anything is launched."""
    import torch

    call, tensors = _every_call()[which]
    there = {name: t.to(DEV) for name, t in tensors.items()}
    for name in tensors:
        with pytest.raises(ValueError):
            call(**{**there, name: tensors[name]})
    torch.cuda.synchronize()
    assert kvd.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("G,D,MB", [(97, 512, 40), (200, 256, 40), (800, 64, 37), (480, 100, 50), (65, 128, 90)])
def test_select_of_wide_groups(G, D, MB):
    """Groups whose query codes do not fit into shared memory together are scored a part at a time."""
    bs, k = 16, 9
    lens = [MB * bs, (k + 1) * bs - 3, k * bs]
    q, bounds, step, table, lens = select_inputs(G, 3, 2, G, D, bs, MB, lens)
    q *= 0.1 + 0.9 * (abs(q[:, :, :1]) > 1.8)  # the heads that weigh most lie anywhere in the group
    step[3::11] = float("nan")
    table[0, 5], table[1, 2] = -1, 10 ** 8
    _check_select(q, bounds, step, table, lens, bs, k, 1, 2)
    assert kvd.device_status() == kvd.KVD_STATUS_BAD_BLOCK
