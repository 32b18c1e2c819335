"""Cases that measure the paged sparse-attention operators of kvdecode against their plain torch forms.

Five operators make the serving steps over a paged INT8 KV cache that read only part of a long context:

* ``plan``   block tables and slot maps from the requests' lengths (``kvdecode.paged_plan``);
* ``write``  new K/V rows quantised into the slots of the map, with the bounds of every touched
             block's keys (``kvdecode.paged_write``), then read back by slot as the values that the
             8-bit rows stand for, which is what a prompt's own attention sees (``kvdecode.paged_read``);
* ``select`` blocks that a cheap upper bound of q.k scores highest, per request and KV head
             (``kvdecode.block_select``);
* ``decode`` attention of one new token over the selected blocks (``kvdecode.sparse_decode``).

``own`` chooses the side that ``run`` computes: False, elementary torch operations in 32 bits;
True, the library's calls.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _kvd():
    here = os.path.join(os.getcwd(), "cuda-operators_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import kvdecode

    return kvdecode


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a few requests with short blocks: launch latency is all of it
        {"name": "plan 8 requests, one token each", "op": "plan", "B": 8, "bs": 16, "max_blocks": 512, "slots": 8,
         "prompts": 0, "ends": 0, "spare": 64},
        # a decode step of the 256-request GQA configuration, some requests ending and some arriving
        {"name": "plan 256 requests, some end", "op": "plan", "B": 256, "bs": 64, "max_blocks": 128, "slots": 4096,
         "prompts": 6, "ends": 9, "spare": 2048},
        # a mixed step with chunked prompts; the pool runs short, so the last ones are refused
        {"name": "plan 1024 requests, 65536 tokens", "op": "plan", "B": 1024, "bs": 16, "max_blocks": 1024,
         "slots": 65536, "prompts": 37, "ends": 20, "spare": 3500},
        # the new token of 256 requests (decode step), pool rows of all heads together
        {"name": "write 256 decode rows bf16", "op": "write", "T": 256, "B": 256, "Hkv": 8, "D": 128, "bs": 16,
         "dtype": "bf16", "layout": "bthd"},
        # a few odd prompts in fp32
        {"name": "write 5003 prompt rows fp32", "op": "write", "T": 5003, "B": 7, "Hkv": 8, "D": 128, "bs": 64,
         "dtype": "fp32", "layout": "bhtd"},
        # a large chunked-prefill step
        {"name": "write 32768 prompt rows bf16", "op": "write", "T": 32768, "B": 24, "Hkv": 8, "D": 128, "bs": 64,
         "dtype": "bf16", "layout": "bhtd"},
        # one request with a long context, GQA: latency
        {"name": "select 1 x 32768 gqa", "op": "select", "B": 1, "Hkv": 8, "G": 8, "D": 128, "bs": 64, "S": 32768,
         "k": 32, "dtype": "bf16"},
        # the long-context MHA configuration (B=4, 32 heads, 131072 tokens)
        {"name": "select 4 x 131072 mha", "op": "select", "B": 4, "Hkv": 32, "G": 1, "D": 128, "bs": 128,
         "S": 131072, "k": 64, "dtype": "fp32"},
        # many long requests with short blocks
        {"name": "select 64 x 131071 gqa", "op": "select", "B": 64, "Hkv": 8, "G": 8, "D": 128, "bs": 32,
         "S": 131071, "k": 128, "dtype": "bf16"},
        # one request: latency
        {"name": "decode 1 x 2048 of 32768 gqa", "op": "decode", "B": 1, "Hkv": 8, "G": 8, "D": 128, "bs": 64,
         "S": 32768, "k": 32, "dtype": "bf16", "layout": "bhtd"},
        # 4 requests, 32 heads (MHA), 4096 tokens selected of long contexts
        {"name": "decode 4 x 4096 of 32767 mha", "op": "decode", "B": 4, "Hkv": 32, "G": 1, "D": 128, "bs": 128,
         "S": 32767, "k": 32, "dtype": "fp32", "layout": "bhtd"},
        # the 256-request GQA configuration: 2048 of up to 8192 tokens, short blocks
        {"name": "decode 256 x 2048 of 8192 gqa", "op": "decode", "B": 256, "Hkv": 8, "G": 8, "D": 128, "bs": 16,
         "S": 8192, "k": 128, "dtype": "bf16", "layout": "bthd"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "write", "select", "decode"])
    if op == "plan":
        B = _log(rng, 1, 1024)
        prompts = rng.randint(0, max(0, min(40, B // 3)))
        ends = rng.randint(0, max(0, min(40, B // 4)))
        tokens = B - prompts - ends + (_log(rng, 1, 65536 - B) if prompts else 0)
        return {"op": op, "B": B, "bs": rng.choice([8, 16, 24, 32, 64, 128]), "max_blocks": _log(rng, 64, 1024),
                "slots": tokens + rng.choice([0, 0, 5]), "prompts": prompts, "ends": ends,
                "spare": _log(rng, 16, 8192)}
    if op == "write":
        T = _log(rng, 1, 32768)
        return {"op": op, "T": T, "B": rng.choice([T if T <= 512 else 3, max(1, T // 700)]), "Hkv": rng.choice([1, 2, 4, 8]),
                "D": rng.choice([64, 128, 128, 256 if T < 8192 else 128]), "bs": rng.choice([8, 16, 32, 64, 128]),
                "dtype": rng.choice(list(TYPES)), "layout": rng.choice(["bhtd", "bthd"])}
    S = _log(rng, 1000, 131072 if op == "select" else 32768)
    bs = rng.choice([16, 32, 64, 128])
    Hkv = rng.choice([1, 2, 4, 8, 32])
    G = rng.choice([1, 2, 4, 8, 16]) if Hkv < 32 else 1
    k = min(_log(rng, 8, 256), max(4, S // bs // 3))
    if op == "select":
        top = 64 * 8 * 131072 // 32  # blocks x heads of the largest listed case
        B = _log(rng, 1, max(1, min(256, top // (Hkv * -(-S // bs)))))
        return {"op": op, "B": B, "Hkv": Hkv, "G": G, "D": rng.choice([64, 128]), "bs": bs, "S": S, "k": k,
                "dtype": rng.choice(list(TYPES))}
    top = 256 * 8 * 2048  # tokens x heads read by the largest listed case
    B = _log(rng, 1, max(1, min(256, top // (Hkv * k * bs), 8 * top // 2 // (Hkv * S))))
    return {"op": op, "B": B, "Hkv": Hkv, "G": G, "D": 128, "bs": bs, "S": S, "k": k, "dtype": rng.choice(list(TYPES)),
            "layout": rng.choice(["bhtd", "bthd"])}


def work(case):
    c, op = case, case["op"]
    if op == "plan":
        # lengths in and out, the slot map, and a table entry and a free-list entry per new block
        blocks = c["slots"] // c["bs"] + c["B"]
        return {"bytes": 4 * 5 * c["B"] + 8 * c["slots"] + 8 * blocks, "flops": 0}
    if op == "write":
        rows = 2 * c["T"] * c["Hkv"]
        e = TYPES[c["dtype"]].itemsize
        written = rows * (c["D"] * e + c["D"] + 4) + 8 * c["T"]  # the rows in, codes and scales out
        read = rows * (c["D"] + 4 + c["D"] * e)  # codes and scales in, values out
        bounds = (c["T"] // c["bs"] + c["B"]) * c["Hkv"] * (2 * c["D"] + 4)
        return {"bytes": written + read + bounds, "flops": 6 * rows * c["D"]}
    if op == "select":
        n = 0.75 * c["B"] * c["Hkv"] * c["S"] / c["bs"]  # lengths are even over [S/2, S]
        q = c["B"] * c["Hkv"] * c["G"] * c["D"]
        return {"bytes": int(n * (2 * c["D"] + 4)) + q * TYPES[c["dtype"]].itemsize + 4 * c["B"] * c["Hkv"] * c["k"],
                "flops": int(n * c["G"] * 4 * c["D"])}
    n = c["B"] * c["Hkv"] * c["k"] * c["bs"]
    q = c["B"] * c["Hkv"] * c["G"] * c["D"]
    return {"bytes": n * (2 * c["D"] + 8) + 2 * q * TYPES[c["dtype"]].itemsize + 4 * c["B"] * c["Hkv"] * c["k"],
            "flops": 4 * n * c["G"] * c["D"]}


# ----------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"plan": _prepare_plan, "write": _prepare_write, "select": _prepare_select, "decode": _prepare_decode}[c["op"]](c, gen, rng)
    s["case"] = c
    if own:
        s["kvd"] = _kvd()
    return s


def _split(rng, total, parts):
    """`total` as `parts` random whole numbers of at least 1."""
    if parts <= 1:
        return np.full(parts, total, np.int64)
    cuts = np.sort(rng.choice(np.arange(1, total), size=parts - 1, replace=False)) if total > parts else np.arange(1, parts)
    return np.diff(np.concatenate([[0], cuts, [max(total, parts)]])).astype(np.int64)


def _prepare_plan(c, gen, rng):
    B, bs, MB = c["B"], c["bs"], c["max_blocks"]
    lens = rng.integers(1, max(2, MB * bs * 3 // 4), size=B)
    new = np.ones(B, np.int64)
    who = rng.permutation(B)
    ends, prompts = who[: c["ends"]], who[c["ends"]: c["ends"] + c["prompts"]]
    new[ends] = -1
    if c["prompts"]:
        room = max(c["prompts"], c["slots"] - (B - c["prompts"] - c["ends"]))
        new[prompts] = _split(rng, room, c["prompts"])
        lens[prompts] = np.where(rng.random(c["prompts"]) < 0.7, 0, lens[prompts] // 2)
    held = -(-lens // bs)
    NB = B * (MB * 3 // 4 + 1) + c["spare"]  # what no request holds and is not free belongs to others
    ids = rng.permutation(NB).astype(np.int32)
    table = np.full((B, MB), -1, np.int32)
    at = 0
    for b in range(B):
        table[b, : held[b]] = ids[at: at + held[b]]
        at += held[b]
    free = np.full(NB, -1, np.int32)
    free[: c["spare"]] = ids[at: at + c["spare"]]
    dev = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to(DEV, t)  # noqa: E731
    s = {"lens": dev(lens, torch.int32), "new": dev(new, torch.int32), "table": dev(table, torch.int32),
         "free": dev(free, torch.int32), "count": dev(np.array([c["spare"]]), torch.int32), "NB": NB}
    s["slots"] = torch.empty(c["slots"], dtype=torch.int64, device=DEV)
    s["starts"] = torch.empty(B + 1, dtype=torch.int32, device=DEV)
    s["lens_out"], s["count_out"] = torch.empty_like(s["lens"]), torch.empty_like(s["count"])
    s["ws"] = torch.zeros(16, dtype=torch.uint8, device=DEV)
    return s


def _write_blocks(c):
    """Pool blocks of a write case: what its requests can touch."""
    return c["T"] // c["bs"] + 2 * c["B"]


def _prepare_write(c, gen, rng):
    T, B, H, D, bs = c["T"], c["B"], c["Hkv"], c["D"], c["bs"]
    n = _split(rng, T, B)[:B]
    start = rng.integers(0, bs, size=B)  # fill of each request's last block
    start[rng.random(B) < 0.3] = 0
    NB = _write_blocks(c)
    ids, at, slots = rng.permutation(NB), 0, []
    for b in range(B):
        pos = start[b] + np.arange(n[b])
        blocks = ids[at: at + pos[-1] // bs + 1]
        at += len(blocks)
        slots.append(blocks[pos // bs] * bs + pos % bs)
    if B >= 8:
        slots[B // 2][:] = -1  # a request that the plan refused
    slots = np.concatenate(slots)[:T]
    shape = (NB + 1, H, bs, D) if c["layout"] == "bhtd" else (NB + 1, bs, H, D)  # one block past the pool: a place
    s = {"NB": NB, "slots": torch.from_numpy(slots.astype(np.int64)).to(DEV)}   # for the plain form's refused rows
    for x in "kv":
        s[x + "_pool"] = torch.randint(-127, 128, shape, dtype=torch.int8, device=DEV, generator=gen)
        s[x + "_scale"] = torch.rand((NB + 1, H, bs), device=DEV, generator=gen) * 0.02 + 0.01
        rows = torch.randn((T, H, D), device=DEV, generator=gen)
        s[x] = (rows * torch.exp(0.5 * torch.randn((T, H, 1), device=DEV, generator=gen))).to(TYPES[c["dtype"]])
    s["k_read"], s["v_read"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    s["bounds"] = torch.zeros((NB + 1, H, 2, D), dtype=torch.int8, device=DEV)
    s["bound_scale"] = torch.zeros((NB + 1, H), device=DEV)
    return s


def _prepare_select(c, gen, rng):
    B, H, G, D, bs = c["B"], c["Hkv"], c["G"], c["D"], c["bs"]
    MB = -(-c["S"] // bs)
    NB = B * MB + 7
    lens = rng.integers(c["S"] // 2, c["S"] + 1, size=B).astype(np.int32)
    lens[0] = c["S"]
    s = {"lens": torch.from_numpy(lens).to(DEV),
         "table": torch.randperm(NB, device=DEV, generator=gen)[: B * MB].view(B, MB).to(torch.int32)}
    centre = torch.randint(-60, 61, (NB, H, 1, D), dtype=torch.int8, device=DEV, generator=gen)
    half = torch.randint(0, 65, (NB, H, 1, D), dtype=torch.int8, device=DEV, generator=gen)
    s["bounds"] = torch.cat([centre + half, centre - half], dim=2)
    s["bound_scale"] = torch.exp(0.3 * torch.randn((NB, H), device=DEV, generator=gen)) * 0.02
    s["q"] = torch.randn((B, H * G, D), device=DEV, generator=gen).to(TYPES[c["dtype"]])
    s["sel"] = torch.empty((B, H, c["k"]), dtype=torch.int32, device=DEV)
    s["sel_lens"] = torch.empty((B, H), dtype=torch.int32, device=DEV)
    return s


FIRST, LAST = 1, 2  # blocks that are always read: the first one and the newest two


def _prepare_decode(c, gen, rng):
    B, H, G, D, bs, k = c["B"], c["Hkv"], c["G"], c["D"], c["bs"], c["k"]
    MB = -(-c["S"] // bs)
    NB = B * MB + 3
    lens = rng.integers(max(c["S"] // 2, min(c["S"], (k - 1) * bs + 1)), c["S"] + 1, size=B)
    n = torch.from_numpy(-(-lens // bs)).to(DEV)
    tail = torch.from_numpy(lens - (-(-lens // bs) - 1) * bs).to(DEV)
    order = torch.rand((B, H, MB), device=DEV, generator=gen)
    j = torch.arange(MB, device=DEV)
    order.masked_fill_(j >= n.view(B, 1, 1), -1.0)
    order.masked_fill_(j == n.view(B, 1, 1) - 1, 2.0)  # the newest block is always read
    idx = order.topk(k, dim=-1).indices.sort(dim=-1).values
    table = torch.randperm(NB, device=DEV, generator=gen)[: B * MB].view(B, MB)
    shape = (NB, H, bs, D) if c["layout"] == "bhtd" else (NB, bs, H, D)
    s = {"sel": table.view(B, 1, MB).expand(B, H, MB).gather(2, idx).to(torch.int32),
         "sel_lens": ((k - 1) * bs + tail).view(B, 1).expand(B, H).contiguous().to(torch.int32)}
    for x in "kv":
        s[x + "_pool"] = torch.randint(-127, 128, shape, dtype=torch.int8, device=DEV, generator=gen)
        s[x + "_scale"] = torch.rand((NB, H, bs), device=DEV, generator=gen) * 0.02 + 0.005
    s["q"] = torch.randn((B, H * G, D), device=DEV, generator=gen).to(TYPES[c["dtype"]])
    s["out"] = torch.empty_like(s["q"])
    if own:  # scratch that a serving loop keeps
        s["ws"] = torch.empty(_kvd().sparse_workspace_size(s["q"], s["k_pool"], s["sel"], c["layout"]), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------------------------------------- runs
def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "write": _own_write, "select": _own_select, "decode": _own_decode}[op](state)
    return {"plan": _plain_plan, "write": _plain_write, "select": _plain_select, "decode": _plain_decode}[op](state)


def _own_plan(s):
    s["kvd"].paged_plan(s["lens"], s["new"], s["table"], s["free"], s["count"], s["case"]["bs"], s["slots"], s["starts"],
                        seq_lens_out=s["lens_out"], free_count_out=s["count_out"], workspace=s["ws"])
    return {"table": s["table"], "slots": s["slots"], "starts": s["starts"], "lens": s["lens_out"], "free": s["free"],
            "count": s["count_out"]}


def _own_write(s):
    NB = s["NB"]
    kp, vp, ks, vs = s["k_pool"][:NB], s["v_pool"][:NB], s["k_scale"][:NB], s["v_scale"][:NB]
    bounds, bscale = s["bounds"][:NB], s["bound_scale"][:NB]
    s["kvd"].paged_write(s["k"], s["v"], s["slots"], kp, vp, ks, vs, bounds=bounds, bound_scale=bscale, layout=s["case"]["layout"])
    s["kvd"].paged_read(s["slots"], kp, vp, ks, vs, k_out=s["k_read"], v_out=s["v_read"], layout=s["case"]["layout"])
    return _written(s["k_read"], s["v_read"], ks, vs, bounds, bscale)


def _own_select(s):
    c = s["case"]
    s["kvd"].block_select(s["q"], s["bounds"], s["bound_scale"], s["table"], s["lens"], c["bs"], c["k"], first=FIRST,
                          last=LAST, sel_table=s["sel"], sel_lens=s["sel_lens"])
    return {"sel": s["sel"], "lens": s["sel_lens"]}


def _own_decode(s):
    return s["kvd"].sparse_decode(s["q"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["sel"], s["sel_lens"],
                                  out=s["out"], layout=s["case"]["layout"], workspace=s["ws"])


def _plain_plan(s):
    c = s["case"]
    bs, MB, NB, T = c["bs"], c["max_blocks"], s["NB"], c["slots"]
    lens, new, table, free, fc = s["lens"].long(), s["new"].long(), s["table"], s["free"], s["count"].long()
    ending = new < 0
    n = new.clamp(min=0)
    held = (lens + bs - 1) // bs
    stop = n.cumsum(0)
    start = stop - n
    over = (lens + n > MB * bs) | (stop > T)
    need = ((lens + n + bs - 1) // bs - held).masked_fill(ending | over, 0)
    back = held.masked_fill(~ending, 0)
    back_stop = back.cumsum(0)
    total = fc + back_stop[-1]
    need_stop = need.cumsum(0)
    ok = ~ending & ~over & ((need == 0) | (need_stop <= total))
    take = need * ok
    left = total - take.sum()

    def stack(i):  # entry i of the free list with the ended requests' blocks on top
        r = i - fc
        b = torch.searchsorted(back_stop, r.clamp(min=0), right=True).clamp(max=lens.numel() - 1)
        j = (r - (back_stop[b] - back[b])).clamp(0, MB - 1)
        return torch.where(r < 0, free[i.clamp(0, NB - 1)], table[b, j])

    j = torch.arange(MB, device=DEV)
    first = (need_stop - need).unsqueeze(1)
    fresh = (j >= held.unsqueeze(1)) & (j < (held + take).unsqueeze(1))
    table_out = torch.where(fresh, stack(total - 1 - (first + j - held.unsqueeze(1))), table)
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(stop, t, right=True).clamp(max=lens.numel() - 1)
    pos = lens[b] + t - start[b]
    slots = table_out[b, (pos // bs).clamp(0, MB - 1)].long() * bs + pos % bs
    slots = torch.where(ok[b] & (t < stop[-1]), slots, -1)
    v = torch.arange(NB, device=DEV)
    free_out = torch.where((v >= fc) & (v < left), stack(v), free)
    lens_out = torch.where(ending, 0, torch.where(ok, lens + n, lens))
    starts = torch.cat([torch.zeros_like(stop[:1]), stop]).clamp(max=T)
    return {"table": table_out, "slots": slots, "starts": starts.int(), "lens": lens_out.int(), "free": free_out,
            "count": left.int()}


def _divide(a, b):
    """a / b rounded once: by a Python number torch multiplies by its rounded reciprocal instead."""
    return a / torch.full_like(a, b)


def _plain_quantise(x):
    x = x.float()
    scale = _divide(x.abs().amax(-1), 127.0)
    s = scale.unsqueeze(-1)
    codes = torch.where(s > 0, (x / s).round().clamp(-127, 127), 0.0)
    return codes.to(torch.int8), scale


def _plain_write(s):
    c, NB, bs = s["case"], s["NB"], s["case"]["bs"]
    slots = torch.where(s["slots"] < 0, NB * bs, s["slots"])
    blk, off = slots // bs, slots % bs
    for x in "kv":
        codes, scale = _plain_quantise(s[x])
        if c["layout"] == "bhtd":
            s[x + "_pool"][blk, :, off] = codes
        else:
            s[x + "_pool"][blk, off] = codes
        s[x + "_scale"][blk, :, off] = scale
    # bounds of the blocks that were written to, over the tokens up to the newest one of each
    last = torch.full((NB + 1,), -1, dtype=torch.int64, device=DEV).scatter_reduce_(0, blk, off, "amax")
    at = (last[:NB] >= 0).nonzero().squeeze(1)
    codes = s["k_pool"][at].float()
    codes = codes if c["layout"] == "bhtd" else codes.transpose(1, 2)
    scale = s["k_scale"][at].unsqueeze(-1)
    out = (torch.arange(bs, device=DEV) > last[at].unsqueeze(1)).view(-1, 1, bs, 1)
    value = codes * scale
    hi = value.masked_fill(out, -math.inf).amax(2)
    lo = value.masked_fill(out, math.inf).amin(2)
    step = _divide(torch.maximum(hi.abs(), lo.abs()).amax(-1), 127.0)
    d = step.unsqueeze(-1)
    some = d > 0
    s["bounds"][at, :, 0] = torch.where(some, (hi / d).ceil().clamp(-127, 127), 0.0).to(torch.int8)
    s["bounds"][at, :, 1] = torch.where(some, (lo / d).floor().clamp(-127, 127), 0.0).to(torch.int8)
    s["bound_scale"][at] = step
    # read the rows back as the values that their codes stand for; a refused row reads as zeros
    there = (s["slots"] >= 0).view(-1, 1, 1)
    rows = {}
    for x in "kv":
        codes = s[x + "_pool"][blk, :, off] if c["layout"] == "bhtd" else s[x + "_pool"][blk, off]
        value = codes.float() * s[x + "_scale"][blk, :, off].unsqueeze(-1)
        rows[x] = torch.where(there, value, 0.0).to(s[x].dtype)
    return _written(rows["k"], rows["v"], *(s[x][:NB] for x in ("k_scale", "v_scale", "bounds", "bound_scale")))


def _written(k, v, ks, vs, bounds, bscale):
    """The rows that were written, the scale pools, and the bounds as the values that they stand for."""
    return {"k": k, "v": v, "ks": ks, "vs": vs, "bounds": torch.mul(bounds, bscale.view(bscale.shape + (1, 1))),
            "bscale": bscale}


def _plain_select(s):
    c = s["case"]
    B, H, G, D, bs, k = c["B"], c["Hkv"], c["G"], c["D"], c["bs"], c["k"]
    MB = s["table"].shape[1]
    codes, scale = _plain_quantise(s["q"])
    qc = codes.float().view(B, H, G, D)
    qc = torch.cat([qc.clamp(min=0), qc.clamp(max=0)], dim=-1)  # meets [upper, lower] bounds: the larger product each
    table = s["table"].long()
    rows = s["bounds"][table].float().view(B, MB, H, 2 * D)
    dots = torch.einsum("bhgd,bnhd->bhgn", qc, rows)  # whole numbers below 2^24: exact in any order
    score = (dots * scale.view(B, H, G, 1)).amax(2) * s["bound_scale"][table].transpose(1, 2)
    score = torch.where(torch.isnan(score), math.inf, score)
    n = ((s["lens"] + bs - 1) // bs).view(B, 1, 1)
    j = torch.arange(MB, device=DEV).view(1, 1, MB)
    always = (j < FIRST) | ((j >= n - LAST) & (j < n))
    score = score.masked_fill(j >= n, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices
    rank = always.expand(B, H, MB).gather(2, order).to(torch.int8).sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(2, rank)[..., :k]
    count = n.clamp(max=k)
    order = torch.where(torch.arange(k, device=DEV) < count, order, MB).sort(dim=-1).values
    ids = table.view(B, 1, MB).expand(B, H, MB).gather(2, order.clamp(max=MB - 1))
    sel = torch.where(order < MB, ids, -1).int()
    lens = ((count - n) * bs).squeeze(2) + s["lens"].view(B, 1)
    return {"sel": sel, "lens": lens.expand(B, H).int()}


def _plain_decode(s):
    c = s["case"]
    B, H, G, D, bs, k = c["B"], c["Hkv"], c["G"], c["D"], c["bs"], c["k"]
    sel = s["sel"].long().clamp(min=0)
    h = torch.arange(H, device=DEV).view(1, H, 1)

    def rows(x):
        p = s[x + "_pool"][sel, h] if c["layout"] == "bhtd" else s[x + "_pool"].transpose(1, 2)[sel, h]
        return p.reshape(B, H, k * bs, D).float(), s[x + "_scale"][sel, h].reshape(B, H, 1, k * bs)

    kc, ks = rows("k")
    q = s["q"].float().view(B, H, G, D)
    score = (q @ kc.transpose(2, 3)) * ks * (1.0 / math.sqrt(D))
    out = torch.arange(k * bs, device=DEV) >= s["sel_lens"].view(B, H, 1, 1)
    score = score.masked_fill(out, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    vc, vs = rows("v")
    return ((p * vs) @ vc).view(B, H * G, D).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """From the definitions in 64 bits; a plan and a selection hold whole numbers only."""
    if case["op"] in ("plan", "select"):
        return None
    s = prepare(case, seed)
    return _exact_write(case, s) if case["op"] == "write" else _exact_decode(case, s)


def _exact_write(c, s):
    NB, bs, H, D = s["NB"], c["bs"], c["Hkv"], c["D"]
    keep = s["slots"] >= 0
    slots = s["slots"][keep]
    found = {}
    for x in "kv":
        pool = s[x + "_pool"][:NB] if c["layout"] == "bhtd" else s[x + "_pool"][:NB].permute(0, 2, 1, 3)
        codes = pool.permute(0, 2, 1, 3).reshape(NB * bs, H, D).double()  # one row per slot
        scale = s[x + "_scale"][:NB].permute(0, 2, 1).reshape(NB * bs, H).double()
        new = s[x][keep].double()
        step = (new.abs().max(dim=2).values / 127).float().double()  # the scale is kept in 32 bits
        codes[slots] = (new / step[..., None].clamp_min(1e-300)).float().double().round()  # quotients too
        scale[slots] = step
        found[x], found[x + "s"] = codes * scale[..., None], scale
        found[x + "r"] = torch.zeros(s[x].shape, dtype=torch.float64, device=DEV)
        found[x + "r"][keep] = found[x][slots]
    filled = torch.zeros(NB * bs, dtype=torch.bool, device=DEV)
    filled[slots] = True
    filled = filled.view(NB, bs).flip(1).cumsum(1).flip(1) > 0  # tokens up to the newest of a touched block
    touched = filled.any(1)
    keys = found["k"].float().double().view(NB, bs, H, D)
    hi = torch.where(filled[:, :, None, None], keys, -math.inf).amax(1)
    lo = torch.where(filled[:, :, None, None], keys, math.inf).amin(1)
    most = torch.stack([hi.abs(), lo.abs()]).amax(0).amax(-1)
    step = torch.where(touched[:, None], (most / 127).float().double(), 0.0)
    at = step.clamp_min(1e-300)[..., None]
    up = (hi / at).float().double().ceil().clamp(-127, 127)
    down = (lo / at).float().double().floor().clamp(-127, 127)
    both = torch.stack([up, down], dim=2)
    bounds = torch.where((step > 0)[..., None, None], both, 0.0) * step[..., None, None]

    scales = lambda a: a.view(NB, bs, H).permute(0, 2, 1).contiguous()  # noqa: E731
    return {"k": found["kr"], "v": found["vr"], "ks": scales(found["ks"]), "vs": scales(found["vs"]),
            "bounds": bounds, "bscale": step}


def _exact_decode(c, s):
    B, H, G, D, bs, k = c["B"], c["Hkv"], c["G"], c["D"], c["bs"], c["k"]
    out = torch.empty((B, H, G, D), dtype=torch.float64, device=DEV)
    kp, vp = (s[x] if c["layout"] == "bhtd" else s[x].permute(0, 2, 1, 3) for x in ("k_pool", "v_pool"))
    for b in range(B):
        for h in range(H):
            n = int(s["sel_lens"][b, h])
            ids = s["sel"][b, h].long()[: -(-n // bs)]
            keys = (kp[ids, h].double() * s["k_scale"][ids, h].double()[..., None]).reshape(-1, D)[:n]
            vals = (vp[ids, h].double() * s["v_scale"][ids, h].double()[..., None]).reshape(-1, D)[:n]
            q = s["q"].double().view(B, H, G, D)[b, h]
            out[b, h] = torch.softmax(q @ keys.T / math.sqrt(D), dim=-1) @ vals
    return out.view(B, H * G, D)


if __name__ == "__main__":
    for case in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(case, work(case))
