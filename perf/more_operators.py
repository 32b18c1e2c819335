"""Cases that measure chunked attention over kvdecode's paged INT8 cache, and the calls that share, copy, free and
move its blocks, against their plain torch forms.

* ``chunk``    causal attention of the new tokens of every request (packed rows, any number a request, single tokens
               among them) over the request's blocks (``kvdecode.paged_prefill``);
* ``cross``    the same rows attending to all states of an encoder that the blocks hold (``causal=False``);
* ``fork``     rows of the block table become copies of other rows: full blocks are shared, a partly filled last block
               is copied, blocks that no row holds any more go back on the free list (``kvdecode.paged_fork``);
* ``compact``  the blocks in use move to the lowest ids, so that the pools can shrink (``kvdecode.paged_compact``).

``own`` chooses the side that ``run`` computes: False, elementary torch operations in 32 bits; True, the library's
calls.
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
        # a step that checks one to five drafted tokens a request: launch latency and few rows
        {"name": "chunk 8 requests, drafted tokens", "op": "chunk", "B": 8, "T": 23, "singles": 2, "S": 4096,
         "fresh": False, "Hkv": 8, "G": 8, "D": 128, "bs": 16, "dtype": "bf16", "layout": "bthd"},
        # one chunk of a prompt that is read piece by piece
        {"name": "chunk 512 of 8192", "op": "chunk", "B": 1, "T": 512, "singles": 0, "S": 8192, "fresh": False,
         "Hkv": 8, "G": 8, "D": 128, "bs": 64, "dtype": "fp16", "layout": "bhtd"},
        # a mixed step: most requests decode one token, some read a stretch of their prompts
        {"name": "chunk 64 requests, 60 decode", "op": "chunk", "B": 64, "T": 2107, "singles": 60, "S": 16384,
         "fresh": False, "Hkv": 8, "G": 8, "D": 128, "bs": 16, "dtype": "bf16", "layout": "bhtd"},
        # new prompts of odd lengths with one head per KV head, 32-bit rows
        {"name": "chunk 5 whole prompts mha fp32", "op": "chunk", "B": 5, "T": 7003, "singles": 0, "S": 4096,
         "fresh": True, "Hkv": 32, "G": 1, "D": 128, "bs": 16, "dtype": "fp32", "layout": "bhtd"},
        # the last chunk of a long prompt: the matrix products are all of it
        {"name": "chunk 4096 of 32768", "op": "chunk", "B": 1, "T": 4096, "singles": 0, "S": 32768, "fresh": False,
         "Hkv": 8, "G": 8, "D": 128, "bs": 128, "dtype": "bf16", "layout": "bhtd"},
        # decoder steps over an encoder's states, a token a request
        {"name": "cross 64 tokens of 1500 states", "op": "cross", "B": 64, "T": 64, "singles": 64, "S": 1500,
         "fresh": False, "Hkv": 16, "G": 1, "D": 64, "bs": 16, "dtype": "fp16", "layout": "bthd"},
        # decoder rows of a batch of transcripts over their encoders' states
        {"name": "cross 5000 tokens of 1500 states", "op": "cross", "B": 17, "T": 5000, "singles": 1, "S": 1500,
         "fresh": False, "Hkv": 16, "G": 1, "D": 64, "bs": 64, "dtype": "bf16", "layout": "bhtd"},
        # a beam search step of a few requests: launch latency
        {"name": "fork 8 requests of 4 beams", "op": "fork", "B": 32, "group": 4, "how": "beams", "S": 700, "bs": 16,
         "Hkv": 8, "D": 128, "spare": 100, "bounds": False, "layout": "bthd"},
        # prompts that were read once, and eight answers to be sampled from each; the pool runs short, so the last
        # copies are refused
        {"name": "fork 32 prompts into 256", "op": "fork", "B": 256, "group": 8, "how": "prompts", "S": 4096, "bs": 64,
         "Hkv": 8, "D": 128, "spare": 200, "bounds": True, "layout": "bhtd"},
        # a beam search step of many requests, some of which have ended
        {"name": "fork 512 requests of 4 beams", "op": "fork", "B": 2048, "group": 4, "how": "beams", "S": 2048,
         "bs": 16, "Hkv": 4, "D": 128, "spare": 200, "bounds": False, "layout": "bhtd"},
        # a small pool after a few requests have ended
        {"name": "compact 16 requests", "op": "compact", "B": 16, "NB": 2048, "fill": 0.3, "bs": 16, "Hkv": 8, "D": 128,
         "bounds": True, "layout": "bthd"},
        # a large pool that is to shrink to the half that is in use
        {"name": "compact 128 requests", "op": "compact", "B": 128, "NB": 8192, "fill": 0.5, "bs": 64, "Hkv": 8,
         "D": 128, "bounds": False, "layout": "bhtd"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


MOST_PAIRS = 64 * 4096 * 30720 * 128  # heads x rows x tokens x dims of the largest listed case
MOST_POOL = 8192 * 64 * 8 * 128       # codes of the largest listed pool


def draw(rng):
    op = rng.choice(["chunk", "chunk", "cross", "fork", "compact"])
    c = {"op": op, "bs": rng.choice([8, 16, 32, 64, 128]), "layout": rng.choice(["bhtd", "bthd"])}
    if op in ("chunk", "cross"):
        c["dtype"] = rng.choice(list(TYPES))
        c["Hkv"] = rng.choice([1, 2, 4, 8, 16, 32])
        c["G"] = rng.choice([1, 1, 2, 3, 4, 8, 16]) if c["Hkv"] < 16 else 1
        c["D"] = rng.choice([64, 128, 128])
        c["S"] = _log(rng, 1, 32768) if op == "chunk" else _log(rng, 1, 4096)
        c["fresh"] = op == "chunk" and rng.random() < 0.3
        heads = c["Hkv"] * c["G"] * c["D"]
        half = 2 if c["dtype"] != "fp32" else 8  # 32-bit rows cost more of the card
        rows = max(1, MOST_PAIRS // half // (heads * max(64, c["S"])))
        c["B"] = _log(rng, 1, max(1, min(128, rows, MOST_POOL // (c["Hkv"] * c["D"] * (c["S"] + c["bs"])))))
        most = max(c["B"], min(16384, rows, c["B"] * c["S"] if op == "chunk" else 1 << 30))
        c["T"] = _log(rng, c["B"], most)
        c["singles"] = min(c["B"], rng.choice([0, 0, c["B"] // 2, c["B"] - 1, c["B"]]))
        if c["singles"] == c["B"]:
            c["T"] = c["B"]
        return c
    c["Hkv"] = rng.choice([1, 2, 4, 8])
    c["D"] = rng.choice([64, 128, 128, 256])
    c["bounds"] = rng.random() < 0.5
    block = c["bs"] * c["Hkv"] * c["D"]
    if op == "fork":
        c["group"] = rng.choice([2, 3, 4, 8])
        c["how"] = rng.choice(["beams", "prompts"])
        c["S"] = _log(rng, 1, 8192)
        groups = _log(rng, 1, max(1, min(2048 // c["group"], MOST_POOL // block // (c["S"] // c["bs"] + c["group"] + 2))))
        c["B"] = groups * c["group"]
        c["spare"] = _log(rng, 1, 4096)
        c["spare"] = min(c["spare"], max(1, MOST_POOL // block // 4))
        return c
    c["NB"] = _log(rng, 8, max(8, MOST_POOL // block))
    c["fill"] = rng.choice([0.1, 0.3, 0.5, 0.7, 0.95])
    c["B"] = _log(rng, 1, 256)
    return c


# What a case's requests look like follows from the case alone, so that the work of a case is one number.
def _rng(c):
    return np.random.default_rng([c["B"], c.get("T", 0), c.get("S", 0), c.get("NB", 0), c["bs"]])


def _split(rng, total, parts):
    """`total` as `parts` random whole numbers of at least 1."""
    if parts <= 0:
        return np.zeros(0, np.int64)
    total = max(total, parts)
    cuts = np.sort(rng.choice(np.arange(1, total), size=parts - 1, replace=False)) if parts > 1 else np.zeros(0, np.int64)
    return np.diff(np.concatenate([[0], cuts, [total]])).astype(np.int64)


def _requests(c):
    """(new tokens, tokens held with them) of every request of an attention case."""
    rng, B, S = _rng(c), c["B"], c["S"]
    n = np.ones(B, np.int64)
    who = rng.permutation(B)
    rest = who[c["singles"]:]
    n[rest] = _split(rng, c["T"] - c["singles"], len(rest))
    if c["op"] == "cross":
        return n, rng.integers(max(1, S * 3 // 4), S + 1, size=B)
    held = n if c["fresh"] else np.maximum(n, rng.integers(max(1, S // 2), S + 1, size=B))
    if len(rest) == B == 1:
        held = np.maximum(n, S)
    return n, held


def _forks(c):
    """(parents, lengths) of a fork case."""
    rng, B, g, S = _rng(c), c["B"], c["group"], c["S"]
    first = np.arange(B) // g * g
    if c["how"] == "prompts":  # the first row of each group holds a prompt, the others nothing yet
        lens = np.where(np.arange(B) == first, rng.integers(max(1, S // 2), S + 1, size=B), 0)
        return first, lens
    lens = np.repeat(rng.integers(max(1, S // 2), S + 1, size=B // g), g)
    parents = first + rng.integers(0, g, size=B)
    if B >= 16:
        ends = rng.integers(0, B // g, size=max(1, B // g // 16))
        for e in ends:  # requests that have found their answers
            parents[e * g:(e + 1) * g] = -1
    return parents, lens


def work(case):
    c = case
    if c["op"] in ("chunk", "cross"):
        n, held = _requests(c)
        e = TYPES[c["dtype"]].itemsize
        rows = int(n.sum()) * c["Hkv"] * c["G"] * c["D"]
        pairs = int((n * held - (n * (n - 1) // 2 if c["op"] == "chunk" else 0)).sum())
        return {"bytes": int(held.sum()) * c["Hkv"] * (2 * c["D"] + 8) + 2 * rows * e,
                "flops": 4 * pairs * c["Hkv"] * c["G"] * c["D"]}
    token = c["Hkv"] * (2 * c["D"] + 8)
    bound = c["Hkv"] * (2 * c["D"] + 4) if c["bounds"] else 0
    if c["op"] == "fork":
        parents, lens = _forks(c)
        live = parents >= 0
        heirs = np.unique(parents[live])
        copies = [p for p in parents[live]]
        for p in heirs:
            copies.remove(p)
        tail = sum(int(lens[p]) % c["bs"] for p in copies)
        blocks = sum(1 for p in copies if lens[p] % c["bs"])
        entries = int((-(-lens // c["bs"])).sum()) + int((-(-lens[parents[live]] // c["bs"])).sum())
        return {"bytes": 2 * (tail * token + blocks * bound) + 4 * entries + 12 * c["B"], "flops": 0}
    used = int(c["NB"] * c["fill"])
    moves = used - int(used * c["fill"])  # blocks of random ids that lie above the used ones' number
    return {"bytes": 2 * moves * (c["bs"] * token + bound) + 8 * used + 8 * (c["NB"] - used), "flops": 0}


# ----------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"chunk": _prepare_attend, "cross": _prepare_attend, "fork": _prepare_fork, "compact": _prepare_compact}[c["op"]](c, gen, rng)
    s["case"] = c
    if own:
        s["kvd"] = _kvd()
    return s


def _dev(a, t=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, t)


def _pools(c, NB, gen):
    H, D, bs = c["Hkv"], c["D"], c["bs"]
    shape = (NB, H, bs, D) if c["layout"] == "bhtd" else (NB, bs, H, D)
    s = {}
    for x in "kv":
        s[x + "_pool"] = torch.randint(-127, 128, shape, dtype=torch.int8, device=DEV, generator=gen)
        s[x + "_scale"] = torch.rand((NB, H, bs), device=DEV, generator=gen) * 0.02 + 0.005
    return s


def _tables(lens, bs, MB, ids):
    """Table rows of their own blocks for every length, and the ids that are left."""
    table, at = np.full((len(lens), MB), -1, np.int32), 0
    for b, n in enumerate(-(-lens // bs)):
        table[b, :n] = ids[at: at + n]
        at += n
    return table, ids[at:]


def _prepare_attend(c, gen, rng):
    n, held = _requests(c)
    bs, B = c["bs"], c["B"]
    MB = int(-(-held.max() // bs)) + 1
    NB = int((-(-held // bs)).sum()) + 5
    table, _ = _tables(held, bs, MB, rng.permutation(NB))
    s = _pools(c, NB, gen)
    s |= {"n": n.tolist(), "held": held.tolist(), "table": _dev(table), "lens": _dev(held),
          "starts": _dev(np.concatenate([[0], np.cumsum(n)]))}
    rows = torch.randn((int(n.sum()), c["Hkv"] * c["G"], c["D"]), device=DEV, generator=gen)
    s["q"] = rows.to(TYPES[c["dtype"]])
    s["out"] = torch.empty_like(s["q"])
    if own:  # scratch that a serving loop keeps
        size = _kvd().paged_prefill_workspace_size(s["q"], s["k_pool"], s["table"], c["layout"])
        s["ws"] = torch.empty(size, dtype=torch.uint8, device=DEV)
    return s


def _prepare_fork(c, gen, rng):
    parents, lens = _forks(c)
    B, bs, g = c["B"], c["bs"], c["group"]
    held = -(-lens // bs)
    MB = int(held.max()) + 2
    if c["how"] == "beams":  # the rows of a group share all but their last blocks
        own_blocks = np.where(lens % bs > 0, 1, 0)
        shared = held - own_blocks
        NB = int(shared[::g].sum() + own_blocks.sum()) + c["spare"] + 9
        ids, at = rng.permutation(NB), 0
        table = np.full((B, MB), -1, np.int32)
        for b in range(0, B, g):
            table[b:b + g, : shared[b]] = ids[at: at + shared[b]]
            at += shared[b]
            if own_blocks[b]:
                table[np.arange(b, b + g), shared[b]] = ids[at: at + g]
                at += g
        left = ids[at:]
    else:
        NB = int(held.sum()) + c["spare"] + 9
        table, left = _tables(lens, bs, MB, rng.permutation(NB))
    free = np.full(NB, -1, np.int32)
    free[: c["spare"]] = left[: c["spare"]]
    s = _pools(c, NB, gen)
    s |= {"parents": _dev(parents), "lens": _dev(lens), "table": _dev(table), "free": _dev(free),
          "count": _dev(np.array([c["spare"]]))}
    s |= {"table_out": torch.full_like(s["table"], -1), "lens_out": torch.empty_like(s["lens"]),
          "count_out": torch.empty_like(s["count"])}
    return _more(c, s, NB, gen, "paged_fork_workspace_size")


def _prepare_compact(c, gen, rng):
    B, bs, NB = c["B"], c["bs"], c["NB"]
    used = int(NB * c["fill"])
    B = min(B, used) or 1
    held = _split(_rng(c), used, B) if used else np.zeros(B, np.int64)
    lens = held * bs - np.where(held > 0, rng.integers(0, bs, size=B), 0)
    MB = int(held.max()) + 1
    table, left = _tables(lens, bs, MB, rng.permutation(NB))
    free = np.full(NB, -1, np.int32)
    free[: len(left)] = left
    s = _pools(c, NB, gen)
    s |= {"lens": _dev(lens), "table": _dev(table), "free": _dev(free), "count": _dev(np.array([len(left)]))}
    s |= {"table_out": torch.full_like(s["table"], -1), "free_out": torch.full_like(s["free"], -1),
          "used": torch.empty_like(s["count"])}
    return _more(c, s, NB, gen, "paged_compact_workspace_size")


def _more(c, s, NB, gen, size):
    """Key bounds, and the scratch that a serving loop keeps."""
    s["bounds"] = s["bound_scale"] = None
    if c["bounds"]:
        s["bounds"] = torch.randint(-127, 128, (NB, c["Hkv"], 2, c["D"]), dtype=torch.int8, device=DEV, generator=gen)
        s["bound_scale"] = torch.rand((NB, c["Hkv"]), device=DEV, generator=gen)
    if own:
        s["ws"] = torch.zeros(getattr(_kvd(), size)(s["table"], s["free"]), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------------------------------------- runs
def run(state):
    op = state["case"]["op"]
    if own:
        return {"chunk": _own_attend, "cross": _own_attend, "fork": _own_fork, "compact": _own_compact}[op](state)
    return {"chunk": _plain_attend, "cross": _plain_attend, "fork": _plain_fork, "compact": _plain_compact}[op](state)


def _own_attend(s):
    c = s["case"]
    return s["kvd"].paged_prefill(s["q"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["table"], s["lens"],
                                  s["starts"], out=s["out"], layout=c["layout"], causal=c["op"] == "chunk",
                                  workspace=s["ws"])


def _own_fork(s):
    s["kvd"].paged_fork(s["parents"], s["lens"], s["table"], s["free"], s["count"], s["k_pool"], s["v_pool"],
                        s["k_scale"], s["v_scale"], bounds=s["bounds"], bound_scale=s["bound_scale"],
                        layout=s["case"]["layout"], seq_lens_out=s["lens_out"], block_table_out=s["table_out"],
                        free_count_out=s["count_out"], workspace=s["ws"])
    return _forked(s)


def _own_compact(s):
    s["kvd"].paged_compact(s["lens"], s["table"], s["free"], s["count"], s["k_pool"], s["v_pool"], s["k_scale"],
                           s["v_scale"], bounds=s["bounds"], bound_scale=s["bound_scale"], layout=s["case"]["layout"],
                           block_table_out=s["table_out"], free_blocks_out=s["free_out"], used=s["used"],
                           workspace=s["ws"])
    return _compacted(s)


def _moved(s):
    """The pools, whose codes move as they are: whole numbers that have to be equal."""
    return {x: s[x] for x in ("k_pool", "v_pool", "k_scale", "v_scale", "bounds", "bound_scale")}


def _forked(s):
    return {"table": s["table_out"], "lens": s["lens_out"], "free": s["free"], "count": s["count_out"], **_moved(s)}


def _compacted(s):
    return {"table": s["table_out"], "free": s["free_out"], "count": s["count"], "used": s["used"], **_moved(s)}


SCORES = 1 << 28  # scores that the plain form holds at a time


def _plain_attend(s):
    c, n, held = s["case"], s["n"], s["held"]
    B, H, G, D, bs = c["B"], c["Hkv"], c["G"], c["D"], c["bs"]
    if B * max(n) * H * G * max(held) <= SCORES:  # all requests at once, filled up to the longest
        i = torch.arange(max(n), device=DEV)
        first, stop = s["starts"][:-1].long().unsqueeze(1), s["starts"][1:].long().unsqueeze(1)
        at = first + i
        rows = s["q"][at.clamp(max=s["q"].shape[0] - 1)]
        out = _attend(s, rows, s["table"], s["lens"], stop - first, slice(0, H), max(held))
        s["out"][at[at < stop]] = out[at < stop].to(s["q"].dtype)
        return s["out"]
    t = 0
    for b in range(B):
        step = max(1, SCORES // (n[b] * G * held[b]))
        for h in range(0, H, step):
            heads = slice(h, min(H, h + step))
            rows = s["q"][t: t + n[b], heads.start * G: heads.stop * G].unsqueeze(0)
            out = _attend(s, rows, s["table"][b: b + 1], s["lens"][b: b + 1],
                          torch.full((1, 1), n[b], device=DEV), heads, held[b])
            s["out"][t: t + n[b], heads.start * G: heads.stop * G] = out[0].to(s["q"].dtype)
        t += n[b]
    return s["out"]


def _attend(s, q, table, lens, n, heads, most):
    """Attention of rows [b, i, heads, D] over the first `most` tokens of the table's blocks, in 32 bits."""
    c = s["case"]
    G, D, bs = c["G"], c["D"], c["bs"]
    b, rows, H = q.shape[0], q.shape[1], heads.stop - heads.start
    ids = table[:, : -(-most // bs)].long().clamp(min=0)

    def gather(x):
        p = s[x + "_pool"][:, heads] if c["layout"] == "bhtd" else s[x + "_pool"].transpose(1, 2)[:, heads]
        codes = p[ids].transpose(1, 2).reshape(b, H, -1, D).float()
        return codes, s[x + "_scale"][:, heads][ids].transpose(1, 2).reshape(b, H, 1, -1)

    codes, scale = gather("k")
    x = q.float().view(b, rows, H, G, D).permute(0, 2, 1, 3, 4).reshape(b, H, rows * G, D)
    score = (x @ codes.transpose(2, 3)) * scale * (1.0 / math.sqrt(D))
    token = torch.arange(score.shape[-1], device=DEV)
    see = lens.long().view(b, 1).expand(b, rows)
    if c["op"] == "chunk":
        see = see - n + torch.arange(rows, device=DEV) + 1
    see = see.repeat_interleave(G, dim=1).view(b, 1, rows * G, 1)
    score = score.masked_fill(token >= see, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    codes, scale = gather("v")
    out = (e * scale) @ codes / torch.where(total == 0, 1.0, total)
    return out.view(b, H, rows, G, D).permute(0, 2, 1, 3, 4).reshape(b, rows, H * G, D)


def _marks(NB, ids, which):
    """Truth values of the pool's blocks: those of `ids` where `which` is true."""
    there = torch.zeros(NB + 1, dtype=torch.bool, device=DEV)
    there[torch.where(which, ids, NB)] = True
    return there[:NB]


def _copy_tokens(s, src, dst, count):
    """The first `count` tokens of blocks `src`, and their bounds, into blocks `dst`."""
    c, bs = s["case"], s["case"]["bs"]
    keep = torch.arange(bs, device=DEV) < count.unsqueeze(1)
    shape = (-1, 1, bs, 1) if c["layout"] == "bhtd" else (-1, bs, 1, 1)
    for x in "kv":
        pool, scale = s[x + "_pool"], s[x + "_scale"]
        pool[dst] = torch.where(keep.view(shape), pool[src], pool[dst])
        scale[dst] = torch.where(keep.unsqueeze(1), scale[src], scale[dst])
    if s["bounds"] is not None:
        s["bounds"][dst] = s["bounds"][src]
        s["bound_scale"][dst] = s["bound_scale"][src]


def _plain_fork(s):
    c = s["case"]
    bs, B = c["bs"], c["B"]
    parents, lens, table, free = s["parents"].long(), s["lens"].long(), s["table"].long(), s["free"]
    fc, NB, MB = s["count"].long(), free.numel(), table.shape[1]
    live = (parents >= 0) & (parents < B)
    p = parents.clamp(0, B - 1)
    b = torch.arange(B, device=DEV)
    rank = torch.where(live, torch.where(p == b, -1, b), B)  # a parent itself comes first, then its lowest row
    heir = torch.full((B,), B, device=DEV).scatter_reduce_(0, p, rank, "amin")
    held = (lens + bs - 1) // bs
    inside = torch.arange(MB, device=DEV) < held.unsqueeze(1)
    kept = _marks(NB, table, inside & (heir < B).unsqueeze(1))
    freed = _marks(NB, table, inside & (heir == B).unsqueeze(1)) & ~kept
    at = fc + freed.cumsum(0) - 1  # freed blocks go on the stack in the order of their ids
    stack = torch.cat([free, free[:1]])
    stack[torch.where(freed, at, NB)] = torch.arange(NB, device=DEV, dtype=torch.int32)
    stack = stack[:NB]
    total = fc + freed.sum()
    tail = lens[p] % bs
    copy = live & (tail > 0) & (rank != heir[p])
    k = copy.cumsum(0) - 1
    served = copy & (k < total)
    ok = live & (served | ~copy)
    lens_out = torch.where(ok, lens[p], 0)
    fresh = stack[(total - 1 - k).clamp(0, NB - 1)]
    last = (held[p] - 1).clamp(min=0)
    j = torch.arange(MB, device=DEV)
    rows = torch.where(served.unsqueeze(1) & (j == last.unsqueeze(1)), fresh.unsqueeze(1), table[p].int())
    s["table_out"].copy_(torch.where(ok.unsqueeze(1) & (j < held[p].unsqueeze(1)), rows, s["table_out"]))
    s["lens_out"].copy_(lens_out)
    s["count_out"].copy_(total - served.sum())
    free.copy_(stack)
    at = served.nonzero().squeeze(1)
    _copy_tokens(s, table[p[at], last[at]], fresh[at].long(), tail[at])
    return _forked(s)


def _plain_compact(s):
    c, table, free = s["case"], s["table"].long(), s["free"].long()
    bs, NB, MB = c["bs"], free.numel(), table.shape[1]
    held = (s["lens"].long() + bs - 1) // bs
    inside = torch.arange(MB, device=DEV) < held.unsqueeze(1)
    used = _marks(NB, table, inside)
    unused = _marks(NB, free.clamp(min=0), torch.arange(NB, device=DEV) < s["count"]) & ~used
    n = used.sum()
    low = (used | unused).cumsum(0) <= n  # the lowest ids that these requests may have
    src, dst = (used & ~low).nonzero().squeeze(1), (unused & low).nonzero().squeeze(1)
    to = torch.arange(NB + 1, device=DEV)
    to[src] = dst
    s["table_out"].copy_(torch.where(inside, to[table.clamp(0, NB)].int(), s["table_out"]))
    rest = ((used | unused) & ~low).nonzero().squeeze(1).flip(0)  # the lowest id on top
    s["free_out"][: rest.numel()] = rest.int()
    s["count"].fill_(rest.numel())
    now = low & (used | unused)
    s["used"].copy_(torch.where(now, to[:NB] + 1, 0).amax())
    _copy_tokens(s, src, dst, torch.full_like(src, bs))
    return _compacted(s)


# ------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """From the definition in 64 bits; forks and moves only carry what is there to other places."""
    if case["op"] in ("fork", "compact"):
        return None
    c, s = case, prepare(case, seed)
    H, G, D, bs = c["Hkv"], c["G"], c["D"], c["bs"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    kp, vp = (s[x] if c["layout"] == "bhtd" else s[x].permute(0, 2, 1, 3) for x in ("k_pool", "v_pool"))
    t = 0
    for b, (n, held) in enumerate(zip(s["n"], s["held"])):
        ids = s["table"][b, : -(-held // bs)].long()
        for h in range(H):
            keys = (kp[ids, h].double() * s["k_scale"][ids, h].double()[..., None]).reshape(-1, D)[:held]
            vals = (vp[ids, h].double() * s["v_scale"][ids, h].double()[..., None]).reshape(-1, D)[:held]
            for i in range(0, n, 512):
                m = min(512, n - i)
                q = s["q"][t + i: t + i + m, h * G: (h + 1) * G].double()
                score = torch.einsum("igd,td->igt", q, keys) / math.sqrt(D)
                if c["op"] == "chunk":
                    pos = held - n + i + torch.arange(m, device=DEV)
                    score.masked_fill_(torch.arange(held, device=DEV) > pos.view(m, 1, 1), -math.inf)
                out[t + i: t + i + m, h * G: (h + 1) * G] = torch.softmax(score, dim=-1) @ vals
        t += n
    return out


if __name__ == "__main__":
    for case in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(case, work(case))
