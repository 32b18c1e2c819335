"""Several answers to each of a few prompts from one paged INT8 cache.

Prompts are read in chunks, each is forked into samples that share its blocks, every sample gets one token a step,
some are dropped and replaced by copies of better ones as in a beam search, and at the end the cache is compacted. All
on one stream, without a copy to the host:

    plan     blocks for the step's tokens                                           kvdecode.paged_plan
    write    their K/V rows quantised into the blocks                               kvdecode.paged_write
    prefill  attention of every request's new tokens, a chunk or a single one       kvdecode.paged_prefill
    fork     samples of a prompt, beams that continue others, ended requests        kvdecode.paged_fork
    compact  blocks in use to the lowest ids, so that the pools could shrink        kvdecode.paged_compact

Queries, keys and values are random; a model would compute them. Usage, on a B200 with the library built:

    python examples/shared_prompts.py [--prompts 4] [--samples 8] [--context 3000] [--steps 24]
"""
import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "cuda-operators_b200"))


def serve(prompts=4, samples=8, context=3000, steps=24, chunk=512, kv_heads=8, group=4, head_dim=128, block_size=16,
          seed=0):
    """Runs the loop; returns the largest difference between the steps' outputs and attention over the rows read back
    from the cache, blocks in use before and after compaction, and what the same samples would hold without sharing."""
    import torch

    import kvdecode as kvd

    dev, i32 = "cuda", torch.int32
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    rnd = lambda *shape: torch.randn(shape, device=dev, generator=gen).to(torch.bfloat16)  # noqa: E731
    rows, H, D, bs = prompts * samples, kv_heads, head_dim, block_size
    max_blocks = -(-(context + steps) // bs)
    num_blocks = prompts * max_blocks + rows * (steps // bs + 2)
    k_pool, v_pool = (torch.zeros((num_blocks, H, bs, D), dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros((num_blocks, H, bs), device=dev) for _ in range(2))
    table = torch.full((rows, max_blocks), -1, dtype=i32, device=dev)
    lens = torch.zeros(rows, dtype=i32, device=dev)
    free = torch.arange(num_blocks, dtype=i32, device=dev)
    count = torch.tensor([num_blocks], dtype=i32, device=dev)
    pools = (k_pool, v_pool, ks, vs)
    fork_ws = torch.zeros(kvd.paged_fork_workspace_size(table, free), dtype=torch.uint8, device=dev)
    worst = 0.0

    def step(new_lens):
        """One engine step: new_lens[b] tokens for row b, and their attention."""
        total = sum(new_lens)
        slots = torch.empty(total, dtype=torch.int64, device=dev)
        _, starts = kvd.paged_plan(lens, torch.tensor(new_lens, dtype=i32, device=dev), table, free, count, bs, slots)
        q = rnd(total, H * group, D)
        kvd.paged_write(rnd(total, H, D), rnd(total, H, D), slots, *pools)
        return q, kvd.paged_prefill(q, *pools, table, lens, starts, out_dtype=torch.float32)

    def difference(b, q, out):
        """Between one row's newest outputs and attention over its rows of the cache."""
        n = int(lens[b])
        at = table[b, : -(-n // bs)].long().repeat_interleave(bs)[:n] * bs + torch.arange(n, device=dev) % bs
        k, v = (x.double() for x in kvd.paged_read(at, *pools))
        see = torch.arange(n, device=dev) <= torch.arange(n - len(q), n, device=dev).unsqueeze(1)
        s = torch.einsum("ihd,thd->hit", q.double(), k.repeat_interleave(group, 1)) / D ** 0.5
        p = s.masked_fill(~see, -torch.inf).softmax(-1)
        return float((torch.einsum("hit,thd->ihd", p, v.repeat_interleave(group, 1)) - out).abs().max())

    # the prompts, each in the first row of its samples, a chunk a step
    lengths = torch.randint(max(1, context // 2), context + 1, (prompts,), generator=host).tolist()
    left = list(lengths)
    while any(left):
        new = [0] * rows
        for i in range(prompts):
            new[i * samples] = min(left[i], chunk)
            left[i] -= new[i * samples]
        q, out = step(new)
    last = max(i for i in range(prompts) if new[i * samples])  # its chunk is the last one of the packed rows
    worst = max(worst, difference(last * samples, q[-new[last * samples]:], out[-new[last * samples]:]))

    # the samples, and beam steps: every fourth step the second half of a prompt's samples continue the first half
    first = torch.arange(rows, dtype=i32, device=dev) // samples * samples
    kvd.paged_fork(first, lens, table, free, count, *pools, workspace=fork_ws)
    own = torch.arange(rows, dtype=i32, device=dev)
    beams = first + (own - first) % max(1, samples // 2)
    for i in range(steps):
        q, out = step([1] * rows)
        if i % 4 == 3:
            kvd.paged_fork(beams, lens, table, free, count, *pools, workspace=fork_ws)
    for b in (0, rows - 1):
        # (a fork keeps a continued row's tokens, and this row's last query may not be its new one's)
        if steps % 4:
            worst = max(worst, difference(b, q[b: b + 1], out[b: b + 1]))

    # one sample of each prompt goes on, the cache shrinks
    kvd.paged_fork(torch.where(own == first, own, -1), lens, table, free, count, *pools, workspace=fork_ws)
    before = int(num_blocks - count)
    used = int(kvd.paged_compact(lens, table, free, count, *pools))
    q, out = step([1 if b % samples == 0 else 0 for b in range(rows)])
    worst = max(worst, difference(0, q[:1], out[:1]))
    status = kvd.device_status()
    if status:
        raise RuntimeError(f"device status {status}")
    held = sum(-(-n // bs) for n in lens.tolist())
    if held + int(count) != num_blocks:
        raise RuntimeError(f"{held} blocks held and {int(count)} free of {num_blocks}")
    alone = samples * sum(-(-(n + steps) // bs) for n in lengths)
    return {"difference": worst, "blocks": before, "used": used, "unshared": alone, "pool": num_blocks}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("prompts", 4), ("samples", 8), ("context", 3000), ("steps", 25)):
        ap.add_argument(f"--{name}", type=int, default=value)
    got = serve(**vars(ap.parse_args()))
    print(f"largest difference from attention over the rows read back {got['difference']:.3g}; the samples without "
          f"sharing would hold {got['unshared']} blocks of {got['pool']}; the last ones hold {got['blocks']}, all below {got['used']}")
