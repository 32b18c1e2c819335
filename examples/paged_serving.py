"""A serving loop over a paged INT8 cache that reads a part of each long context.

Requests arrive with prompts, get one token a step and leave. Every step runs, on one stream and without
a copy to the host:

    plan    blocks for the step's tokens, and the blocks of ended requests back   kvdecode.paged_plan
    write   their K/V rows quantised into the blocks, with the blocks' key bounds kvdecode.paged_write
    select  the blocks whose bounds promise the largest products, per KV head      kvdecode.block_select
    decode  attention of each request's new token over the selected blocks        kvdecode.sparse_decode

Queries, keys and values are random (stretches of a prompt have keys along the direction of the request's
queries, so that some blocks matter more than others); a model would compute them. Usage, on a B200 with the library built:

    python examples/paged_serving.py [--steps 40] [--batch 16] [--context 8192] [--budget 32]
"""
import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "cuda-operators_b200"))


def serve(steps=40, batch=16, context=8192, budget=32, kv_heads=8, group=4, head_dim=128, block_size=64, seed=0):
    """Runs the loop; returns tokens decoded, blocks in use at the end, the largest difference between the last
    step's output and attention over the whole caches, and the share of the caches that the last step read."""
    import torch

    import kvdecode as kvd

    dev, i32 = "cuda", torch.int32
    gen = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *shape: torch.randn(shape, device=dev, generator=gen).to(torch.bfloat16)  # noqa: E731
    H, D = kv_heads, head_dim
    max_blocks = -(-(context + steps) // block_size)
    num_blocks = batch * max_blocks
    k_pool, v_pool = (torch.zeros((num_blocks, H, block_size, D), dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros((num_blocks, H, block_size), device=dev) for _ in range(2))
    bounds = torch.zeros((num_blocks, H, 2, D), dtype=torch.int8, device=dev)
    bound_scale = torch.zeros((num_blocks, H), device=dev)
    table = torch.full((batch, max_blocks), -1, dtype=i32, device=dev)
    lens = torch.zeros(batch, dtype=i32, device=dev)
    free = torch.arange(num_blocks, dtype=i32, device=dev)
    count = torch.tensor([num_blocks], dtype=i32, device=dev)
    topic = rnd(batch, H, D)  # what a request's queries look for

    def step(new_lens, q=None):
        """One engine step: new_lens[b] tokens for request b (-1: it has ended)."""
        n = [max(0, x) for x in new_lens]
        total = sum(n)
        slots = torch.empty(total, dtype=torch.int64, device=dev)
        kvd.paged_plan(lens, torch.tensor(new_lens, dtype=i32, device=dev), table, free, count, block_size, slots)
        if total:
            who = torch.repeat_interleave(torch.arange(batch, device=dev), torch.tensor(n, device=dev))
            hot = torch.arange(total, device=dev) // 200 % 16 == 3  # stretches of a prompt that are to the point
            k = rnd(total, H, D) + topic[who] * hot.view(-1, 1, 1)
            kvd.paged_write(k, rnd(total, H, D), slots, k_pool, v_pool, ks, vs, bounds, bound_scale)
        if q is None:
            return None
        sel, sel_lens = kvd.block_select(q, bounds, bound_scale, table, lens, block_size, budget)
        return kvd.sparse_decode(q, k_pool, v_pool, ks, vs, sel, sel_lens), sel_lens

    host = torch.Generator().manual_seed(seed)
    prompts = torch.randint(context // 2, context, (batch,), generator=host).tolist()
    step(prompts)
    decoded = 0
    for i in range(steps):
        q = rnd(batch, H * group, D) + topic.repeat_interleave(group, dim=1)
        new = [1] * batch
        if i % 10 == 9 and i + 1 < steps:  # a request ends; the next step starts another in its place
            new[i % batch] = -1
        elif i % 10 == 0 and i > 0:
            new[(i - 1) % batch] = context // 2
        out, sel_lens = step(new, q)
        decoded += sum(x > 0 for x in new)
    full = kvd.paged_decode(q, k_pool, v_pool, ks, vs, table, lens)
    status = kvd.device_status()
    if status:
        raise RuntimeError(f"device status {status}")
    held = int(((lens + block_size - 1) // block_size).sum())
    if held + int(count) != num_blocks:
        raise RuntimeError(f"{held} blocks held and {int(count)} free of {num_blocks}")
    return {"decoded": decoded, "blocks": held, "difference": float((out - full).abs().max()),
            "read": float(sel_lens.sum()) / float(lens.sum() * H)}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("steps", 40), ("batch", 16), ("context", 8192), ("budget", 32)):
        ap.add_argument(f"--{name}", type=int, default=value)
    got = serve(**vars(ap.parse_args()))
    print(f"{got['decoded']} tokens decoded, {got['blocks']} blocks held; the last step read {got['read']:.1%} of the "
          f"caches and differs from attention over all of them by at most {got['difference']:.3g}")
