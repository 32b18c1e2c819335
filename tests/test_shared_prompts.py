"""The example of shared prompts: its loop keeps every block either held or free, and what a request's new tokens get
is attention over the rows of its blocks, whether they are its own, shared, copied or moved."""
import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


def test_example_imports_without_a_gpu():
    import shared_prompts

    assert callable(shared_prompts.serve)


@pytest.mark.gpu
@pytest.mark.parametrize("block_size,head_dim,group,context,chunk", [(16, 128, 4, 700, 200), (64, 64, 1, 300, 512), (8, 96, 2, 90, 33)])
def test_samples_share_a_prompt(block_size, head_dim, group, context, chunk):
    import shared_prompts

    got = shared_prompts.serve(prompts=3, samples=4, context=context, steps=21, chunk=chunk, kv_heads=2, group=group,
                               head_dim=head_dim, block_size=block_size)
    # within 2e-5 + 1e-4 |out| of the exact one; outputs are means of unit normals, below 4 in size
    assert got["difference"] < 2e-5 + 1e-4 * 4
    assert got["used"] == got["blocks"] < got["unshared"] / 3
