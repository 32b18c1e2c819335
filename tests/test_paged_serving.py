"""The serving example: its loop keeps every block either held or free, and with a budget that covers the
caches its output is attention over all of them."""
import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


def test_example_imports_without_a_gpu():
    import paged_serving

    assert callable(paged_serving.serve)


@pytest.mark.gpu
def test_loop_reads_a_part_of_the_caches():
    import paged_serving

    got = paged_serving.serve(steps=25, batch=5, context=2000, budget=8, kv_heads=2, group=4, block_size=16)
    assert got["decoded"] == 25 * 5 - 2 and 0.05 < got["read"] < 0.2


@pytest.mark.gpu
@pytest.mark.parametrize("block_size,head_dim", [(16, 128), (64, 64)])
def test_full_budget_is_full_attention(block_size, head_dim):
    import paged_serving

    got = paged_serving.serve(steps=21, batch=3, context=600, budget=64, kv_heads=2, group=3, head_dim=head_dim,
                              block_size=block_size)
    # two fp32 evaluations, each within 2e-5 + 1e-4 |out| of the exact one; outputs are means of unit normals
    assert got["read"] == 1.0 and got["difference"] < 2 * (2e-5 + 1e-4 * 4)
