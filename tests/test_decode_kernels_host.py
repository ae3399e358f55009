"""The GPU tests' shapes against the attention kernels that exist, without a GPU."""
import os
import re

from tests import test_gpu_decode_edges as edges

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "commitllm_b200", "csrc", "paged_attn.cu")


def test_every_attention_kernel_has_a_test():
    kernels = int(re.search(r"constexpr int kVariants = (\d+);", open(SOURCE).read()).group(1))
    reached = set()
    for dtype, heads, kv, new, dim in edges.CALLS:
        rows, wide = edges.rows_and_width(dtype, heads, kv, new, dim)
        reached.add(edges.kernel_of(dtype, rows, dim, wide))
    assert reached == set(range(kernels))
