"""Tiles split along the keys (leanstream_amd.decode.PagedAttention), against the formula
in 64 bits with the tolerance of test_gpu_attention.
"""
import pytest

from test_gpu_attention import Problem, log

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,heads,kv_heads,lengths", [
    (128, 7, 1, [(31, 1400)]), (64, 5, 5, [(33, 1700), (2, 900)]), (256, 3, 1, [(101, 900)]), (256, 7, 1, [(31, 800), (2, 300)])])
def test_parts_of_odd_sizes(torch_gpu, dim, heads, kv_heads, lengths, dtype):
    """An odd number of rows (tokens times heads) in every part."""
    log("case:", dim, heads, lengths, dtype)
    p = Problem(torch_gpu, dtype, dim, heads, kv_heads, 16, lengths)
    assert sum(n for n, _ in lengths) * heads % 2
    p.on_gpu().enqueue()
    p.check()
