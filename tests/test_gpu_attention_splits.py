"""Tiles split along the keys and many sequences in one call (leanstream_amd.decode.PagedAttention), against the formula
in 64 bits with the tolerance of test_gpu_attention.
"""
import random

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


def many(count, seed, chunks):
    """`count` sequences: idle ones, single tokens and a few tokens, and the chunks {sequence: (new tokens, keys)}."""
    r = random.Random(seed)
    out = []
    for s in range(count):
        keys = r.randint(1, 150)
        out.append(chunks.get(s) or r.choice([(0, 0), (0, keys), (1, keys), (1, keys), (min(3, keys), keys)]))
    return out


SPLIT, WHOLE = (40, 1500), (33, 90)


@pytest.mark.parametrize("dim,heads,kv_heads,window,sinks", [(128, 4, 2, 0, 0), (64, 4, 4, 0, 0), (256, 2, 1, 0, 0),
                                                             (128, 4, 2, 600, 5)])
@pytest.mark.parametrize("count,chunks", [
    (65, {64: SPLIT}), (65, {63: SPLIT, 64: (17, 900)}), (128, {0: WHOLE, 63: SPLIT, 64: WHOLE, 127: SPLIT}),
    (130, {62: WHOLE, 64: SPLIT, 65: SPLIT, 128: SPLIT, 129: WHOLE}), (200, {}), (200, {150: SPLIT}),
    (330, {5: WHOLE, 64: WHOLE, 191: SPLIT, 192: SPLIT, 329: SPLIT})])
def test_more_than_64_sequences(torch_gpu, dim, heads, kv_heads, window, sinks, count, chunks):
    """The kernels look through the sequences 64 at a time: for the rows' tiles, their splits and the join."""
    log("case:", dim, window, count, chunks)
    p = Problem(torch_gpu, "float16", dim, heads, kv_heads, 16, many(count, count + dim, chunks), window=window, sinks=sinks)
    p.on_gpu().enqueue()
    p.check()
