"""What a token does not see leaves its result alone to the last bit (leanstream_amd.decode.PagedAttention): outputs
with other keys and values in such slots are compared for equality, so there is no tolerance.
"""
import math

import pytest

from test_gpu_attention import Problem, log

pytestmark = pytest.mark.gpu


def outputs(torch, p):
    p.on_gpu().enqueue()
    torch.cuda.synchronize()
    return p.out.clone(), p.lse.clone()


def change(torch, p, s, key, kind):
    """Another key and value at position `key` of sequence s."""
    at, slot = int(p.table[s, key // p.page]), key % p.page
    g = torch.Generator().manual_seed(99)
    shape = p.k[at, :, slot].shape
    if kind == "large":      # scores far above all others, for some rows
        p.k[at, :, slot] = (25 * torch.randn(shape, generator=g)).to(p.dtype)
        p.v[at, :, slot] = (100 * torch.randn(shape, generator=g)).to(p.dtype)
    else:                    # a value that is not finite: in every third dimension
        p.k[at, :, slot] = (3 * torch.randn(shape, generator=g)).to(p.dtype)
        p.v[at, :, slot, ::3] = kind


# (dim, heads, kv_heads, new tokens, keys): tiles, tiles split along the keys, few rows, few rows split
TILES = [(128, 8, 2, 40, 300), (64, 4, 4, 150, 300), (256, 4, 2, 20, 300), (128, 8, 2, 40, 3000), (64, 4, 1, 30, 2500)]
ROWS = [(128, 8, 2, 4, 300), (64, 8, 1, 2, 300), (256, 4, 2, 5, 300), (128, 8, 2, 3, 6000)]


def unseen_slots(torch_gpu, shape, dtype, kind):
    torch = torch_gpu
    dim, heads, kv_heads, n, keys = shape
    for window, sinks in ((0, 0), (37, 3)):
        for seed in (1, 2):
            p = Problem(torch, dtype, dim, heads, kv_heads, 16, [(n, keys)], window=window, sinks=sinks, seed=seed)
            want, want_lse = outputs(torch, p)
            # later tokens' keys, and with a window one that only the first token still sees
            spots = [(keys - 1, range(n - 1)), (keys - n + n // 2, range(n // 2))]
            if window:
                spots.append((keys - n - window + 1, range(1, n)))
            for key, blind in spots:
                log("case:", shape, dtype, kind, window, seed, key)
                k, v = p.k.clone(), p.v.clone()
                change(torch, p, 0, key, kind)
                got, got_lse = outputs(torch, p)
                rows = list(blind)
                assert torch.equal(got[rows], want[rows])
                assert torch.equal(got_lse[rows], want_lse[rows])
                assert not torch.equal(got, want)
                p.k, p.v = k, v


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("kind", ["large", math.inf, math.nan])
@pytest.mark.parametrize("shape", TILES)
def test_tiles_of_rows(torch_gpu, shape, dtype, kind):
    unseen_slots(torch_gpu, shape, dtype, kind)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("kind", ["large", math.inf, math.nan])
@pytest.mark.parametrize("shape", ROWS)
def test_few_rows(torch_gpu, shape, dtype, kind):
    unseen_slots(torch_gpu, shape, dtype, kind)
