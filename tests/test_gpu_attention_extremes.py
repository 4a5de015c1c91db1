"""Attention at the ends of the types' ranges (leanstream_amd.decode.PagedAttention): values that are not finite where
some tokens see them, values at fp16's largest, scores near fp32's lowest.
"""
import math

import pytest

from test_gpu_attention import Problem, log

pytestmark = pytest.mark.gpu


def place(p, s, key):
    return int(p.table[s, key // p.page]), key % p.page


@pytest.mark.parametrize("keys", [300, 2300])      # one piece, and split along the keys
@pytest.mark.parametrize("dim,heads,kv_heads,n", [(128, 8, 2, 40), (64, 4, 4, 60), (256, 4, 2, 20), (128, 8, 2, 4)])
@pytest.mark.parametrize("first,second,want", [(math.nan, math.inf, math.nan), (math.inf, -math.inf, math.nan),
                                               (math.inf, math.inf, math.inf), (-math.inf, 1.0, -math.inf)])
def test_what_is_not_finite_adds_up(torch_gpu, dim, heads, kv_heads, n, keys, first, second, want):
    """One value among the keys that every token sees, one that only the last tokens see: a row's result is what
    their sum is. The weights of both are large enough for the type (all scores are alike)."""
    torch = torch_gpu
    log("case:", dim, heads, n, keys, first, second)
    p = Problem(torch, "float16", dim, heads, kv_heads, 16, [(n, keys)], spread=0.0)
    late = keys - 2
    for key, value in ((keys - n - 200, first), (late, second)):
        at, slot = place(p, 0, key)
        p.v[at, :, slot, 5] = value
    p.on_gpu().enqueue()
    torch.cuda.synchronize()
    got = p.out.cpu().float()
    both = list(range(n - 2, n))           # positions keys - 2 and keys - 1
    before = list(range(n - 2))
    sees_both, sees_one = got[both][:, :, 5], got[before][:, :, 5]
    assert bool(sees_both.isnan().all()) if want != want else bool((sees_both == want).all())
    assert bool(sees_one.isnan().all()) if first != first else bool((sees_one == first).all())
    rest = [d for d in range(dim) if d != 5]
    assert got[:, :, rest].isfinite().all()


@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 32, 8), (64, 8, 8), (256, 8, 1)])
@pytest.mark.parametrize("lengths", [[(1, k) for k in range(4, 60, 5)], [(30, 60), (20, 33)], [(1, 5000)], [(40, 3000)]])
def test_values_at_the_largest_fp16(torch_gpu, dim, heads, kv_heads, lengths):
    """A mean of values is no larger than they are, however its weights were rounded. All keys but one are alike, so
    that their weights round the same way."""
    torch = torch_gpu
    log("case:", dim, heads, lengths)
    for seed in (1, 2, 3):
        p = Problem(torch, "float16", dim, heads, kv_heads, 16, lengths, seed=seed)
        g = torch.Generator().manual_seed(seed)
        p.k[:] = torch.randn(dim, generator=g).half()
        for s, (_, keys) in enumerate(lengths):
            at, slot = place(p, s, 0)
            p.k[at, :, slot] += (0.5 * torch.randn(p.k[at, :, slot].shape, generator=g)).half()
        p.v[:] = 65504.0
        p.v[..., ::2] = -65504.0
        p.on_gpu().enqueue()
        p.check()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dim,heads,kv_heads,lengths", [
    (128, 8, 2, [(1, 120), (3, 40)]), (128, 8, 2, [(40, 90)]), (64, 4, 4, [(60, 128)]), (256, 4, 2, [(20, 100), (1, 9)]),
    (128, 8, 2, [(40, 900)])])
def test_scores_beyond_whole_numbers(torch_gpu, dim, heads, kv_heads, lengths, sign, dtype):
    """Scores of 1e10 and more, whose neighbours in fp32 lie further apart than exponentials reach. Every product is
    exact in fp32, and scores differ by 2^-8 of their size: all weight lies on the best visible key, or evenly on those
    that share its score."""
    torch = torch_gpu
    log("case:", dim, heads, lengths, sign, dtype)
    p = Problem(torch, dtype, dim, heads, kv_heads, 16, lengths)
    p.q[:] = 2.0 ** 15
    p.k.zero_()
    g = torch.Generator().manual_seed(6)
    step = {}
    for s, (n, keys) in enumerate(lengths):
        step[s] = torch.randperm(keys, generator=g) % 128
        for key in range(keys):
            at, slot = place(p, s, key)
            p.k[at, :, slot] = sign * 2.0 ** 14 * (1 + float(step[s][key]) / 128)
    p.on_gpu().enqueue()
    torch.cuda.synchronize()
    got, lse = p.out.cpu().double(), p.lse.cpu().double()
    for s, (n, keys) in enumerate(lengths):
        for i in range(n):
            t = p.starts[s] + i
            seen = sign * step[s][: keys - n + i + 1]
            best = (seen == seen.max()).nonzero()[:, 0]
            v = torch.stack([p.v[place(p, s, int(b))[0], :, place(p, s, int(b))[1]] for b in best]).double()
            v = v.repeat_interleave(heads // kv_heads, 1)
            want, size = v.mean(0), v.abs().mean(0)
            assert ((got[t] - want).abs() <= p.u * want.abs() + (p.u + 2.0 ** -12) * size).all(), (s, i)
            z = sign * 2.0 ** 29 * dim * (1 + sign * float(seen.max()) / 128) * p.scale
            assert ((lse[t] - z - math.log(len(best))).abs() <= 2.0 ** -12 + 2.0 ** -20 * abs(z)).all()


@pytest.mark.parametrize("dim,heads,kv_heads,lengths", [
    (128, 8, 2, [(1, 300), (3, 40)]), (64, 4, 4, [(1, 2500)]), (128, 8, 2, [(40, 300)]), (64, 4, 1, [(30, 2500)]),
    (256, 4, 2, [(20, 200), (1, 9)])])
def test_scores_near_the_lowest(torch_gpu, dim, heads, kv_heads, lengths):
    """bf16 reaches scores of -1e31 and below. One dimension of q and k is not zero, its products are exact in fp32 and
    differ by 2^-8 of their size and more: all weight lies on the best visible key, whose value is the result. The
    logarithm of the sum is its score: 2^-20 of its size, as elsewhere."""
    torch = torch_gpu
    log("case:", dim, heads, lengths)
    p = Problem(torch, "bfloat16", dim, heads, kv_heads, 16, lengths)
    p.q.zero_()
    p.q[..., 0] = 2.0 ** 60
    p.k.zero_()
    g = torch.Generator().manual_seed(4)
    size = {}
    for s, (n, keys) in enumerate(lengths):
        j = torch.randperm(keys, generator=g)
        size[s] = (1 + (j % 128) / 128).double() * 2.0 ** (46 + j // 128).double()
        for key in range(keys):
            at, slot = place(p, s, key)
            p.k[at, :, slot, 0] = -float(size[s][key])
    p.on_gpu().enqueue()
    torch.cuda.synchronize()
    got, lse = p.out.cpu(), p.lse.cpu().double()
    for s, (n, keys) in enumerate(lengths):
        for i in range(n):
            p_i, t = keys - n + i, p.starts[s] + i
            best = int(size[s][: p_i + 1].argmin())
            at, slot = place(p, s, best)
            assert torch.equal(got[t], p.v[at, :, slot].repeat_interleave(heads // kv_heads, 0)), (s, i)
            z = -float(size[s][best]) * 2.0 ** 60 * p.scale
            assert ((lse[t] - z).abs() <= 2.0 ** -20 * abs(z)).all()
