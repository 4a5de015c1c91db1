"""Prompts and many sequences through the cache's append (decode.AppendKV), against the formula in 64 bits. A rotated
value is rounded once: it lies between the roundings, to its type, of the formula's values 2^-21 (|a| + |b|) below and
above. What is copied is equal.
"""
import random

import pytest

from test_gpu_block_ops import append_problem, log

pytestmark = pytest.mark.gpu


def check(torch, dtype, dim, q_heads, kv_heads, page, lengths, rot, interleaved, in_place=False, seed=1):
    from leanstream_amd import decode

    H, K = q_heads, kv_heads
    p = append_problem(torch, dtype, dim, H, K, page, lengths, rot, interleaved, "head", seed)
    k, v, qkv = p["k"].cuda(), p["v"].cuda(), p["qkv"].cuda()
    q, kn, vn = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
    q_out = q if in_place else torch.empty(q.shape, dtype=q.dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    decode.AppendKV(q, kn, vn, p["cos"].cuda() if rot else None, p["sin"].cuda() if rot else None,
                    decode.PagedCache(k, v), p["table"].cuda(), torch.tensor(p["starts"], dtype=torch.int32, device="cuda"),
                    torch.tensor([m for _, m in lengths], dtype=torch.int32, device="cuda"), q_out, interleaved=interleaved,
                    status=status).enqueue()
    torch.cuda.synchronize()
    assert int(status) == 0
    seq = torch.tensor([s for s, (n, _) in enumerate(lengths) for _ in range(n)])
    pos = torch.tensor([m - n + i for n, m in lengths for i in range(n)])
    x = p["qkv"][:, :H + K].double()
    if rot:
        i = torch.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = p["cos"][pos].double()[:, None], p["sin"][pos].double()[:, None]
        y = x.clone()
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size = torch.zeros_like(x)      # dimensions from rot on are copied
        size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
        x = y
        off = 2.0 ** -21 * size
    else:
        off = torch.zeros_like(x)
    low, high = (x - off).to(k.dtype), (x + off).to(k.dtype)
    got = q_out.cpu()
    assert ((low[:, :H] <= got) & (got <= high[:, :H])).all()
    low_k, high_k, want_v = p["k"].clone(), p["k"].clone(), p["v"].clone()
    at, slot = p["table"][seq, pos // page].long(), pos % page
    low_k[at, :, slot], high_k[at, :, slot] = low[:, H:], high[:, H:]
    want_v[at, :, slot] = p["qkv"][:, H + K:]
    got = k.cpu()
    assert ((low_k <= got) & (got <= high_k)).all()
    assert torch.equal(v.cpu(), want_v)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,q_heads,kv_heads,page,rot,lengths", [
    (128, 8, 2, 16, 128, [(300, 500), (1, 7)]), (128, 64, 8, 64, 64, [(257, 257)]), (64, 6, 3, 1, 32, [(400, 450), (0, 9)]),
    (256, 16, 4, 64, 256, [(258, 1000)]), (80, 3, 1, 8, 20, [(260, 300)]), (10, 3, 1, 32, 6, [(1000, 1010), (2, 2)]),
    (128, 8, 2, 16, 0, [(511, 600)])])
def test_more_than_256_tokens(torch_gpu, dim, q_heads, kv_heads, page, rot, lengths, interleaved, in_place):
    """Where a token's threads are fewer: in 16-byte words and dimension by dimension."""
    log("case:", dim, q_heads, rot, lengths, interleaved, in_place)
    check(torch_gpu, "float16", dim, q_heads, kv_heads, page, lengths, rot, interleaved, in_place)


@pytest.mark.parametrize("tokens", [256, 257])
def test_either_side_of_the_rule(torch_gpu, tokens):
    log("case:", tokens)
    check(torch_gpu, "bfloat16", 128, 32, 8, 16, [(tokens - 1, 700), (1, 3)], 128, False)


@pytest.mark.parametrize("dim,rot", [(64, 64), (10, 4)])
@pytest.mark.parametrize("count", [64, 65, 128, 129, 130, 330])
def test_many_sequences(torch_gpu, count, dim, rot):
    """A token's sequence is looked for 64 sequences at a time. Idle sequences, single tokens, and chunks whose first or
    last one is a multiple of 64."""
    r = random.Random(count)
    for most in (1, 9):
        lengths = []
        for s in range(count):
            n = r.choice([0, 1, 1, r.randint(0, most)])
            lengths.append((n, n + r.randint(0, 60)))
        for s in (0, 63, 64, 127, 128, count - 1):
            if s < count:
                lengths[s] = (most, most + s)
        log("case:", count, dim, most, sum(n for n, _ in lengths))
        check(torch_gpu, "float16", dim, 3, 2, 16, lengths, rot, False)
        lengths[-1] = lengths[0] = (0, 0)       # idle at either end
        check(torch_gpu, "float16", dim, 3, 2, 16, lengths, rot, True)
