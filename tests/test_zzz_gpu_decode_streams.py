"""The decode-step operators on a stream other than torch's current one, and in graphs.

Named to run last: torch keeps the streams that it makes here, and the device has four hardware queues. Tests that
copy on side streams beside a waiting kernel need a queue of their own for them.
"""
import math

import pytest

from test_gpu_attention import CASES, Problem
from test_gpu_sampling import random_rows

pytestmark = pytest.mark.gpu


def calls(torch):
    """(name, call, outputs, function that changes its inputs)"""
    from leanstream_amd import decode

    out = []
    for name in ("decode", "few_tokens", "ragged", "window_sinks"):
        p = Problem(torch, "float16", **CASES[name])
        out.append((f"attention {name}", p.on_gpu(), (p.out, p.lse), lambda i, p=p: p.q_gpu.copy_((p.q * (1 + i)).to(p.q.dtype))))

    x, residual, gate = (torch.randn(33, 4096, device="cuda").half() for _ in range(3))
    w = torch.rand(4096, device="cuda").half()
    hidden, normed = torch.empty_like(x), torch.empty_like(x)
    out.append(("norm", decode.BlockNorm(x, residual, hidden, normed, w, w, gate), (hidden, normed), lambda i: x.normal_()))

    q, k, v = (torch.randn(9, h, 128, device="cuda").half() for h in (8, 2, 2))
    cache = decode.PagedCache(*(torch.zeros(12, 2, 16, 128, device="cuda", dtype=torch.float16) for _ in range(2)))
    table = torch.randperm(12, device="cuda").to(torch.int32).view(3, 4)
    start = torch.tensor([0, 1, 8, 9], dtype=torch.int32, device="cuda")
    context = torch.tensor([5, 40, 64], dtype=torch.int32, device="cuda")
    angle = torch.rand(64, 64, device="cuda") * 6
    rotated = torch.empty_like(q)
    out.append(("append", decode.AppendKV(q, k, v, angle.cos(), angle.sin(), cache, table, start, context, rotated),
                (rotated, cache.k, cache.v), lambda i: (q.normal_(), k.normal_(), v.normal_())))

    for kw in (dict(top_p=torch.full((7,), 0.9, device="cuda")), dict(top_k=torch.full((7,), 30, device="cuda", dtype=torch.int32)), {}):
        logits, u, _ = random_rows(torch, 7, 50000, "bfloat16", 9)
        uniform, tokens = torch.tensor(u, device="cuda"), torch.empty(7, dtype=torch.int32, device="cuda")
        logprob = torch.empty(7, device="cuda")
        out.append((f"sample {list(kw)}", decode.Sampler(logits, uniform, tokens, logprob, **kw), (tokens, logprob),
                    lambda i, logits=logits, uniform=uniform: (uniform.uniform_(), logits.normal_().mul_(2))))
    return out


def spoil(tensors):
    for t in tensors:
        t.fill_(math.nan if t.is_floating_point() else -9)


def bits(tensors):
    return [t.clone().view(torch_int(t)) for t in tensors]


def torch_int(t):
    import torch

    return torch.int16 if t.element_size() == 2 else torch.int32


def same(a, b):
    return all(bool((x == y).all()) for x, y in zip(a, b))


def test_another_stream(torch_gpu):
    torch = torch_gpu
    side = torch.cuda.Stream()
    for name, call, outputs, change in calls(torch):
        print("case:", name, flush=True)
        for i in range(3):
            change(i)
            spoil(outputs)
            call.enqueue()
            torch.cuda.synchronize()
            want = bits(outputs)
            spoil(outputs)
            torch.cuda.synchronize()
            if i % 2:
                with torch.cuda.stream(side):   # torch's current stream, inside
                    call.enqueue()
            else:
                call.enqueue(side.cuda_stream)
            side.synchronize()
            assert same(bits(outputs), want), name


def test_in_graphs(torch_gpu):
    """Replays, with eager work between them, against eager calls on the same inputs."""
    torch = torch_gpu
    for name, call, outputs, change in calls(torch):
        print("case:", name, flush=True)
        call.enqueue()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call.enqueue()
        for i in range(4):
            change(i)
            spoil(outputs)
            call.enqueue()
            torch.cuda.synchronize()
            want = bits(outputs)
            spoil(outputs)
            graph.replay()
            torch.cuda.synchronize()
            assert same(bits(outputs), want), name
