"""A call's own workspace and streams other than the one on which the call was bound (leanstream_amd.decode).

Named to run last: torch keeps the streams that it makes here, and the device has four hardware queues.
"""
import math

import pytest

from test_gpu_attention import CASES, Problem
from test_gpu_sampling import random_rows

pytestmark = pytest.mark.gpu

CYCLES = 50_000_000     # some 20 ms of a stream's time


def attention(torch):
    """(function that binds the call anew, outputs, tensors to keep): splits of few rows, whose counters begin at 0."""
    from leanstream_amd import decode

    p = Problem(torch, "float16", 128, 8, 2, 16, [(1, 6000), (3, 4000)])
    q, out, lse, k, v, table, q_start, context, _ = p.on_gpu()._keep
    return lambda: decode.PagedAttention(q, decode.PagedCache(k, v), table, q_start, context, out, max_new=3,
                                         max_context=6000, lse=lse), (out, lse), p


def sampler(torch):
    from leanstream_amd import decode

    logits, u, _ = random_rows(torch, 7, 50000, "bfloat16", 9)
    uniform, tokens = torch.tensor(u, device="cuda"), torch.empty(7, dtype=torch.int32, device="cuda")
    top_p, logprob = torch.full((7,), 0.9, device="cuda"), torch.empty(7, device="cuda")
    return lambda: decode.Sampler(logits, uniform, tokens, logprob, top_p=top_p), (tokens, logprob), None


def spoil(torch, outputs):
    for t in outputs:
        t.fill_(math.nan if t.is_floating_point() else -9)
    torch.cuda.synchronize()


def bits(outputs):
    return [t.clone() for t in outputs]


def same(torch, outputs, want):
    return all(torch.equal(a, b) for a, b in zip(outputs, want))


def used_memory(torch, size):
    """A block of that size that held other bytes before, for the next allocation."""
    torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("make", [attention, sampler])
def test_first_call_on_another_stream(torch_gpu, make):
    """The stream on which the call is bound is busy, so that its workspace is zeroed late."""
    torch = torch_gpu
    bind, outputs, _ = make(torch)
    first = bind()
    first.enqueue()
    torch.cuda.synchronize()
    want, need = bits(outputs), first.workspace.numel()
    side = torch.cuda.Stream()
    for by_handle in (True, False, True):
        spoil(torch, outputs)
        used_memory(torch, need)
        torch.cuda.synchronize()
        torch.cuda._sleep(CYCLES)
        call = bind()
        for _ in range(2):
            if by_handle:
                call.enqueue(side.cuda_stream)
            else:
                with torch.cuda.stream(side):
                    call.enqueue()
        side.synchronize()
        assert same(torch, outputs, want)
        torch.cuda.synchronize()
        call.enqueue(side.cuda_stream)      # and from now on without a wait
        torch.cuda.synchronize()
        assert same(torch, outputs, want)
    # bound on the other stream, used on torch's default one
    spoil(torch, outputs)
    with torch.cuda.stream(side):
        used_memory(torch, need)
        torch.cuda._sleep(CYCLES)
        call = bind()
    call.enqueue()
    torch.cuda.current_stream().synchronize()
    assert same(torch, outputs, want)


@pytest.mark.parametrize("make", [attention, sampler])
def test_a_call_dropped_while_its_work_runs(torch_gpu, make):
    """Its workspace is nobody else's before that work has ended."""
    torch = torch_gpu
    bind, outputs, _ = make(torch)
    call = bind()
    call.enqueue()
    torch.cuda.synchronize()
    want, need = bits(outputs), call.workspace.numel()
    side = torch.cuda.Stream()
    spoil(torch, outputs)
    with torch.cuda.stream(side):
        torch.cuda._sleep(CYCLES)
    where = call.workspace.data_ptr()
    call.enqueue(side.cuda_stream)
    del call
    others = [torch.full((need,), 0xff, dtype=torch.uint8, device="cuda") for _ in range(4)]
    assert where not in [t.data_ptr() for t in others]
    torch.cuda.synchronize()
    assert same(torch, outputs, want)


def test_captures(torch_gpu):
    """A call bound before the capture goes into it. Inside, attention is refused a workspace of its own, which would be
    zeroed in the graph alone; the sampler's may hold anything."""
    torch = torch_gpu
    for make in (attention, sampler):
        bind, outputs, _ = make(torch)
        call = bind()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call.enqueue()
            if make is attention:
                with pytest.raises(RuntimeError, match="before the capture"):
                    bind()
            else:
                inside = bind()
                inside.enqueue()
        call.enqueue()
        torch.cuda.synchronize()
        want = bits(outputs)
        for _ in range(3):
            spoil(torch, outputs)
            graph.replay()
            torch.cuda.synchronize()
            assert same(torch, outputs, want)
