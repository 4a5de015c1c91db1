"""Shapes at the edge of the decode-step operators (leanstream_amd.decode): no tokens, no rows."""
import pytest

pytestmark = pytest.mark.gpu


def ints(torch, *values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("sequences", [0, 3])
def test_no_tokens_and_no_rows(torch_gpu, sequences):
    torch = torch_gpu
    from leanstream_amd import decode

    def half(*shape):
        return torch.full(shape, 1.5, dtype=torch.float16, device="cuda")

    cache = decode.PagedCache(half(4, 2, 16, 64), half(4, 2, 16, 64))
    table = torch.zeros(sequences, 4, dtype=torch.int32, device="cuda")
    start, context = ints(torch, *[0] * (sequences + 1)), ints(torch, *[9] * sequences)
    status = ints(torch, 0)
    cos = torch.ones(64, 32, device="cuda")
    q, kv = half(0, 8, 64), half(0, 2, 64)
    calls = [decode.PagedAttention(q, cache, table, start, context, half(0, 8, 64), max_new=1, max_context=64,
                                   lse=torch.empty(0, 8, device="cuda"), status=status),
             decode.AppendKV(q, kv, kv, cos, cos, cache, table, start, context, half(0, 8, 64), status=status),
             decode.AppendKV(None, kv, kv, None, None, cache, table, start, context, None, status=status),
             decode.BlockNorm(half(0, 128), half(0, 128), half(0, 128), half(0, 128), half(128), half(128)),
             decode.Sampler(half(0, 1000), torch.empty(0, device="cuda"), ints(torch), torch.empty(0, device="cuda"))]
    for call in calls:
        call.enqueue()
    torch.cuda.synchronize()
    assert int(status) == 0
    assert (cache.k == 1.5).all() and (cache.v == 1.5).all()
