"""Shapes at the edge of the decode-step operators (leanstream_amd.decode): no tokens, no rows, one of everything."""
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


def test_the_stride_of_a_dimension_of_one_does_not_matter(torch_gpu):
    """One token from a row of an odd width, one KV head, one slot a page, one page: equal to plain tensors' results."""
    torch = torch_gpu
    from leanstream_amd import decode

    g = torch.Generator().manual_seed(3)
    heads, dim, keys = 4, 64, 5
    for pages, page in ((5, 1), (1, 16)):
        q, k, v = (torch.randn(*shape, generator=g).half().cuda()
                   for shape in ((1, heads, dim), (pages, 1, page, dim), (pages, 1, page, dim)))
        table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        start, context = ints(torch, 0, 1), ints(torch, keys)
        out = torch.empty_like(q)
        decode.PagedAttention(q, decode.PagedCache(k, v), table, start, context, out, max_new=1, max_context=keys).enqueue()

        def odd(t):     # the same elements, an odd stride wherever a dimension is 1
            strides = [t.stride(d) if t.shape[d] > 1 else 7 + 2 * d for d in range(t.dim() - 1)] + [1]
            return t.as_strided(t.shape, strides)

        got = torch.empty_like(q)
        decode.PagedAttention(odd(q), decode.PagedCache(odd(k), odd(v)), table, start, context, odd(got), max_new=1,
                              max_context=keys).enqueue()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and out.isfinite().all()
