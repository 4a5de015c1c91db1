"""The argument checks of the decode-step operators (CPU: decided before any HIP call)."""
import ctypes as C

import pytest

from leanstream_amd import _native

EINVAL, ENOTSUP, ENOSPC = 22, 95, 28
NAN, INF = float("nan"), float("inf")


def attention(**kw):
    f = dict(q=0x1000, out=0x2000, k_pages=0x3000, v_pages=0x4000, page_table=0x5000, q_start=0x6000, context=0x7000,
             q_token_stride=4096, q_head_stride=128, out_token_stride=4096, out_head_stride=128, k_page_stride=16384,
             k_head_stride=2048, k_slot_stride=128, v_page_stride=16384, v_head_stride=2048, v_slot_stride=128,
             table_stride=8, tokens=4, sequences=2, q_heads=32, kv_heads=8, head_dim=128, pages=16, page_size=16,
             table_width=8, max_new=2, max_context=128, dtype=0, scale=0.1)
    f.update(kw)
    return _native.Attention(**f)


def append(**kw):
    f = dict(q=0x1000, k=0x1000, v=0x1000, cos=0x1000, sin=0x1000, q_out=0x1000, k_pages=0x3000, v_pages=0x4000,
             page_table=0x5000, q_start=0x6000, context=0x7000, table_stride=8, tokens=4, sequences=2, q_heads=32,
             kv_heads=8, head_dim=128, rot=128, positions=64, pages=16, page_size=16, table_width=8, dtype=1)
    f.update(kw)
    return _native.Append(**f)


def norm(**kw):
    f = dict(block=0x1000, residual=0x2000, pre_weight=0x3000, hidden=0x4000, normed=0x5000, block_stride=64,
             residual_stride=64, hidden_stride=64, normed_stride=64, rows=2, width=64, dtype=0, residual_scale=1.0,
             eps=1e-5)
    f.update(kw)
    return _native.BlockNorm(**f)


def sample(**kw):
    f = dict(logits=0x1000, uniform=0x2000, tokens=0x3000, row_stride=100, rows=2, vocab=100, dtype=2)
    f.update(kw)
    return _native.Sample(**f)


LONG = dict(max_context=16384, table_width=1024, table_stride=1024)
CASES = [
    ("attention", attention, [
        (dict(q=None), EINVAL), (dict(out=None), EINVAL), (dict(k_pages=None), EINVAL), (dict(context=None), EINVAL),
        (dict(sequences=0), EINVAL), (dict(kv_heads=0), EINVAL), (dict(kv_heads=5), EINVAL), (dict(pages=0), EINVAL),
        (dict(page_size=24), EINVAL), (dict(page_size=0), EINVAL), (dict(max_context=129), EINVAL),
        (dict(max_new=5), EINVAL), (dict(table_stride=7), EINVAL), (dict(scale=NAN), EINVAL), (dict(scale=INF), EINVAL),
        (dict(q=0x1008), EINVAL), (dict(out=0x1002), EINVAL), (dict(workspace=0x1004), EINVAL),
        (dict(q_head_stride=132), EINVAL), (dict(v_slot_stride=-128), EINVAL), (dict(dtype=3), EINVAL),
        (dict(window=0x40000000), EINVAL), (dict(dtype=2), ENOTSUP), (dict(head_dim=96), ENOTSUP),
        (dict(k_slot_stride=1 << 27), ENOTSUP), (dict(LONG), ENOSPC),
        (dict(LONG, workspace=0x1000, workspace_bytes=64), ENOSPC)]),
    ("append", append, [
        (dict(k=None), EINVAL), (dict(v_pages=None), EINVAL), (dict(q=None), EINVAL), (dict(q_out=None), EINVAL),
        (dict(cos=None), EINVAL), (dict(positions=0), EINVAL), (dict(rot=130), EINVAL), (dict(rot=127), EINVAL),
        (dict(head_dim=127), EINVAL), (dict(page_size=12), EINVAL), (dict(table_stride=1), EINVAL),
        (dict(k=0x1001), EINVAL), (dict(k_token_stride=-8), EINVAL), (dict(dtype=3), EINVAL), (dict(dtype=2), ENOTSUP)]),
    ("block_norm", norm, [
        (dict(block=None), EINVAL), (dict(residual=None), EINVAL), (dict(hidden=None, normed=None), EINVAL),
        (dict(pre_weight=None), EINVAL), (dict(width=0), EINVAL), (dict(eps=-1.0), EINVAL), (dict(eps=NAN), EINVAL),
        (dict(residual_scale=INF), EINVAL), (dict(gate=0x1001), EINVAL), (dict(hidden_stride=63), EINVAL),
        (dict(dtype=3), EINVAL), (dict(width=16385, hidden_stride=16385, normed_stride=16385), ENOTSUP)]),
    ("sample", sample, [
        (dict(logits=None), EINVAL), (dict(uniform=None), EINVAL), (dict(tokens=None), EINVAL), (dict(vocab=0), EINVAL),
        (dict(dtype=3), EINVAL), (dict(logits=0x1002), EINVAL), (dict(tokens=0x1001), EINVAL),
        (dict(row_stride=-1), EINVAL), (dict(workspace=0x1008), EINVAL), (dict(vocab=(1 << 20) + 1), ENOTSUP),
        (dict(), ENOSPC), (dict(workspace=0x1000, workspace_bytes=64), ENOSPC)]),
]


@pytest.mark.parametrize("name,make,change,code", [(n, m, ch, code) for n, m, rows in CASES for ch, code in rows])
def test_refused(name, make, change, code):
    enqueue = getattr(_native.library(), f"ls_hip_{name}_enqueue")
    assert enqueue(C.byref(make(**change)), None) == code


@pytest.mark.parametrize("name,make,empty", [("attention", attention, dict(tokens=0, max_new=0)),
                                             ("attention", attention, dict(max_new=0)), ("append", append, dict(tokens=0)),
                                             ("block_norm", norm, dict(rows=0)), ("sample", sample, dict(rows=0))])
def test_null_block_is_refused_and_nothing_to_do_is_fine(name, make, empty):
    enqueue = getattr(_native.library(), f"ls_hip_{name}_enqueue")
    assert enqueue(None, None) == EINVAL
    assert enqueue(C.byref(make(**empty)), None) == 0


def test_blocks_have_the_c_layout():
    """Pointers and 64-bit words first, so the sizes follow from the counts."""
    assert C.sizeof(_native.Attention) == 11 * 8 + 11 * 8 + 14 * 4
    assert C.sizeof(_native.Append) == 12 * 8 + 15 * 8 + 12 * 4
    assert C.sizeof(_native.BlockNorm) == 7 * 8 + 5 * 8 + 6 * 4
    assert C.sizeof(_native.Sample) == 9 * 8 + 2 * 8 + 3 * 4 + 4   # padded to 8 bytes


def test_classes_refuse_tensors_off_the_gpu():
    torch = pytest.importorskip("torch")
    from leanstream_amd import decode

    pages = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="not on the GPU"):
        decode.PagedCache(pages, pages)
    with pytest.raises(ValueError, match="not on the GPU"):
        decode.BlockNorm(pages[0, 0], pages[0, 0], pages[0, 0], None)
    with pytest.raises(ValueError, match="not on the GPU"):
        decode.Sampler(torch.zeros(1, 8), torch.zeros(1), torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("name,make,fields", [
    ("attention", attention, ["page_table", "q_start", "context", "lse", "status"]),
    ("append", append, ["cos", "sin", "page_table", "q_start", "context", "status"])])
def test_words_off_their_alignment_are_refused(name, make, fields):
    call = getattr(_native.library(), f"ls_hip_{name}_enqueue")
    for field in fields:
        assert call(C.byref(make(**{field: 0x9002})), None) == EINVAL, field


@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_scales_that_are_not_positive_are_refused(scale):
    """Masks and maxima are taken before the scale."""
    assert _native.library().ls_hip_attention_enqueue(C.byref(attention(scale=scale)), None) == EINVAL
