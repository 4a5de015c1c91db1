"""The layout of attention's workspace where parts of split tiles are stored in words of 16 bytes."""
import ctypes as C

import pytest

from leanstream_amd import _native
from test_decode_refusals import attention


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,q_heads,kv_heads", [(31, 7, 1), (33, 5, 5), (101, 3, 1), (32, 8, 2)])
def test_parts_begin_at_multiples_of_16_bytes(dim, tokens, q_heads, kv_heads):
    """A part is tokens x q_heads rows of dim + 2 floats; the workspace ends with the last of an odd number of them."""
    steps = 256 if dim == 256 else 512
    for parts in (3, 5):
        block = attention(tokens=tokens, max_new=tokens, sequences=1, q_heads=q_heads, kv_heads=kv_heads, head_dim=dim,
                          q_token_stride=q_heads * dim, out_token_stride=q_heads * dim, q_head_stride=dim, out_head_stride=dim,
                          k_slot_stride=dim, v_slot_stride=dim, max_context=parts * steps, table_width=1024, table_stride=1024)
        need = _native.library().ls_hip_attention_workspace(C.byref(block))
        assert need >= parts * tokens * q_heads * (dim + 2) * 4
        assert need % 16 == 0
