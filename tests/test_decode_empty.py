"""Calls without tokens or rows are fine (CPU: decided before any HIP call): the pointers of empty tensors are NULL."""
import ctypes as C

import pytest

from leanstream_amd import _native
from test_decode_refusals import EINVAL, append, attention, norm, sample

EMPTY = [
    ("attention", attention, dict(tokens=0, max_new=0, q=None, out=None)),
    ("attention", attention, dict(tokens=0, max_new=0, q=None, out=None, sequences=0, page_table=None, q_start=None,
                                  context=None)),
    ("append", append, dict(tokens=0, q=None, k=None, v=None, q_out=None)),
    ("append", append, dict(tokens=0, q=None, k=None, v=None, q_out=None, cos=None, sin=None, positions=0)),
    ("append", append, dict(tokens=0, q=None, k=None, v=None, q_out=None, sequences=0, page_table=None, q_start=None,
                            context=None)),
    ("block_norm", norm, dict(rows=0, block=None, residual=None, hidden=None, normed=None)),
    ("sample", sample, dict(rows=0, logits=None, uniform=None, tokens=None)),
]


@pytest.mark.parametrize("name,make,fields", EMPTY)
def test_nothing_to_do_without_pointers(name, make, fields):
    lib = _native.library()
    block = make(**fields)
    assert getattr(lib, f"ls_hip_{name}_enqueue")(C.byref(block), None) == 0
    if hasattr(block, "workspace"):
        assert getattr(lib, f"ls_hip_{name}_workspace")(C.byref(block)) == 0


@pytest.mark.parametrize("name,make,fields", [
    ("attention", attention, dict(tokens=0, max_new=0, head_dim=128, kv_heads=5)), ("append", append, dict(tokens=0, rot=130)),
    ("block_norm", norm, dict(rows=0, eps=-1.0)), ("sample", sample, dict(rows=0, dtype=3))])
def test_what_does_not_depend_on_tensors_is_checked_all_the_same(name, make, fields):
    assert getattr(_native.library(), f"ls_hip_{name}_enqueue")(C.byref(make(**fields)), None) == EINVAL
