"""Strides of dimensions of size 1 as the C entry points see them (past that check, a missing workspace ends the call)."""

from fast_infer_b200 import _lib
from tests.test_chunk_host import ALIGN, WORKSPACE, _chunk


def test_chunk_output_of_one_token_or_head():
    lib = _lib.load()
    for odd in (dict(total=1, o_strides=(771, 128, 1)), dict(hq=1, hk=1, o_strides=(128, 129, 1)),
                dict(total=1, hq=1, hk=1, o_strides=(129, 131, 1))):
        assert _chunk(lib, ws=16, ws_bytes=64, **odd) == WORKSPACE, odd
    for bad in (dict(total=2, o_strides=(771, 128, 1)), dict(total=1, o_strides=(768, 129, 1)),
                dict(total=1, o_strides=(768, 128, 2))):
        assert _chunk(lib, ws=16, ws_bytes=64, **bad) == ALIGN, bad
