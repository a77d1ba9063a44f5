"""The operators around drafted tokens and 8-bit caches, as far as they answer without a GPU: what the C entry points and
the Python functions refuse, empty calls, workspace sizes, a cache of codes."""

import ctypes

import numpy as np
import pytest
import torch

from fast_infer_b200 import _lib
from fast_infer_b200.kv_cache import KVCache

BAD, UNSUPPORTED, ALIGN, WORKSPACE, OK = (_lib.FI_ERR_INVALID_ARG, _lib.FI_ERR_UNSUPPORTED, _lib.FI_ERR_ALIGNMENT,
                                          _lib.FI_ERR_WORKSPACE, _lib.FI_OK)
NAN, INF = float("nan"), float("inf")
I8, E4M3, F32 = _lib.FI_DTYPE_I8, _lib.FI_DTYPE_E4M3, _lib.FI_DTYPE_F32
CPU = torch.device("cpu")


def _tree(lib, ptr=16, scale_ptr=16, mask=None, depths=None, words=1, batch=2, total=5, hq=6, hk=2, d=128, nb=4, bs=64,
          mb=4, scale=0.1, cap=0.0, window=0, dtype=0, cache=0, q_strides=(768, 128, 1), o_strides=(768, 128, 1),
          kv_strides=(64 * 256, 256, 128, 1), ws=None, ws_bytes=0):
    kv, ss = _lib.strides(*kv_strides), _lib.strides(128, 64, 1)
    return lib.fi_paged_tree(ptr, ptr, ptr, scale_ptr, scale_ptr, ptr, None, ptr, ptr, ptr, mask, depths, words, batch,
                             total, hq, hk, d, nb, bs, mb, _lib.strides(*q_strides), kv, kv, ss, ss,
                             _lib.strides(*o_strides), _lib.strides(mb, 1), scale, cap, window, dtype, cache, ws,
                             ws_bytes, None, None)


def test_tree_attention_refusals():
    lib = _lib.load()
    big = dict(ws=16, ws_bytes=1 << 40)
    for bad in (dict(batch=-1), dict(total=-1), dict(hq=0), dict(hk=0), dict(hq=7), dict(nb=0), dict(mb=0), dict(window=-1),
                dict(dtype=2), dict(dtype=4), dict(cache=1), dict(cache=4), dict(cache=-1), dict(scale=0.0), dict(scale=NAN),
                dict(cap=-1.0), dict(cap=INF), dict(ptr=None), dict(mask=16, words=0), dict(mask=16, words=65537),
                dict(mask=16, window=5), dict(cache=I8, scale_ptr=None), dict(cache=E4M3, dtype=1, scale_ptr=None)):
        assert _tree(lib, **{**big, **bad}) == BAD, bad
    for unsup in (dict(d=64), dict(bs=16), dict(hq=130, hk=2), dict(batch=2049), dict(total=(1 << 28) + 1),
                  dict(cache=I8, batch=2049)):
        assert _tree(lib, **{**big, **unsup}) == UNSUPPORTED, unsup
    for kind in (0, I8, E4M3):
        assert _tree(lib, cache=kind) == WORKSPACE
        assert _tree(lib, cache=kind, ws=16, ws_bytes=64) == WORKSPACE
        assert _tree(lib, cache=kind, ws=8, ws_bytes=1 << 40) == ALIGN
        assert _tree(lib, cache=kind, o_strides=(770, 128, 1), **big) == ALIGN
        assert _tree(lib, cache=kind, ptr=None, batch=0) == OK and _tree(lib, cache=kind, ptr=None, total=0) == OK
    assert _tree(lib, cache=I8, q_strides=(770, 128, 1), **big) == ALIGN
    assert _tree(lib, cache=I8, q_strides=(768, 128, 2), **big) == ALIGN
    assert _tree(lib, cache=I8, total=50, kv_strides=(64 * 256, 256, 128, 2), **big) == ALIGN


def test_tree_workspace_is_that_of_the_kernels_it_launches():
    lib = _lib.load()
    for size in ((1, 24, 8), (10, 24, 8), (11, 24, 8), (5000, 24, 8), (0, 24, 8), (1, 25, 8), (1, 65, 1)):
        assert lib.fi_paged_tree_workspace_size(*size) == lib.fi_paged_chunk_workspace_size(*size)


def _rope8(lib, ptr=16, sp=16, total=5, batch=2, nq=6, nkv=2, d=128, nb=4, bs=64, mb=4, dtype=0, cache=I8,
           kv_strides=(64 * 256, 256, 128, 1)):
    kv, ss = _lib.strides(*kv_strides), _lib.strides(128, 64, 1)
    return lib.fi_rope_axes_store8(ptr, ptr, ptr, ptr, sp, sp, ptr, ptr, ptr, ptr, ptr, ptr, total, batch, nq, nkv, d, 1,
                                   _lib.strides(64), total, 100, 128, nb, bs, mb, _lib.strides(1280, 1),
                                   _lib.strides(768, 128, 1), kv, kv, ss, ss, _lib.strides(mb, 1), dtype, cache, None, None)


def _read8(lib, ptr=16, sp=16, total=5, batch=2, nkv=2, d=128, nb=4, bs=64, mb=4, dtype=0, cache=I8,
           kv_strides=(64 * 256, 256, 128, 1), out_strides=(256, 128, 1)):
    kv, ss, out = _lib.strides(*kv_strides), _lib.strides(128, 64, 1), _lib.strides(*out_strides)
    return lib.fi_read_kv8(ptr, ptr, sp, sp, ptr, ptr, ptr, ptr, ptr, total, batch, nkv, d, nb, bs, mb, kv, kv, ss, ss,
                           out, out, _lib.strides(mb, 1), dtype, cache, None, None)


@pytest.mark.parametrize("call", [_rope8, _read8])
def test_store_and_read_refusals(call):
    lib = _lib.load()
    for bad in (dict(total=-1), dict(batch=-1), dict(nkv=0), dict(nb=0), dict(mb=0), dict(dtype=2), dict(cache=0),
                dict(cache=1), dict(cache=4), dict(ptr=None), dict(sp=None)):
        assert call(lib, **bad) == BAD, bad
    for unsup in (dict(d=64), dict(bs=16), dict(total=(1 << 28) + 1), dict(nb=(1 << 30) + 1)):
        assert call(lib, **unsup) == UNSUPPORTED, unsup
    for strides in ((64 * 256, 256, 128, 2), (64 * 256, 264, 128, 1), (64 * 256 + 8, 256, 128, 1)):
        assert call(lib, kv_strides=strides) == ALIGN, strides  # (multiples of 8 are not enough for codes)
    assert call(lib, ptr=24) == ALIGN
    assert call(lib, ptr=None, total=0) == OK and call(lib, ptr=None, batch=0) == OK
    if call is _read8:
        assert call(lib, out_strides=(260, 128, 1)) == ALIGN


def test_drafting_refusals():
    lib = _lib.load()
    tree = lambda ptr=16, total=5, batch=2, words=1, window=0: lib.fi_draft_tree(  # noqa: E731
        ptr, ptr, ptr, ptr, total, batch, words, window, None, None)
    for bad in (dict(total=-1), dict(batch=-1), dict(words=0), dict(window=-1), dict(ptr=None)):
        assert tree(**bad) == BAD, bad
    for unsup in (dict(total=(1 << 28) + 1), dict(batch=(1 << 20) + 1), dict(words=(1 << 16) + 1)):
        assert tree(**unsup) == UNSUPPORTED
    assert tree(ptr=None, total=0) == OK and tree(ptr=None, batch=0) == OK
    accept = lambda ptr=16, total=5, batch=2: lib.fi_accept_drafts(  # noqa: E731
        ptr, ptr, ptr, ptr, ptr, ptr, ptr, total, batch, None, None)
    assert accept(total=-1) == accept(batch=-1) == accept(ptr=None) == BAD and accept(ptr=None, batch=0) == OK
    assert accept(total=(1 << 28) + 1) == UNSUPPORTED

    def keep(ptr=16, sp=None, layers=1, batch=2, total=5, heads=2, d=128, nb=4, bs=64, mb=4, dtype=0,
             strides=(65536, 16384, 256, 128, 1)):
        st, ss = _lib.strides(*strides), _lib.strides(512, 128, 64, 1)
        return lib.fi_keep_accepted(ptr, ptr, sp, sp, ptr, ptr, ptr, ptr, ptr, layers, batch, total, heads, d, nb, bs, mb,
                                    st, st, ss, ss, _lib.strides(mb, 1), dtype, None, None)
    for bad in (dict(layers=-1), dict(batch=-1), dict(total=-1), dict(heads=0), dict(nb=0), dict(mb=0), dict(dtype=4),
                dict(dtype=-1), dict(ptr=None), dict(dtype=I8), dict(dtype=E4M3)):  # (codes without scales)
        assert keep(**bad) == BAD, bad
    for unsup in (dict(d=64), dict(bs=16), dict(layers=65536), dict(nb=(1 << 30) + 1)):
        assert keep(**unsup) == UNSUPPORTED, unsup
    assert keep(ptr=24) == ALIGN and keep(strides=(65536, 16384, 260, 128, 1)) == ALIGN
    assert keep(dtype=I8, sp=16, strides=(65536, 16384, 264, 128, 1)) == ALIGN
    assert keep(ptr=None, layers=0) == OK and keep(ptr=None, batch=0) == OK and keep(ptr=None, total=0) == OK


def test_sampling_refusals():
    lib = _lib.load()

    def sample(ptr=16, rows=3, vocab=100, dtype=F32):
        return lib.fi_sample_tokens(ptr, ptr, None, None, None, None, 1.0, 0, 1.0, 0.0, ptr, rows, vocab, vocab, dtype, None)
    for bad in (dict(rows=-1), dict(vocab=0), dict(dtype=2), dict(dtype=3), dict(dtype=5), dict(ptr=None)):
        assert sample(**bad) == BAD, bad
    assert sample(vocab=262145) == UNSUPPORTED and sample(rows=(1 << 24) + 1) == UNSUPPORTED
    assert sample(ptr=18) == ALIGN and sample(ptr=None, rows=0) == OK


def test_python_functions_reject_cpu_tensors_and_types():
    from fast_infer_b200.kernels.attention import paged_tree_attention
    from fast_infer_b200.kernels.drafting import accept_drafts, draft_tree, keep_accepted
    from fast_infer_b200.kernels.rope import read_kv
    from fast_infer_b200.kernels.sampling import sample_tokens
    q = torch.zeros(3, 6, 128, dtype=torch.float16)
    kv = torch.zeros(4, 64, 2, 128, dtype=torch.int8)
    i, t, s = torch.zeros(2, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(4, 2, 64)
    for call in (lambda: paged_tree_attention(q, kv, kv, t, 64, i, i[:1], k_scale=s, v_scale=s),
                 lambda: read_kv(kv, kv, s, s, t, 64, i, i[:1], 3), lambda: draft_tree(i, i, 2),
                 lambda: accept_drafts(i, i, i, i), lambda: sample_tokens(torch.zeros(2, 9), torch.zeros(2)),
                 lambda: keep_accepted(kv[None], kv[None], t, 64, i, i[:1], i, i[:1], k_scale=s[None], v_scale=s[None])):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: paged_tree_attention(None, kv, kv, t, 64, i, i[:1]), lambda: draft_tree(None, i, 2),
                 lambda: accept_drafts([1], i, i, i), lambda: sample_tokens(None, i), lambda: read_kv(None, kv, s, s, t, 64, i, i, 1),
                 lambda: keep_accepted(None, kv, t, 64, i, i, i, i)):
        with pytest.raises(TypeError):
            call()


def test_cache_of_codes():
    for dtype in (torch.int8, torch.float8_e4m3fn):
        cache = KVCache(2, 3, 128, 256, 64, CPU, num_blocks=5, dtype=dtype)
        assert cache.k.dtype == cache.v.dtype == dtype and cache.k.shape == (2, 5, 64, 3, 128)
        assert cache.k_scale.shape == cache.v_scale.shape == (2, 5, 3, 64) and cache.k_scale.dtype == torch.float32
        cu, ctx = cache.extend([70, 3])
        assert cu.tolist() == [0, 70, 73] and ctx.tolist() == [70, 3]
        rows = torch.zeros(1, 1, 3, 128, dtype=dtype)
        with pytest.raises(ValueError, match="rope_axes_store"):
            cache.write_tokens(0, rows, rows, 0)
        with pytest.raises(ValueError, match="batch larger"):
            cache.accept(torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), cu, cu)
    assert KVCache(1, 2, 128, 64, 64, CPU).k_scale is None
    with pytest.raises(TypeError, match="int8"):
        KVCache(1, 2, 128, 64, 64, CPU, dtype=torch.float32)


def test_sizes_of_scales_are_checked():
    from fast_infer_b200.kernels.attention import _check_scales
    codes, halves = torch.zeros(1, dtype=torch.int8), torch.zeros(1, dtype=torch.float16)
    good = torch.zeros(4, 2, 64)
    _check_scales(codes, good, good, (4, 2, 64))
    _check_scales(halves, None, None, (4, 2, 64))
    for k, v in ((None, good), (good, None), (good[:3], good), (good, good.double()), (good, good.transpose(1, 2))):
        with pytest.raises(ValueError, match="scale"):
            _check_scales(codes, k, v, (4, 2, 64))
    with pytest.raises(ValueError, match="scale"):
        _check_scales(halves, good, good, (4, 2, 64))
