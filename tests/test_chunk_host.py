"""The operators over new tokens and a paged cache, as far as they answer without a GPU: arguments
that the C entry points and the Python functions refuse, empty calls, workspace sizes, and the
cache's bookkeeping around them."""

import ctypes

import numpy as np
import pytest
import torch

from fast_infer_b200 import _lib
from fast_infer_b200.kv_cache import KVCache

BAD, UNSUPPORTED, ALIGN, WORKSPACE, OK = (_lib.FI_ERR_INVALID_ARG, _lib.FI_ERR_UNSUPPORTED,
                                          _lib.FI_ERR_ALIGNMENT, _lib.FI_ERR_WORKSPACE, _lib.FI_OK)
NAN, INF = float("nan"), float("inf")


def _chunk(lib, ptr=16, batch=2, total=5, hq=6, hk=2, d=128, nb=4, bs=64, mb=4, scale=0.1, cap=0.0,
           window=0, dtype=0, o_strides=(768, 128, 1), q_strides=(768, 128, 1), ws=None, ws_bytes=0):
    kv = _lib.strides(64 * 256, 256, 128, 1)
    return lib.fi_paged_chunk(ptr, ptr, ptr, ptr, None, ptr, ptr, ptr, None, None, batch, total, hq, hk,
                              d, nb, bs, mb, _lib.strides(*q_strides), kv, kv,
                              _lib.strides(*o_strides), _lib.strides(mb, 1), scale, cap, window, dtype,
                              ws, ws_bytes, None, None)


def _mass(lib, ptr=16, batch=2, total=5, hq=6, hk=2, d=128, nb=4, bs=64, mb=4, cap=256, accumulate=1,
          scale=0.1, softcap=0.0, window=0, dtype=0, ws=None, ws_bytes=0):
    return lib.fi_attention_mass(ptr, ptr, ptr, ptr, ptr, ptr, ptr, None, None, batch, total, hq, hk, d,
                                 nb, bs, mb, _lib.strides(768, 128, 1),
                                 _lib.strides(64 * 256, 256, 128, 1), _lib.strides(mb, 1), cap,
                                 accumulate, scale, softcap, window, dtype, ws, ws_bytes, None, None)


@pytest.mark.parametrize("call", [_chunk, _mass])
def test_chunk_and_mass_refusals(call):
    lib = _lib.load()
    for bad in (dict(batch=-1), dict(total=-1), dict(hq=0), dict(hk=0), dict(hq=7), dict(nb=0), dict(mb=0),
                dict(window=-1), dict(dtype=2), dict(scale=0.0), dict(scale=-0.1), dict(scale=NAN),
                dict(scale=INF), dict(ptr=None)):
        assert call(lib, **bad) == BAD, bad
    soft = "softcap" if call is _mass else "cap"
    for x in (-1.0, NAN, INF, 1e-45, 3e38):  # (the last two: scale / cap or cap * log2(e) past fp32)
        assert call(lib, **{soft: x}) == BAD
    assert call(lib, scale=3e38) == BAD
    for unsup in (dict(d=64), dict(bs=16), dict(hq=130, hk=2), dict(batch=2049), dict(total=(1 << 28) + 1),
                  dict(mb=(1 << 20) + 1)):
        assert call(lib, **unsup) == UNSUPPORTED, unsup
    assert call(lib) == WORKSPACE and b"workspace" in lib.fi_last_error()
    assert call(lib, ws=16, ws_bytes=64) == WORKSPACE
    assert call(lib, ws=8, ws_bytes=1 << 40) == ALIGN
    assert call(lib, ptr=None, batch=0) == OK
    if call is _chunk:
        assert call(lib, ptr=None, total=0) == OK
        assert call(lib, o_strides=(770, 128, 1), ws=16, ws_bytes=1 << 40) == ALIGN
        assert call(lib, o_strides=(768, 128, 2), ws=16, ws_bytes=1 << 40) == ALIGN
        assert call(lib, total=1 << 20, batch=1, hq=16, ws=16, ws_bytes=1 << 40) == UNSUPPORTED
        assert b"split the batch" in lib.fi_last_error()
    else:
        assert call(lib, ptr=None, cap=0) == OK
        assert call(lib, total=0, ws=None) == OK  # nothing to add
        assert call(lib, cap=-1) == BAD


def test_workspace_sizes():
    """One kernel's partial rows where all tokens fit one narrow unit, both kernels' else; 0 for sizes
    that are refused (148 SMs: a B200, and the count the library assumes with no device)."""
    if torch.cuda.is_available() and \
            torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("sizes below are for 148 SMs")
    lib = _lib.load()
    up = lambda n: -(-n // 256) * 256

    def part(rows):
        slots = 148 * 2 * rows
        return up(slots * 512) + up(slots * 4) + up(148 * 32)
    size = lib.fi_paged_chunk_workspace_size
    assert size(1, 24, 8) == part(32) == size(10, 24, 8)
    assert size(11, 24, 8) == part(32) + part(256) == size(100000, 24, 8)
    for bad in ((0, 24, 8), (1, 24, 0), (1, 25, 8), (1, 4, 8), (1, 65, 1)):
        assert size(*bad) == 0
    assert lib.fi_attention_mass_workspace_size() == 148 * (2 * 512 * 4 + 24)


def _evict(lib, ptr=16, out=32, layers=1, batch=2, heads=2, d=128, nb=4, nbo=4, bs=64, mb=4, mbo=4,
           cap=256, budget=64, recent=8, sinks=4, strides=(65536, 16384, 256, 128, 1), v_out=None, bt_out=None,
           out_strides=None):
    st = _lib.strides(*strides)
    so = _lib.strides(*(out_strides or strides))
    return lib.fi_kv_evict(ptr, ptr, ptr, ptr, ptr, out, out if v_out is None else v_out,
                           out if bt_out is None else bt_out, ptr, ptr, layers, batch, heads, d, nb, nbo, bs,
                           mb, mbo, cap, budget, recent, sinks, st, st, so, so, _lib.strides(mb, 1),
                           _lib.strides(mbo, 1), None, None)


def test_evict_refusals():
    lib = _lib.load()
    for bad in (dict(layers=-1), dict(batch=-1), dict(heads=0), dict(nb=0), dict(mbo=0), dict(cap=-1),
                dict(budget=0), dict(recent=-1), dict(sinks=-1), dict(recent=60, sinks=5),
                dict(budget=257), dict(ptr=None), dict(out=16, v_out=32), dict(out=16, bt_out=32),
                dict(v_out=16), dict(out=16, out_strides=(65536, 16384, 256, 0, 1))):
        assert _evict(lib, **bad) == BAD, bad
    for unsup in (dict(d=64), dict(bs=16), dict(layers=1 << 21), dict(nb=(1 << 30) + 1)):
        assert _evict(lib, **unsup) == UNSUPPORTED, unsup
    assert _evict(lib, strides=(65536, 16384, 256, 128, 2)) == ALIGN
    assert _evict(lib, strides=(65536, 16384, 260, 128, 1)) == ALIGN
    assert _evict(lib, out=40) == ALIGN
    assert _evict(lib, ptr=None, layers=0) == OK and _evict(lib, ptr=None, batch=0) == OK


def _rope(lib, ptr=16, total=5, batch=2, nq=6, nkv=2, d=128, sections=(16, 24, 24), rows=100,
          table_stride=128, nb=4, bs=64, mb=4, dtype=0, qkv_strides=(1280, 1), axes=None):
    kv = _lib.strides(64 * 256, 256, 128, 1)
    return lib.fi_rope_axes_store(ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, total, batch, nq, nkv, d,
                                  len(sections) if axes is None else axes, _lib.strides(*sections), total,
                                  rows, table_stride, nb, bs, mb, _lib.strides(*qkv_strides),
                                  _lib.strides(768, 128, 1), kv, kv, _lib.strides(mb, 1), dtype, None, None)


def test_rope_axes_refusals():
    lib = _lib.load()
    for bad in (dict(total=-1), dict(batch=-1), dict(nq=0), dict(nkv=0), dict(rows=0), dict(dtype=7),
                dict(sections=(16, 24, 25)), dict(sections=(16, 24)), dict(sections=(-1, 65)),
                dict(axes=0), dict(sections=(10, 10, 10, 10, 24)), dict(table_stride=127), dict(ptr=None)):
        assert _rope(lib, **bad) == BAD, bad
    for unsup in (dict(d=64), dict(bs=16), dict(total=(1 << 28) + 1)):
        assert _rope(lib, **unsup) == UNSUPPORTED, unsup
    assert _rope(lib, qkv_strides=(1281, 1)) == ALIGN and _rope(lib, qkv_strides=(1280, 2)) == ALIGN
    assert _rope(lib, ptr=None, total=0) == OK and _rope(lib, ptr=None, batch=0) == OK


def test_python_functions_reject_cpu_tensors_and_types():
    from fast_infer_b200.kernels.attention import attention_mass, paged_chunk_attention
    from fast_infer_b200.kernels.eviction import evict_tokens
    from fast_infer_b200.kernels.rope import rope_axes_store
    q = torch.zeros(3, 6, 128, dtype=torch.float16)
    kv = torch.zeros(4, 64, 2, 128, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged_chunk_attention(q, kv, kv, t, 64, i, i[:1])
    with pytest.raises(ValueError, match="CUDA"):
        attention_mass(q, kv, t, 64, i, i[:1], torch.zeros(3, 6))
    with pytest.raises(ValueError, match="CUDA"):
        evict_tokens(kv[None], kv[None], t, i[:1], torch.zeros(1, 1, 2, 256), 64)
    with pytest.raises(ValueError, match="CUDA"):
        rope_axes_store(torch.zeros(3, 10 * 128, dtype=torch.float16), 6, torch.zeros(9, 128),
                        torch.zeros(9, 128), torch.zeros(1, 3).int(), (64,), kv, kv, t, 64, i, i[:1])
    for f in (paged_chunk_attention, attention_mass):
        with pytest.raises(TypeError):
            f(None, kv, kv, t, 64, i, i[:1])


def test_cache_extend_is_all_or_nothing():
    cache = KVCache(1, 2, 128, 256, 64, torch.device("cpu"), num_blocks=5, dtype=torch.bfloat16)
    assert cache.k.dtype == torch.bfloat16
    cu, ctx = cache.extend([70, 0, 64])
    assert cu.tolist() == [0, 70, 70, 134] and ctx.tolist() == [70, 0, 64]
    assert cu.dtype == ctx.dtype == torch.int32
    assert cache.free_blocks == [3, 4] and cache.block_table.tolist() == \
        [[0, 1, -1, -1], [-1] * 4, [2, -1, -1, -1]]
    for bad, match in (([0, 65, 65], "out of memory"), ([200, 0, 0], "table full")):
        before = (cache._bt.copy(), list(cache.free_blocks), cache.seq_lens.copy())
        with pytest.raises(RuntimeError, match=match):
            cache.extend(bad)
        assert np.array_equal(before[0], cache._bt) and before[1] == cache.free_blocks
        assert np.array_equal(before[2], cache.seq_lens)
    with pytest.raises(ValueError, match="negative"):
        cache.extend([-1])
    _, ctx = cache.extend([58, 1])  # fills the second page; the third sequence is not in this step
    assert ctx.tolist() == [128, 1] and list(cache.seq_lens) == [128, 1, 64]
    with pytest.raises(TypeError):
        KVCache(1, 2, 128, 256, 64, torch.device("cpu"), dtype=torch.float32)


def test_evict_needs_lengths_and_room():
    cache = KVCache(1, 2, 128, 256, 64, torch.device("cpu"), num_blocks=5)
    cache.num_tokens = 10  # the reference's batch-wide counter alone says nothing per sequence
    with pytest.raises(ValueError, match="per-sequence"):
        cache.evict(torch.zeros(1, 1, 2, 256), 8)
    with pytest.raises(ValueError, match="per-sequence"):  # it would write over those 10 tokens
        cache.extend([100])
    cache.reset()
    cache.extend([100])
    with pytest.raises(ValueError, match="holds 64"):
        cache.evict(torch.zeros(1, 1, 2, 64), 8)
    with pytest.raises(ValueError, match="batch larger"):
        cache.evict(torch.zeros(1, 3, 2, 256), 8)


def test_oracle_against_itself():
    """The oracle's parts agree: weights of all rows sum to one a row, lse is what they divide by."""
    from oracle.chunk_oracle import chunk, evict_keep, mass, rope_axes
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(3, 64, 2, 128, generator=g).half() for _ in range(2))
    q = torch.randn(9, 4, 128, generator=g).half()
    table = torch.tensor([[2, 0], [1, -1]]).int()
    cu, ctx = torch.tensor([0, 5, 9]), torch.tensor([100, 60])
    o, lse, absv = chunk(q, k, v, table, cu, ctx, softcap=5.0, window=20, prefix=torch.tensor([3, 0]))
    m = mass(q, k, table, cu, ctx, lse, softcap=5.0, window=20, prefix=torch.tensor([3, 0]))
    assert torch.allclose(m.sum(-1), torch.tensor([[10.0, 10.0], [8.0, 8.0]], dtype=torch.float64))
    assert (o.abs() <= absv + 1e-12).all() and not m[0, :, 3:76].any() and m[0, :, :3].all()
    assert evict_keep([1.0, 3.0, NAN, 2.0, 3.0, -1.0, 0.0], 4, 1, 1) == [0, 1, 4, 6]
    x = torch.randn(3, 2, 128, generator=g)
    ident = rope_axes(x, torch.zeros(2, 3).int(), (30, 34), torch.ones(1, 128), torch.zeros(1, 128))
    assert torch.equal(ident, x.double())
