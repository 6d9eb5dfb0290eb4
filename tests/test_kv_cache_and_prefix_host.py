"""Refusals of the K/V cache entry points and of shared-prefix attention: codes returned before anything touches a GPU, and
what the Python face rejects.  Addresses are never dereferenced here."""
import pytest
import torch

import decoding_attention_amd as da
from decoding_attention_amd import _lib

BIG = 1 << 33


def _append(lib, k=16, v=16, ks=(512, 128), vs=(512, 128), kp=16, vp=16, table=16, lens=16, cu=16, tokens=4, batch=2, hk=4,
            d=128, dv=128, page=16, blocks=8, pages=10, kst=None, vst=None, fmt=0, form=0, sk=None, sv=None):
    kst = page * hk * d if kst is None else kst
    vst = page * hk * dv if vst is None else vst
    return lib.da_kv_cache_append(k, v, *ks, *vs, kp, vp, table, lens, cu, tokens, batch, hk, d, dv, page, blocks, pages, kst,
                                  vst, 1, fmt, form, sk, sv, None)


def _read(lib, kp=16, vp=16, k=16, v=16, table=16, lens=16, cu=16, tokens=4, batch=2, hk=4, d=128, dv=128, page=16, blocks=8,
          pages=10, fmt=0, form=0, sk=None, sv=None):
    return lib.da_kv_cache_read(kp, vp, k, v, table, lens, cu, tokens, batch, hk, d, dv, page, blocks, pages, page * hk * d,
                                page * hk * dv, 1, fmt, form, sk, sv, None)


@pytest.mark.parametrize("call", [_append, _read])
def test_cache_calls_refuse(call):
    lib = _lib.load()
    inv, uns = _lib.DA_ERR_INVALID_ARGUMENT, _lib.DA_ERR_UNSUPPORTED
    assert call(lib, kp=None) == inv and b"k_pages" in lib.da_last_error()
    assert call(lib, v=None) == inv and call(lib, vp=None) == inv
    assert call(lib, k=None) == inv
    assert call(lib, table=None) == inv and call(lib, lens=None) == inv
    assert call(lib, d=80, dv=80) == uns and call(lib, d=128, dv=64) == uns
    assert call(lib, v=None, vp=None) == inv  # (V inside K only at (576, 512))
    for page in (0, 3, 48, 1 << 21):
        assert call(lib, page=page) == inv
    assert call(lib, fmt=4) == inv and call(lib, fmt=-1) == inv and call(lib, form=3) == inv
    assert call(lib, fmt=0, form=1, sk=16, sv=16) == uns and call(lib, fmt=1, form=1, sk=16, sv=16) == uns
    assert call(lib, fmt=2, form=1, sk=16) == inv and call(lib, fmt=3, form=2, sk=16, sv=12) == inv
    assert call(lib, fmt=3, form=2, d=96, dv=96, sk=16, sv=16) == uns
    assert call(lib, cu=None) == inv and b"one token per sequence" in lib.da_last_error()
    assert call(lib, kp=8) == inv
    assert call(lib, tokens=BIG) == inv and call(lib, batch=BIG) == inv and call(lib, pages=BIG) == inv
    assert call(lib, hk=0) == inv and call(lib, hk=4096) == inv
    # nothing to do: no launch
    assert call(lib, tokens=0) == _lib.DA_OK and call(lib, tokens=0, batch=0, cu=None) == _lib.DA_OK


def test_cache_strides_and_alignment_refuse():
    lib = _lib.load()
    inv = _lib.DA_ERR_INVALID_ARGUMENT
    assert _append(lib, kst=16 * 4 * 128 - 16) == inv and _append(lib, vst=16 * 4 * 128 + 8) == inv
    assert _append(lib, k=17) == inv and _append(lib, v=33) == inv
    assert _read(lib, k=8) == inv and _read(lib, v=24) == inv


def _prefix(lib, q=16, pk=16, pv=16, plen=64, k=16, v=16, o=16, cu=16, most=8, batch=2, hq=8, hk=4, d=128, dv=128, ws=None, nb=0):
    return lib.da_decoding_attn_shared_prefix(q, pk, pv, plen, k, v, o, cu, most, batch, hq, hk, d, dv, 0, 1, 0.0, None, 0, ws,
                                              nb, None)


def _paged_prefix(lib, q=16, kp=16, vp=16, o=16, ids=16, plen=64, table=16, lens=16, most=80, batch=2, hq=8, hk=4, d=128, dv=128,
                  page=16, blocks=8, ws=None, nb=0):
    return lib.da_decoding_attn_paged_shared_prefix(q, kp, vp, o, ids, plen, table, lens, most, batch, hq, hk, d, dv, page,
                                                    blocks, page * hk * d, page * hk * dv, 0, 1, 0.0, None, 0, ws, nb, None)


@pytest.mark.parametrize("call", [_prefix, _paged_prefix])
def test_prefix_calls_refuse(call):
    lib = _lib.load()
    inv, uns = _lib.DA_ERR_INVALID_ARGUMENT, _lib.DA_ERR_UNSUPPORTED
    assert call(lib, q=None) == inv and call(lib, o=None) == inv and call(lib, q=8) == inv and call(lib, o=8) == inv
    assert call(lib, hq=6) == inv and call(lib, hk=0) == inv and call(lib, hq=0) == inv
    assert call(lib, d=576, dv=512) == uns and call(lib, d=80, dv=80) == uns and call(lib, d=128, dv=64) == uns
    assert call(lib, plen=BIG) == inv and call(lib, most=BIG) == inv and call(lib, batch=BIG) == inv
    assert call(lib, hq=1 << 17, hk=1) == inv and call(lib, batch=1 << 24, hq=32, hk=1) == inv
    assert call(lib, ws=16, nb=64) == _lib.DA_ERR_WORKSPACE
    assert call(lib, ws=24, nb=1 << 30) == inv
    assert call(lib, batch=0) == _lib.DA_OK


def test_prefix_layout_refusals():
    lib = _lib.load()
    inv = _lib.DA_ERR_INVALID_ARGUMENT
    assert _prefix(lib, pk=None) == inv and _prefix(lib, pv=None) == inv and _prefix(lib, cu=None) == inv
    assert _prefix(lib, k=None) == inv and _prefix(lib, plen=0, v=None) == inv and _prefix(lib, pk=24) == inv
    assert _paged_prefix(lib, ids=None) == inv and _paged_prefix(lib, plen=40) == inv
    assert b"multiple of page_size" in lib.da_last_error()
    assert _paged_prefix(lib, kp=None) == inv and _paged_prefix(lib, vp=None) == inv
    assert _paged_prefix(lib, most=129) == inv and _paged_prefix(lib, page=24) == inv


def test_prefix_workspace_covers_both_parts():
    """Partials of the prefix and of the own tokens, (dim + 2) floats for every row and split; hints move the plan, and the size
    that belongs to it is what the call asks for."""
    lib = _lib.load()
    for prefix, own, batch, hq, hk, d in [(1, 0, 1, 8, 8, 64), (4096, 1024, 64, 32, 8, 128), (8192, 128, 33, 32, 1, 256)]:
        row = batch * hq * (d + 2) * 4
        for total in (0, 1, own * batch // 2, own * batch, 1 << 40):
            packed = lib.da_workspace_bytes_shared_prefix(prefix, own, batch, hq, hk, d, d, total, 0)
            paged = lib.da_workspace_bytes_shared_prefix(prefix, prefix + own, batch, hq, hk, d, d,
                                                         total and total + prefix * batch, 16)
            for n in (packed, paged):
                assert row * (2 if own else 1) <= n <= row * 128
    assert lib.da_workspace_bytes_shared_prefix(64, 64, 2, 8, 3, 128, 128, 0, 0) == 0
    assert lib.da_workspace_bytes_shared_prefix(64, 64, 2, 8, 4, 576, 512, 0, 0) == 0
    # without a prefix it is the plain call's
    assert (lib.da_workspace_bytes_shared_prefix(0, 4096, 4, 32, 8, 128, 128, 0, 0) ==
            lib.da_workspace_bytes(4096, 4, 32, 8, 128, 128, 0))


def test_python_face_rejects_cpu_tensors_and_types():
    k = torch.zeros(2, 4, 64, dtype=torch.float16)
    pool = torch.zeros(3, 16, 4, 64, dtype=torch.float16)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        da.kv_cache_append(k, k, pool, pool, table, lens)
    with pytest.raises(RuntimeError, match="FP16 and BF16"):
        da.kv_cache_append(k.float(), k.float(), pool, pool, table, lens)
    with pytest.raises(RuntimeError, match="rows' dtype"):
        da.kv_cache_append(k.bfloat16(), k.bfloat16(), pool, pool, table, lens)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        da.kv_cache_read(pool, pool, table, lens, None, 2, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="FP16 and BF16"):
        da.kv_cache_read(pool, pool, table, lens, None, 2, dtype=torch.float32)
    cu = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        da.decoding_attn_shared_prefix_fwd(k, k, k, k, k, cu, 1, 64, False)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        da.decoding_attn_paged_shared_prefix_fwd(k, pool, pool, table[0], 16, table, lens, 16, 64, False)


def test_prefix_bound_of_zero():
    """Rows come as K and V or not at all, and the workspace for a bound of zero is enough for either."""
    lib = _lib.load()
    inv = _lib.DA_ERR_INVALID_ARGUMENT
    assert _prefix(lib, most=0, k=None) == inv and _prefix(lib, most=0, v=None) == inv
    for prefix in (1, 300, 5000, 16384):
        for batch in (1, 8, 200):
            zero = lib.da_workspace_bytes_shared_prefix(prefix, 0, batch, 32, 8, 128, 128, 0, 0)
            assert zero >= 2 * batch * 32 * 130 * 4
            one = lib.da_workspace_bytes_shared_prefix(prefix, 1, batch, 32, 8, 128, 128, 0, 0)
            assert zero >= one


def test_prefix_calls_refuse_more_work_groups_than_a_launch_has():
    """A grid holds fewer than 2^32 threads, 2^24 - 1 work-groups of 256: a shape beyond that in the sweep or in the merge is
    refused before anything is launched, and the query has no size for it.  (In range: the workspace is what is missing.)"""
    lib = _lib.load()
    inv, small = _lib.DA_ERR_INVALID_ARGUMENT, _lib.DA_ERR_WORKSPACE
    few = dict(ws=16, nb=64)
    # the merge: sixteen rows a work-group at d 64, eight at 128, four at 256, a quarter of them from six partials
    for d, most, rc in [(64, 1 << 23, small), (128, 1 << 23, small), (256, 1 << 23, small), (256, 1 << 27, inv)]:
        for own in (0, 8):
            assert _prefix(lib, batch=most // 32, hq=32, hk=32, d=d, dv=d, most=own, **few) == rc
            assert _paged_prefix(lib, batch=most // 32, hq=32, hk=32, d=d, dv=d, most=64 + own, **few) == rc
    # the sweep: a work-group for every sequence (1024 own tokens of it, KV head)
    assert _prefix(lib, batch=1 << 24, hq=1, hk=1, d=64, dv=64, most=64, **few) == inv
    assert _prefix(lib, batch=1 << 22, hq=1, hk=1, d=64, dv=64, most=8, **few) == small
    assert _prefix(lib, batch=1 << 15, hq=1, hk=1, d=64, dv=64, most=1 << 20, **few) == inv
    size = lib.da_workspace_bytes_shared_prefix
    assert size(64, 8, 1 << 22, 32, 32, 256, 256, 0, 0) == 0 and size(64, 64, 1 << 24, 1, 1, 64, 64, 0, 0) == 0
    assert size(BIG, 8, 2, 8, 4, 128, 128, 0, 0) == 0 and size(64, BIG, 2, 8, 4, 128, 128, 0, 16) == 0
    assert size(64, 8, BIG, 8, 4, 128, 128, 0, 0) == 0 and size(64, 8, 2, 1 << 17, 1, 128, 128, 0, 0) == 0
    assert size(64, 8, 1 << 22, 1, 1, 64, 64, 0, 0) > 0


@pytest.mark.parametrize("call", [_append, _read])
def test_cache_calls_refuse_more_work_groups_than_a_launch_has(call):
    """A token of 64 heads d 256 is a work-group's share."""
    lib = _lib.load()
    assert call(lib, tokens=1 << 24, hk=64, d=256, dv=256) == _lib.DA_ERR_INVALID_ARGUMENT
    assert b"work-groups" in lib.da_last_error()
