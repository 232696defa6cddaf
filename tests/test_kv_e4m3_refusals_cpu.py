"""What the entries of the 8-bit cache and of the shared prefix refuse, before any CUDA call, and the pool's book of shared pages."""
import ctypes
from ctypes import byref

import pytest
import torch
from test_decode_refusals_cpu import INVALID, LAYER_FAULTS, _append, _batch, _change, _layer, stream  # noqa: F401 (a fixture)

from augur_v100_b200 import abi, kv


def _layer8(**changes):
    l = _layer(**changes)
    tokens = l.pages * l.kv_heads * l.page_tokens
    return abi.KvE4m3Layer(l.keys, l.values, 1 << 47, tokens * l.head_dim, tokens * 2, l.pages, l.kv_heads, l.page_tokens, l.head_dim)


def _append8():
    a, b = abi.header(abi.KvAppendE4m3Args), _append()
    for name, _ in abi.KvAppendArgs._fields_[3:]:
        setattr(a, name, getattr(b, name))
    a.layer = _layer8()
    return a


FAULTS = LAYER_FAULTS + [("layer.scales", 0), ("layer.scales", (1 << 47) + 8), ("layer.scales", 1 << 32), ("layer.scales_len_bytes", 8),
                         ("layer.len_bytes", 10 * 4 * 64 * 256 * 2), ("layer.scales_len_bytes", 10 * 4 * 64)]


@pytest.mark.parametrize("path,value", FAULTS + [
    ("query_heads", 0), ("rotary_dim", 0), ("rotary_dim", 72), ("interleaved", 2), ("epsilon", -1.0), ("query_row_stride", 12), ("key", 8), ("value_len_bytes", 2),
    ("positions_len_bytes", 28), ("norm_len_bytes", 1024), ("query_out", 1 << 32), ("query_out", 1 << 47), ("key", 1 << 47), ("reserved", 1), ("struct_size", 312), ("abi_version", 2)])
def test_append_refuses(stream, path, value):  # noqa: F811
    lib, a = abi.lib(), _append8()
    _change(a, path, value)
    for entry in (lib.augur_cuda_nvfp4_sm100_kv_append_e4m3_preflight_v1, lib.augur_cuda_nvfp4_sm100_kv_append_e4m3_prevalidated_submit_v1):
        assert entry(0, stream, byref(a)).status in (INVALID, abi.STATUS_ABI_VERSION_MISMATCH)


def test_append_accepts(stream):  # noqa: F811
    lib, a = abi.lib(), _append8()
    lib.augur_cuda_nvfp4_sm100_diagnostic_inject_submit_fault_v1(1)
    assert lib.augur_cuda_nvfp4_sm100_kv_append_e4m3_prevalidated_submit_v1(0, stream, byref(a)).status == abi.STATUS_DIAGNOSTIC_FAULT_INJECTED


def test_attentions_refuse_without_a_plan(stream):  # noqa: F811
    for name, kind in (("paged_attention_e4m3", abi.PagedAttentionE4m3Args), ("shared_prefix_attention", abi.SharedPrefixAttentionArgs)):
        a = abi.header(kind)
        for step in ("preflight", "prevalidated_submit"):
            entry = getattr(abi.lib(), f"augur_cuda_nvfp4_sm100_{name}_{step}_v1")
            assert entry(0, stream, None, byref(a)).status == INVALID
            assert entry(0, None, None, byref(a)).status == INVALID
            assert entry(0, stream, None, None).status == INVALID


@pytest.mark.parametrize("query_heads,kv_heads,head_dim,rows,tokens,sms,fine", [
    (24, 4, 256, 64, 8, 148, True), (64, 1, 128, 1, 1, 148, True), (8, 8, 128, 1 << 20, 8, 148, True), (24, 4, 256, 0, 1, 148, False), (24, 4, 256, (1 << 20) + 1, 1, 148, False),
    (24, 4, 256, 64, 9, 148, False), (24, 5, 256, 64, 1, 148, False), (65, 1, 128, 64, 1, 148, False), (24, 4, 192, 64, 1, 148, False), (24, 4, 256, 64, 1, 0, False)])
def test_prefix_scratch(query_heads, kv_heads, head_dim, rows, tokens, sms, fine):
    out = ctypes.c_uint64(7)
    entry = abi.lib().augur_cuda_nvfp4_sm100_shared_prefix_attention_scratch_extent_host_v1
    status = entry(query_heads, kv_heads, head_dim, rows, tokens, sms, byref(out)).status
    assert (status == 0) == fine and (out.value > 7) == fine
    assert entry(24, 4, 256, 64, 1, 148, None).status == INVALID


def _copy(stream, changes, submit=True):  # noqa: F811
    lib, a = abi.lib(), abi.header(abi.KvPageCopyE4m3Args)
    a.keys, a.values, a.scales, a.page_bytes, a.scale_page_bytes, a.layers, a.pages = 1 << 32, 1 << 40, 1 << 44, 1 << 14, 1 << 7, 3, 12
    a.len_bytes, a.scales_len_bytes = a.page_bytes * 36, a.scale_page_bytes * 36
    for name, value in changes.items():
        setattr(a, name, value)
    if not submit:
        return lib.augur_cuda_nvfp4_sm100_kv_page_copy_e4m3_preflight_v1(0, stream, byref(a)).status
    lists = [(ctypes.c_uint32 * 1)(i) for i in range(2)]
    return lib.augur_cuda_nvfp4_sm100_kv_page_copy_e4m3_prevalidated_submit_v1(0, stream, byref(a), *lists, 1).status


@pytest.mark.parametrize("changes", [{"keys": 0}, {"values": 1 << 32}, {"scales": 1 << 40}, {"scales": 0}, {"scales": (1 << 44) + 8}, {"page_bytes": 24}, {"scale_page_bytes": 24},
                                     {"scale_page_bytes": 0}, {"scales_len_bytes": 1 << 7}, {"layers": 0}, {"pages": 13}, {"abi_version": 3}, {"struct_size": 48}])
def test_page_copy_refuses(stream, changes):  # noqa: F811
    assert _copy(stream, changes) in (INVALID, abi.STATUS_ABI_VERSION_MISMATCH)
    assert _copy(stream, changes, submit=False) in (INVALID, abi.STATUS_ABI_VERSION_MISMATCH)


def test_page_copy_accepts(stream):  # noqa: F811
    abi.lib().augur_cuda_nvfp4_sm100_diagnostic_inject_submit_fault_v1(1)
    assert _copy(stream, {}) == abi.STATUS_DIAGNOSTIC_FAULT_INJECTED


def test_struct_sizes():
    assert ctypes.sizeof(abi.KvE4m3Layer) == 56 and ctypes.sizeof(abi.KvAppendE4m3Args) == 328 and ctypes.sizeof(abi.PagedAttentionE4m3Args) == 176
    assert ctypes.sizeof(abi.KvPageCopyE4m3Args) == 72 and ctypes.sizeof(abi.SharedPrefixAttentionArgs) == 192


def _codes(*shape):
    return torch.zeros(shape, dtype=torch.float8_e4m3fn)


def test_cache_refuses():
    shape, scales = (2, 5, 4, 16, 128), torch.zeros((2, 5, 4, 16, 2), dtype=torch.uint8).view(torch.float8_e8m0fnu)
    cache = kv.KvCacheE4m3(_codes(*shape), _codes(*shape), scales)
    assert (cache.layers, cache.pages, cache.kv_heads, cache.page_tokens, cache.head_dim) == shape
    args = cache.layer_args(1)
    assert args.scales == scales.data_ptr() + 5 * 4 * 16 * 2 and args.len_bytes == 5 * 4 * 16 * 128 and args.scales_len_bytes == 5 * 4 * 16 * 2
    with pytest.raises(ValueError):
        cache.layer_args(2)
    for keys, values, other in ((_codes(2, 5, 4, 16), _codes(*shape), scales), (_codes(*shape).view(torch.uint8), _codes(*shape), scales),
                                (_codes(*shape), _codes(2, 5, 4, 16, 256), scales), (_codes(*shape), _codes(*shape), scales.view(torch.uint8)),
                                (_codes(*shape), _codes(*shape), scales[..., :1]), (_codes(*shape), _codes(*shape), scales.transpose(2, 3))):
        with pytest.raises(ValueError):
            kv.KvCacheE4m3(keys, values, other)


def test_the_prefix_is_over_a_bf16_cache():
    shape, scales = (1, 5, 4, 16, 128), torch.zeros((1, 5, 4, 16, 2), dtype=torch.uint8).view(torch.float8_e8m0fnu)
    cache = kv.KvCacheE4m3(_codes(*shape), _codes(*shape), scales)
    with pytest.raises(ValueError):
        kv.SharedPrefixAttention(None, cache, 0, *[None] * 6, 1, None, 1.0)
    with pytest.raises(ValueError):
        kv._entries(object(), "kv_append", "KvAppendArgs")


def test_shared_pages_of_the_pool():
    pool = kv.KvPagePool(40, 16)
    assert pool.shared_prefix([]) == [] and pool.shared_prefix([None]) == []
    a = pool.create()
    pool.extend(a, 40)
    assert pool.shared_prefix([a]) == pool.page_list(a)[:2]          # full pages only
    b, _ = pool.fork(a)
    c, _ = pool.fork(a)
    assert pool.shared_prefix([a, None, b, c]) == pool.page_list(a)[:2]
    pool.extend(a, 30)
    pool.extend(b, 30)
    assert pool.shared_prefix([a, b]) == pool.page_list(a)[:2]       # what was written since differs
    pool.truncate(c, 17)
    assert pool.shared_prefix([a, b, c]) == pool.page_list(a)[:1]
    d = pool.create()
    pool.extend(d, 64)
    assert pool.shared_prefix([a, d]) == []
    pool.extend(c, 0)
    pool.free(b)
    moved = pool.compact()
    assert pool.shared_prefix([a, c]) == pool.page_list(c)[:1] and len(moved.sources) == len(moved.destinations)
