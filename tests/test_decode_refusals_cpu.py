"""What the decoding entries refuse, before any CUDA call: descriptors with made-up device addresses, nothing of which is dereferenced."""
import ctypes
from ctypes import byref, c_void_p

import pytest

from augur_v100_b200 import abi

INVALID = abi.STATUS_INVALID_ARGUMENT


@pytest.fixture
def stream():
    handle = c_void_p()
    assert abi.lib().augur_cuda_nvfp4_sm100_stream_adopt_v1(0, None, byref(handle)).status == 0
    yield handle
    abi.lib().augur_cuda_nvfp4_sm100_stream_destroy_v1(handle)


def _layer(pages=10, kv_heads=4, page_tokens=64, head_dim=256):
    return abi.KvLayer(1 << 32, 1 << 33, pages * kv_heads * page_tokens * head_dim * 2, pages, kv_heads, page_tokens, head_dim)


def _batch(sequences=3, table_pages=5, rows=7):
    return abi.KvBatch(1 << 34, sequences * table_pages * 4, 1 << 35, sequences * 4, 1 << 36, (sequences + 1) * 4, sequences, table_pages, rows, 0)


def _append(query_heads=24, rotary=64):
    a = abi.header(abi.KvAppendArgs)
    a.layer, a.batch = _layer(), _batch()
    rows, heads, size = a.batch.rows, a.layer.kv_heads, a.layer.head_dim
    a.query, a.query_row_stride, a.query_head_stride = 1 << 37, 2 * query_heads * size, 2 * size
    a.query_len_bytes = 2 * ((rows - 1) * a.query_row_stride + (query_heads - 1) * a.query_head_stride + size)
    for name, at in (("key", 38), ("value", 39)):
        setattr(a, name, 1 << at)
        setattr(a, name + "_row_stride", heads * size)
        setattr(a, name + "_head_stride", size)
        setattr(a, name + "_len_bytes", 2 * rows * heads * size)
    a.positions, a.positions_len_bytes, a.inv_freq_f32, a.inv_freq_len_bytes = 1 << 40, rows * 12, 1 << 41, rotary * 2
    a.query_out, a.query_out_len_bytes = 1 << 42, rows * query_heads * size * 2
    a.query_heads, a.rotary_dim, a.epsilon = query_heads, rotary, 1e-6
    a.sections[:] = (11, 11, 10)
    return a


def _change(a, path, value):
    *way, last = path.split(".")
    for name in way:
        a = getattr(a, name)
    setattr(a, last, value)


LAYER_FAULTS = [("layer.pages", 0), ("layer.kv_heads", 0), ("layer.page_tokens", 48), ("layer.page_tokens", 8), ("layer.head_dim", 64),
                ("layer.head_dim", 192), ("layer.len_bytes", 5), ("layer.keys", 0), ("layer.keys", (1 << 32) + 8), ("layer.values", 1 << 32),
                ("batch.sequences", 0), ("batch.table_pages", 0), ("batch.table_pages", 6), ("batch.rows", 0), ("batch.rows", 8),
                ("batch.lengths_len_bytes", 8), ("batch.token_starts_len_bytes", 12), ("batch.page_table", 0), ("batch.lengths", 3), ("batch.reserved", 1)]


@pytest.mark.parametrize("path,value", LAYER_FAULTS + [
    ("query_heads", 0), ("query_heads", 25), ("rotary_dim", 0), ("rotary_dim", 72), ("rotary_dim", 272), ("interleaved", 2), ("epsilon", -1.0),
    ("epsilon", float("nan")), ("query_row_stride", 12), ("query_head_stride", 128), ("key_row_stride", 4), ("query_len_bytes", 8), ("key", 8),
    ("value_len_bytes", 2), ("positions_len_bytes", 28), ("positions", 2), ("inv_freq_len_bytes", 4), ("query_norm_f32", 1 << 43),
    ("norm_len_bytes", 1024), ("query_out", 1 << 32), ("query_out", 1 << 37), ("query_out_len_bytes", 2), ("reserved", 1), ("struct_size", 8),
    ("abi_version", 2)])
def test_append_refuses(stream, path, value):
    lib, a = abi.lib(), _append()
    _change(a, path, value)
    for entry in (lib.augur_cuda_nvfp4_sm100_kv_append_preflight_v1, lib.augur_cuda_nvfp4_sm100_kv_append_prevalidated_submit_v1):
        assert entry(0, stream, byref(a)).status in (INVALID, abi.STATUS_ABI_VERSION_MISMATCH)


def test_append_refuses_sections_and_accepts_the_rest(stream):
    lib, a = abi.lib(), _append()
    # a good descriptor passes every check of the submit: what comes back is the injected fault, before any CUDA call
    lib.augur_cuda_nvfp4_sm100_diagnostic_inject_submit_fault_v1(1)
    assert lib.augur_cuda_nvfp4_sm100_kv_append_prevalidated_submit_v1(0, stream, byref(a)).status == abi.STATUS_DIAGNOSTIC_FAULT_INJECTED
    a.sections[:] = (11, 11, 11)
    assert lib.augur_cuda_nvfp4_sm100_kv_append_prevalidated_submit_v1(0, stream, byref(a)).status == INVALID
    a.sections[:] = (0xffffffff, 22, 11)              # adds up to 32 in 32 bits only
    assert lib.augur_cuda_nvfp4_sm100_kv_append_prevalidated_submit_v1(0, stream, byref(a)).status == INVALID
    assert lib.augur_cuda_nvfp4_sm100_kv_append_prevalidated_submit_v1(1, stream, byref(_append())).status == INVALID


def test_attention_refuses_without_a_plan(stream):
    lib, a = abi.lib(), abi.header(abi.PagedAttentionArgs)
    for entry in (lib.augur_cuda_nvfp4_sm100_paged_attention_preflight_v1, lib.augur_cuda_nvfp4_sm100_paged_attention_prevalidated_submit_v1):
        assert entry(0, stream, None, byref(a)).status == INVALID
        assert entry(0, None, None, byref(a)).status == INVALID
        assert entry(0, stream, None, None).status == INVALID


@pytest.mark.parametrize("query_heads,kv_heads,head_dim,tokens,sms,fine", [
    (24, 4, 256, 8, 148, True), (64, 1, 128, 1, 148, True), (64, 8, 128, 8, 148, True), (24, 4, 256, 0, 148, False), (24, 4, 256, 9, 148, False),
    (24, 5, 256, 1, 148, False), (24, 0, 256, 1, 148, False), (0, 4, 256, 1, 148, False), (65, 1, 128, 1, 148, False), (16, 1, 128, 5, 148, False),
    (24, 4, 64, 1, 148, False), (24, 4, 256, 1, 0, False)])
def test_attention_scratch(query_heads, kv_heads, head_dim, tokens, sms, fine):
    out = ctypes.c_uint64(7)
    status = abi.lib().augur_cuda_nvfp4_sm100_paged_attention_scratch_extent_host_v1(query_heads, kv_heads, head_dim, tokens, sms, byref(out)).status
    assert (status == 0) == fine and (out.value > 7) == fine
    assert abi.lib().augur_cuda_nvfp4_sm100_paged_attention_scratch_extent_host_v1(24, 4, 256, 1, 148, None).status == INVALID


def _copy(stream, sources, destinations, count=None, submit=True, **changes):
    lib, a = abi.lib(), abi.header(abi.KvPageCopyArgs)
    a.keys, a.values, a.page_bytes, a.layers, a.pages = 1 << 32, 1 << 40, 1 << 14, 3, 12
    a.len_bytes = a.page_bytes * a.layers * a.pages
    for name, value in changes.items():
        setattr(a, name, value)
    array = lambda v: None if v is None else (ctypes.c_uint32 * max(len(v), 1))(*v)  # noqa: E731
    if not submit:
        return lib.augur_cuda_nvfp4_sm100_kv_page_copy_preflight_v1(0, stream, byref(a)).status
    return lib.augur_cuda_nvfp4_sm100_kv_page_copy_prevalidated_submit_v1(0, stream, byref(a), array(sources), array(destinations),
                                                                        len(sources) if count is None else count).status


@pytest.mark.parametrize("sources,destinations", [([0], [0]), ([0, 1], [2, 2]), ([0, 1], [2, 0]), ([0, 1], [1, 2]), ([12], [0]), ([0], [12]),
                                                  ([0xffffffff], [1]), (list(range(12)) + [0], list(range(13)))])
def test_page_copy_refuses_lists(stream, sources, destinations):
    assert _copy(stream, sources, destinations) == INVALID


@pytest.mark.parametrize("changes", [{"keys": 0}, {"values": 1 << 32}, {"keys": (1 << 32) + 8}, {"page_bytes": 24}, {"page_bytes": 0}, {"layers": 0}, {"pages": 0},
                                     {"pages": 13}, {"len_bytes": 1}, {"layers": 1025}, {"page_bytes": 1 << 60}, {"abi_version": 3}, {"struct_size": 4}])
def test_page_copy_refuses_descriptors(stream, changes):
    assert _copy(stream, [0], [1], **changes) in (INVALID, abi.STATUS_ABI_VERSION_MISMATCH)
    assert _copy(stream, [0], [1], submit=False, **changes) in (INVALID, abi.STATUS_ABI_VERSION_MISMATCH)


def test_page_copy_accepts(stream):
    assert _copy(stream, [], []) == 0                                      # nothing to do, no CUDA call
    assert _copy(stream, None, None, count=0) == 0
    assert _copy(stream, None, [1], count=1) == INVALID
    for lists in (([0], [1]), ([5, 5, 7], [1, 2, 3])):                      # one source may have several destinations
        abi.lib().augur_cuda_nvfp4_sm100_diagnostic_inject_submit_fault_v1(1)
        assert _copy(stream, *lists) == abi.STATUS_DIAGNOSTIC_FAULT_INJECTED


def test_logprobs_refuse_without_a_plan(stream):
    lib, a = abi.lib(), abi.header(abi.TokenLogprobsArgs)
    for entry in (lib.augur_cuda_nvfp4_sm100_token_logprobs_preflight_v1, lib.augur_cuda_nvfp4_sm100_token_logprobs_prevalidated_submit_v1):
        assert entry(0, stream, None, byref(a)).status == INVALID
    out = ctypes.c_uint64()
    for rows, alternatives, sms, fine in ((1, 0, 148, True), (4096, 32, 148, True), (0, 0, 148, False), (1, 33, 148, False), (1, 0, 0, False)):
        status = lib.augur_cuda_nvfp4_sm100_token_logprobs_scratch_extent_host_v1(rows, alternatives, sms, byref(out)).status
        assert (status == 0) == fine


def test_struct_sizes():
    assert ctypes.sizeof(abi.KvLayer) == 40 and ctypes.sizeof(abi.KvBatch) == 64
    assert ctypes.sizeof(abi.KvAppendArgs) == 312 and ctypes.sizeof(abi.PagedAttentionArgs) == 160
    assert ctypes.sizeof(abi.KvPageCopyArgs) == 48 and ctypes.sizeof(abi.TokenLogprobsArgs) == 128
