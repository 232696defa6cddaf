"""GPU tests of the decoding operators behind 2^32 elements: pages at the end of a cache of 9 GB a tensor, and rows of logits 2^32 elements apart."""
import pytest
import torch

from augur_v100_b200 import host, kv
from decode_helpers import Batch, attention_reference, rotary_reference
from test_gpu_kv_append import Step
from test_gpu_token_logprobs import _check

pytestmark = pytest.mark.gpu

LAYER, PAGE, PAGES = (24, 4, 256), 64, (1 << 16) + 900     # a page is 2^16 elements of a tensor


@pytest.fixture(scope="module")
def stream():
    torch.cuda.set_device(0)
    s = host.Stream(0)
    yield s
    s.close()
    torch.cuda.empty_cache()


@pytest.fixture(scope="module")
def cache(stream):
    return kv.KvCache.allocate(stream, 1, PAGES, LAYER[1], PAGE, LAYER[2])


def _move(batch, cache):
    """A batch's pages to the end of the large cache: some below 2^32 elements, most above."""
    first = PAGES - batch.pages - 1
    cache.keys[0, first:first + batch.pages] = batch.k[0]
    cache.values[0, first:first + batch.pages] = batch.v[0]
    batch.table = torch.where(batch.table >= 0, batch.table + first, batch.table)
    batch.k, batch.v, batch.pages = cache.keys, cache.values, PAGES


def test_attention(stream, cache):
    batch = Batch([(30000, 2), (77, 1), (32001, 1)], *LAYER, PAGE, seed=1)
    _move(batch, cache)
    assert int(batch.table.max()) * 2 ** 16 > 2 ** 32
    call = kv.PagedAttention.bind(host.Plan(stream, kv.paged_attention_scratch_bytes(*LAYER, 2)), cache, 0, batch.q, batch.table, batch.lengths, batch.starts, 2)
    call.submit_for_plan()
    stream.synchronize()
    want, bound = attention_reference(batch, 1 / 16)
    assert bool(((call.out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("shape", [[(3, 3), (130, 8)], [(900, 700), (800, 800)]])
def test_cache_write(stream, cache, shape):
    step = Step(shape, LAYER, PAGE, (11, 11, 10), seed=2, norm=True)
    batch = step.batch
    _move(batch, cache)
    first = PAGES - 40
    before = cache.keys[0, :40].view(torch.int16).sum(dtype=torch.int64), cache.values[0, :40].view(torch.int16).sum(dtype=torch.int64)
    call = kv.KvAppend.bind(stream, cache, 0, step.q, step.k, step.v, step.positions, step.frequencies, step.sections, batch.table, batch.lengths, batch.starts,
                            q_norm=step.q_norm, k_norm=step.k_norm)
    call.submit()
    stream.synchronize()
    assert first * 2 ** 16 > 2 ** 32 and int(batch.table.min(dim=1).values.max()) < PAGES
    step.close(call.q_out, rotary_reference(step.q, step.q_norm, step.positions, step.frequencies, step.sections, False, 1e-6))
    k = rotary_reference(step.k, step.k_norm, step.positions, step.frequencies, step.sections, False, 1e-6)
    for s, (length, new) in enumerate(shape):
        at = torch.arange(length - new, length, device="cuda:0")
        page, row = batch.table[s, at // PAGE].long(), slice(int(batch.starts[s]), int(batch.starts[s]) + new)
        step.close(cache.keys[0, page, :, at % PAGE], k[row])
        assert torch.equal(cache.values[0, page, :, at % PAGE], step.v[row])
    # the same places modulo 2^32 elements are as they were
    assert (cache.keys[0, :40].view(torch.int16).sum(dtype=torch.int64), cache.values[0, :40].view(torch.int16).sum(dtype=torch.int64)) == before


def test_page_copies(stream, cache):
    g = torch.Generator(device="cuda:0").manual_seed(3)
    sources, destinations = [5, PAGES - 1, PAGES - 2], [PAGES - 3, 9, PAGES - 4]
    for t in (cache.keys, cache.values):
        t[0, sources + destinations] = torch.randn((6, LAYER[1], PAGE, LAYER[2]), generator=g, device="cuda:0").to(torch.bfloat16)
    torch.cuda.synchronize()
    kv.KvPageCopy.bind(stream, cache).submit(sources, destinations)
    stream.synchronize()
    for t in (cache.keys, cache.values):
        assert torch.equal(t[0, destinations], t[0, sources])


@pytest.mark.parametrize("n", [700, 5000])
def test_log_probabilities(stream, n):
    # rows 2^32 elements apart, the largest stride
    memory = torch.empty((1 << 32) + n, dtype=torch.bfloat16, device="cuda:0")
    x = memory.as_strided((2, n), (1 << 32, 1))
    x.copy_(torch.randn((2, n), generator=torch.Generator(device="cuda:0").manual_seed(n), device="cuda:0") * 3)
    _check(stream, x, torch.tensor([1, n - 1], dtype=torch.int32, device="cuda:0"), 20)
