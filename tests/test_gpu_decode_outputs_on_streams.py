"""The outputs that the decoding owners allocate belong to the stream that they are bound to: what the current stream still has to do when they are bound
(filling an output with zeros, writing to memory that was given back) does not reach them."""
import pytest
import torch

from augur_v100_b200 import host, kv
from decode_helpers import Batch

pytestmark = pytest.mark.gpu

CYCLES = 200_000_000      # a tenth of a second that the current stream lags behind


@pytest.fixture
def side():
    torch.cuda.set_device(0)
    s = host.Stream(0, torch.cuda.Stream())
    yield s
    s.close()


def _lag(*tensors):
    """The current stream waits, then writes to memory that goes back to the allocator at once: tensors of the sizes that come next."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    given_back = [torch.empty_like(t) for t in tensors]
    torch.cuda._sleep(CYCLES)
    for t in given_back:
        t.view(torch.uint8).fill_(0x55)


def test_attention(side):
    batch = Batch([(300, 1), (40, 1)], 24, 4, 256, 64, seed=1)
    plan = host.Plan(side, kv.paged_attention_scratch_bytes(24, 4, 256, 1))
    bind = lambda out: kv.PagedAttention.bind(plan, kv.KvCache(batch.k, batch.v), 0, batch.q, batch.table, batch.lengths, batch.starts, 1, out)  # noqa: E731
    want = torch.zeros_like(batch.q)
    torch.cuda.synchronize()
    bind(want).submit_for_plan()
    side.synchronize()
    want = want.clone()
    _lag(want)
    call = bind(None)
    call.submit_for_plan()
    torch.cuda.synchronize()
    assert torch.equal(call.out, want)


def test_cache_write(side):
    batch = Batch([(30, 2)], 24, 4, 256, 16, seed=2)
    g = torch.Generator(device="cuda:0").manual_seed(2)
    k, v = (torch.randn((2, 4, 256), generator=g, device="cuda:0").to(torch.bfloat16) for _ in range(2))
    positions = torch.randint(1000, (3, 2), generator=g, device="cuda:0", dtype=torch.int32)
    frequencies = torch.rand(32, generator=g, device="cuda:0")
    bind = lambda out: kv.KvAppend.bind(side, kv.KvCache(batch.k, batch.v), 0, batch.q, k, v, positions, frequencies, (11, 11, 10), batch.table,  # noqa: E731
                                        batch.lengths, batch.starts, q_out=out)
    want = torch.zeros_like(batch.q)
    torch.cuda.synchronize()
    bind(want).submit()
    side.synchronize()
    want = want.clone()
    _lag(want)
    call = bind(None)
    call.submit()
    torch.cuda.synchronize()
    assert torch.equal(call.q_out, want)


def test_log_probabilities(side):
    g = torch.Generator(device="cuda:0").manual_seed(3)
    x = torch.randn((8, 5000), generator=g, device="cuda:0")
    targets = torch.randint(5000, (8,), generator=g, device="cuda:0", dtype=torch.int32)
    plan = host.Plan(side, host.logprobs_scratch_bytes(8, 20))
    torch.cuda.synchronize()
    call = host.TokenLogprobs.bind(plan, x, targets, 20)
    call.submit_for_plan()
    torch.cuda.synchronize()
    results = lambda: (call.logprobs, call.entropy, call.ids, call.alternative_logprobs)  # noqa: E731
    want = [t.clone() for t in results()]
    _lag(*want)
    call = host.TokenLogprobs.bind(plan, x, targets, 20)
    call.submit_for_plan()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(results(), want))


def test_cache(side):
    shape = (1, 3, 2, 16, 128)
    _lag(*(torch.empty(shape, dtype=torch.bfloat16, device="cuda:0") for _ in range(2)))
    cache = kv.KvCache.allocate(side, *shape)
    with torch.cuda.stream(side.torch_stream):
        cache.keys.fill_(3)
        cache.values.fill_(4)
    torch.cuda.synchronize()
    assert bool((cache.keys == 3).all()) and bool((cache.values == 4).all())


def test_an_output_that_the_current_stream_still_reads(side):
    # the current stream lags, then copies an output whose owner is gone: the next owner's output lies elsewhere
    batch = Batch([(300, 1), (40, 1)], 24, 4, 256, 64, seed=5)
    plan = host.Plan(side, kv.paged_attention_scratch_bytes(24, 4, 256, 1))
    bind = lambda q: kv.PagedAttention.bind(plan, kv.KvCache(batch.k, batch.v), 0, q, batch.table, batch.lengths, batch.starts)  # noqa: E731
    other = -batch.q
    torch.cuda.synchronize()
    call = bind(batch.q)
    call.submit_for_plan()
    side.synchronize()
    want = call.out.clone()
    torch.cuda.synchronize()
    torch.cuda._sleep(CYCLES)
    got = call.out.clone()
    del call
    second = bind(other)
    second.submit_for_plan()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and not torch.equal(second.out, want)
