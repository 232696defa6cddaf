"""GPU tests of the attention of new tokens over a paged cache, against the formula in 64 bits. The bound of every element's error is
derived in `decode_helpers.attention_reference`."""
import pytest
import torch

from augur_v100_b200 import host, kv
from decode_helpers import Batch, attention_reference

pytestmark = pytest.mark.gpu

LAYER = (24, 4, 256)


@pytest.fixture(scope="module")
def stream():
    torch.cuda.set_device(0)
    s = host.Stream(0)
    yield s
    s.close()


def _bind(stream, batch, tokens, scale=None, plan=None, layer=0, q=None, out=None):
    plan = plan or host.Plan(stream, kv.paged_attention_scratch_bytes(batch.query_heads, batch.kv_heads, batch.head_dim, tokens))
    out = torch.full(batch.q.shape, 77.0, dtype=torch.bfloat16, device="cuda:0") if out is None else out
    return kv.PagedAttention.bind(plan, kv.KvCache(batch.k, batch.v), layer, batch.q if q is None else q, batch.table, batch.lengths, batch.starts, tokens,
                                  out, scale)


def _close(got, batch, scale, layer=0, q=None):
    want, bound = attention_reference(batch, scale, layer, q)
    live = ~torch.isnan(want)
    assert bool(((got.double() - want).abs() <= bound)[live].all()), float(((got.double() - want).abs() - bound)[live].max())
    assert bool((got[~live] == 77.0).all())              # rows of no sequence are left as they were


@pytest.mark.parametrize("page_tokens", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("heads", [LAYER, (32, 8, 128), (3, 3, 128), (8, 1, 128), (2, 2, 256)])
def test_lengths_from_one_token_to_a_page_and_beyond(stream, heads, page_tokens):
    lengths = sorted({1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 300, page_tokens - 1, page_tokens, page_tokens + 1})
    batch = Batch([(n, 1) for n in lengths if n], *heads, page_tokens, seed=page_tokens, fill=float("nan"))
    a = _bind(stream, batch, 1)
    a.submit_for_plan()
    stream.synchronize()
    _close(a.out, batch, heads[2] ** -0.5)
    assert a.plan.device_status() == 0


@pytest.mark.parametrize("heads,tokens", [(LAYER, 8), (LAYER, 3), ((64, 8, 128), 8), ((64, 1, 128), 1), ((48, 1, 256), 1), ((5, 5, 128), 8), ((16, 2, 256), 5),
                                          ((8, 1, 128), 8)])
def test_several_new_tokens_and_idle_slots(stream, heads, tokens):
    shape = [(0, 0), (tokens, tokens), (1, 1), (700, tokens), (333, max(tokens - 1, 1)), (0, 0), (129, 1), (5, 0), (tokens + 127, tokens)]
    batch = Batch(shape, *heads, 32, seed=tokens, fill=float("inf"), spare_rows=2)
    a = _bind(stream, batch, tokens)
    a.submit_for_plan()
    stream.synchronize()
    _close(a.out, batch, heads[2] ** -0.5)
    assert a.plan.device_status() == 0


@pytest.mark.parametrize("heads", [LAYER, (8, 1, 128)])
def test_long_caches_and_many_sequences(stream, heads):
    for shape, page in (([(40001, 1)], 64), ([(9000, 2), (1, 1), (20011, 2)], 128), ([(37 * b % 411 + 1, 1) for b in range(300)], 16),
                        ([(5, 1)] * 1024, 16)):
        batch = Batch(shape, *heads, page, seed=len(shape))
        a = _bind(stream, batch, 2)
        a.submit_for_plan()
        stream.synchronize()
        _close(a.out, batch, heads[2] ** -0.5)
        assert a.plan.device_status() == 0


def test_scores_that_grow_along_the_cache(stream):
    # every tile's maximum is far above the one before it, then far below: the running maximum has to follow
    for order in (1, -1):
        batch = Batch([(2000, 1), (700, 4)], *LAYER, 64, seed=5)
        for b, (length, _) in enumerate(batch.shape):
            ramp = torch.linspace(-6, 6, length, device="cuda:0")[:: order] if order == 1 else torch.linspace(6, -6, length, device="cuda:0")
            for i in range(-(-length // 64)):
                part = ramp[i * 64:(i + 1) * 64]
                batch.k[0, batch.table[b, i], :, :len(part)] *= part[None, :, None].to(torch.bfloat16)
        batch.q.abs_()
        batch.k.abs_()
        for b, (length, _) in enumerate(batch.shape):
            sign = torch.where(torch.arange(length, device="cuda:0") * 2 < length, -order, order)
            for i in range(-(-length // 64)):
                part = sign[i * 64:(i + 1) * 64]
                batch.k[0, batch.table[b, i], :, :len(part)] *= part[None, :, None].to(torch.bfloat16)
        a = _bind(stream, batch, 4, scale=0.25)
        a.submit_for_plan()
        stream.synchronize()
        _close(a.out, batch, 0.25)


@pytest.mark.parametrize("scale", [0.0, -0.0625, 1.0])
def test_scales(stream, scale):
    batch = Batch([(500, 3), (77, 1)], *LAYER, 64, seed=9)
    a = _bind(stream, batch, 3, scale=scale)
    a.submit_for_plan()
    stream.synchronize()
    _close(a.out, batch, scale)


def test_a_table_that_does_not_fit_is_survived_and_reported(stream):
    shape = [(100, 1), (200, 1), (90, 2)]
    batch = Batch(shape, *LAYER, 32, seed=3)
    good = _bind(stream, batch, 2)
    good.submit_for_plan()
    stream.synchronize()
    for page in (-1, -2 ** 31, batch.pages, 2 ** 31 - 1):
        table = batch.table.clone()
        batch.table[1, 2] = page                 # 32 of 200 tokens are not there
        a = _bind(stream, batch, 2)
        a.submit_for_plan()
        stream.synchronize()
        assert a.plan.device_status() == 0x401
        assert torch.equal(a.out[0], good.out[0]) and torch.equal(a.out[2:], good.out[2:])
        batch.table = table
        k, v = batch.cached(1)
        there = torch.ones(200, dtype=torch.bool, device="cuda:0")
        there[64:96] = False
        x = batch.q[1].double().reshape(4, 6, 256)
        want = (torch.softmax(torch.einsum("hgd,hjd->hgj", x, k[:, there]) / 16, -1) @ v[:, there]).reshape(24, 256)
        assert float((a.out[1].double() - want).abs().max()) <= 0.02    # three roundings of 2^-8 on values below 1.5
    lengths = batch.lengths.clone()
    batch.lengths[0] = 32 * batch.table.shape[1] + 5    # longer than its table row
    a = _bind(stream, batch, 2)
    a.submit_for_plan()
    stream.synchronize()
    assert a.plan.device_status() == 0x401
    assert torch.equal(a.out[1:], good.out[1:])
    batch.lengths = lengths
    for starts in ([0, 1, 2, 5], [-1, 1, 2, 4], [0, 1, 2, 2 ** 31 - 1], [0, 1, 2, 99]):
        batch.starts = torch.tensor(starts, dtype=torch.int32, device="cuda:0")
        a = _bind(stream, batch, 2)
        a.submit_for_plan()
        stream.synchronize()
        assert a.plan.device_status() == 0x402
        assert torch.equal(a.out[1], good.out[1])
    batch.starts = torch.tensor([0, 1, 2, 4], dtype=torch.int32, device="cuda:0")
    batch.lengths = torch.tensor([-5, 200, 1], dtype=torch.int32, device="cuda:0")     # no token; fewer tokens than rows
    a = _bind(stream, batch, 2)
    a.submit_for_plan()
    stream.synchronize()
    assert bool((a.out[0] == 0).all()) and torch.equal(a.out[1], good.out[1]) and bool((a.out[2] == 0).all())
    page = batch.table[2, 0].long()
    assert torch.equal(a.out[3].reshape(4, 6, 256), batch.v[0, page, :, 0][:, None].expand(4, 6, 256))


def test_replays_streams_and_plans(stream):
    # a captured call answers for what its tensors hold when it is replayed; two plans on two streams do not meet
    batches = [Batch([(3000, 1), (17, 1)], *LAYER, 64, seed=s, spare_pages=60) for s in (1, 2)]
    side = host.Stream(0, torch.cuda.Stream())
    streams = [stream, side]
    calls = [_bind(s, b, 1) for s, b in zip(streams, batches)]
    torch.cuda.synchronize()
    for _ in range(20):
        for call in calls:
            call.submit_for_plan()
    torch.cuda.synchronize()
    for call, batch in zip(calls, batches):
        _close(call.out, batch, 1 / 16)
    first = calls[1].out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side.torch_stream):
        calls[1].submit_for_plan()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(calls[1].out, first)              # the same bits, whatever order the CTAs finish in
    batch = batches[1]
    batch.lengths.copy_(torch.tensor([700, 16], dtype=torch.int32))
    batch.shape = [(700, 1), (16, 1)]
    batch.q.mul_(-1)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    _close(calls[1].out, batch, 1 / 16)
    assert calls[1].plan.device_status() == 0
    del graph, calls
    side.close()


def test_layers_of_one_cache_and_allocations(stream):
    batch = Batch([(100, 1), (200, 1)], 8, 2, 128, 16, seed=4, layers=3)
    plan = host.Plan(stream, kv.paged_attention_scratch_bytes(8, 2, 128, 1))
    calls = [_bind(stream, batch, 1, plan=plan, layer=layer) for layer in range(3)]
    before = host.allocation_snapshot()
    for call in calls:
        call.submit_for_plan()
    stream.synchronize()
    assert host.allocation_snapshot() == before
    for layer, call in enumerate(calls):
        _close(call.out, batch, 128 ** -0.5, layer)
    with pytest.raises(ValueError):
        _bind(stream, batch, 1, plan=plan, layer=3)
    with pytest.raises(host.CudaRuntimeError):
        _bind(stream, batch, 1, plan=host.Plan(stream, 256))          # too small a plan
    with pytest.raises(host.CudaRuntimeError):
        _bind(stream, batch, 1, plan=plan, out=batch.q)                # the output on top of an input
    for bad in (dict(q=batch.q.float()), dict(q=batch.q[:, :, ::2]), dict(out=torch.zeros(1, device="cuda:0"))):
        with pytest.raises(ValueError):
            _bind(stream, batch, 1, plan=plan, **bad)


@pytest.mark.parametrize("heads,tokens", [(LAYER, 1), (LAYER, 3), (LAYER, 8), ((16, 2, 256), 5), ((32, 8, 128), 4), ((64, 8, 128), 8)])
def test_many_tiles_in_every_ring(stream, heads, tokens):
    # spans of dozens of tiles and several pairs each, again and again: every slot of the rings goes round many times while the warps that load run ahead
    shape = [(3400 - 31 * b, tokens) for b in range(36)] + [(5100 + 17 * b, 1) for b in range(6)]
    batch = Batch(shape, *heads, 32, seed=tokens)
    a = _bind(stream, batch, tokens)
    first = None
    for _ in range(12):
        a.out.fill_(77.0)
        torch.cuda.synchronize()
        a.submit_for_plan()
        stream.synchronize()
        if first is None:
            first = a.out.clone()
            _close(first, batch, heads[2] ** -0.5)
        assert torch.equal(a.out, first)
    assert a.plan.device_status() == 0
