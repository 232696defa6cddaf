"""GPU tests of log probabilities, entropy and alternatives behind the head, against 64 bits.

Ids are compared exactly. Bounds, with n logits and sums of positive F32 terms in any order: a term e^d is good to 2^-22 + |d| 2^-24 relative (the
difference d is rounded once, 2^-24 |d|, and scaled to a power of two, once more), a sum of a thread's n / 128 terms at most (there are no longer chains)
adds n / 128 2^-24. ln L is then off by that relative error, and by 2^-23 of itself. x - m - ln L is rounded twice more. The second sum's terms carry
|d| <= spread; entropy = ln L - W / L takes both errors, W's relative to sum |e^d d|."""
import math

import pytest
import torch

from augur_v100_b200 import host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def stream():
    torch.cuda.set_device(0)
    s = host.Stream(0)
    yield s
    s.close()


def _reference(x, k):
    """Everything in 64 bits, one row after the other: log of the total over the maximum, entropy, the order with the lowest index first."""
    x = x.double().cpu()
    order = torch.sort(torch.where(torch.isnan(x), math.inf, x), dim=1, descending=True, stable=True).indices if not torch.isnan(x).any() else None
    top = x.amax(1, keepdim=True)
    below = x - torch.where(top == -math.inf, 0.0, top)
    weight = below.exp()
    total = weight.sum(1, keepdim=True)
    moment = torch.where(weight > 0, weight * below, 0.0).sum(1, keepdim=True)
    return below, total, moment, None if order is None else order[:, :k]


def _check(stream, logits, targets, k, plan=None):
    plan = plan or host.Plan(stream, host.logprobs_scratch_bytes(logits.shape[0], k))
    call = host.TokenLogprobs.bind(plan, logits, targets, k)
    call.submit_for_plan()
    stream.synchronize()
    n = logits.shape[1]
    below, total, moment, order = _reference(logits, k)
    relative = 2.0 ** -22 + n / 128 * 2.0 ** -24 + 110 * 2.0 ** -23           # terms below e^-110 are nothing
    log_total = total.log()
    given = below.gather(1, targets.long().cpu().clamp(0, n - 1)[:, None])
    bound = relative + 2.0 ** -22 * (given.abs() + log_total.abs())
    finite = given.isfinite()
    got, want = call.logprobs.cpu().double()[:, None], given - log_total
    assert bool(((got - want).abs() <= bound)[finite].all()), float((got - want).abs()[finite].max())
    assert torch.equal(got[~finite], want[~finite])
    entropy = (log_total - moment / total)[:, 0]
    bound = (relative * (1 + 3 * (moment / total).abs()) + 2.0 ** -22 * (log_total.abs() + (moment / total).abs()))[:, 0]
    assert bool(((call.entropy.cpu().double() - entropy).abs() <= bound).all())
    assert torch.equal(call.ids.cpu().long(), order)
    best = below.gather(1, order)
    got, want = call.alternative_logprobs.cpu().double(), best - log_total
    finite = best.isfinite()
    bound = relative + 2.0 ** -22 * (best.abs() + log_total.abs())
    assert bool(((got - want).abs() <= bound)[finite].all()) and torch.equal(got[~finite], want[~finite])
    return call


def _logits(rows, n, seed, kind=torch.float32, scale=3.0, stride=0):
    g = torch.Generator(device="cuda:0").manual_seed(seed)
    x = torch.randn((rows, max(stride, n)), generator=g, device="cuda:0") * scale
    return x.to(kind)[:, :n], torch.randint(n, (rows,), generator=g, device="cuda:0", dtype=torch.int32)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 1, 0), (2, 2, 2), (3, 31, 31), (1, 32, 32), (5, 33, 32), (2, 127, 20), (3, 128, 5), (1, 511, 20), (2, 1000, 32), (7, 4096, 20),
                                      (4, 4099, 1), (1, 50257, 20), (8, 32000, 0), (300, 1500, 7), (1000, 64, 3), (1, 248320, 20), (8, 248320, 32), (150, 151936, 20)])
def test_rows_of_all_sizes(stream, rows, n, k, kind):
    _check(stream, *_logits(rows, n, rows + n + k, kind), k)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("stride,offset", [(1003, 0), (1001, 1), (2048, 3)])
def test_strides_and_alignments(stream, stride, offset, kind):
    x, _ = _logits(6, 2048, 5, kind, stride=stride + 1100)
    view = x.reshape(-1)[offset:]
    view = view.as_strided((5, 1000), (stride, 1), view.storage_offset())
    _check(stream, view, torch.arange(5, dtype=torch.int32, device="cuda:0"), 20)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [40, 8192, 100003])
def test_orders_that_are_hard_to_select_from(stream, n, kind):
    ramp = torch.linspace(-4, 4, n, device="cuda:0")
    index = torch.arange(n, device="cuda:0")
    rows = [ramp, ramp.flip(0), torch.zeros(n, device="cuda:0"), torch.where(index % 2 == 0, 0.0, -0.0), torch.full((n,), -3e38, device="cuda:0"),
            (index % 7).float(), torch.where(index % 2048 == 5, 3.0, ramp * 0.1), torch.where(index >= n - 3, 9.0, 0.0), torch.where(index < n // 2, -math.inf, 1.0),
            torch.where(index == n // 3, 0.0, -math.inf), torch.where(index == n - 1, 88.0, -88.0), ramp * 1e4, torch.where(index < 33, -math.inf, ramp)]
    x = torch.stack(rows).to(kind)
    _check(stream, x, torch.full((len(rows),), n - 1, dtype=torch.int32, device="cuda:0"), 32)
    _check(stream, x.flip(1).contiguous(), torch.zeros(len(rows), dtype=torch.int32, device="cuda:0"), 20)


@pytest.mark.parametrize("n", [40, 8192, 100003])
def test_rows_with_nothing_infinities_and_nan(stream, n):
    x, targets = _logits(6, n, 3)
    x = x.clone()
    x[0] = -math.inf
    x[1, n // 2] = math.nan
    x[2, 7] = math.inf
    x[3, 5:9] = math.nan
    targets = torch.tensor([3, 1, 7, 2, -1, n], dtype=torch.int32, device="cuda:0")
    call = host.TokenLogprobs.bind(host.Plan(stream, host.logprobs_scratch_bytes(6, 8)), x, targets, 8)
    call.submit_for_plan()
    stream.synchronize()
    logprobs, entropy, ids, best = (t.cpu() for t in (call.logprobs, call.entropy, call.ids, call.alternative_logprobs))
    assert logprobs[0] == -math.inf and entropy[0] == 0 and ids[0].tolist() == list(range(8)) and bool((best[0] == -math.inf).all())
    for row in (1, 2, 3):
        assert bool(logprobs[row].isnan()) and bool(entropy[row].isnan()) and bool(best[row].isnan().all())
    assert ids[1, 0] == n // 2 and ids[2, 0] == 7 and ids[3, :4].tolist() == [5, 6, 7, 8]
    assert bool(logprobs[4:].isnan().all()) and bool(entropy[4:].isfinite().all())          # no such token
    clean, _ = _logits(6, n, 3)
    _check(stream, clean[4:], torch.tensor([0, n - 1], dtype=torch.int32, device="cuda:0"), 8)


def test_replays_streams_and_repeats(stream):
    side = host.Stream(0, torch.cuda.Stream())
    inputs = [_logits(8, 248320, 11), _logits(8, 248320, 12)]
    calls = [host.TokenLogprobs.bind(host.Plan(s, host.logprobs_scratch_bytes(8, 20)), *i, 20) for s, i in zip((stream, side), inputs)]
    torch.cuda.synchronize()
    results = []
    for _ in range(30):
        for call in calls:
            call.submit_for_plan()
        torch.cuda.synchronize()
        results.append([t.clone() for call in calls for t in (call.logprobs, call.entropy, call.ids, call.alternative_logprobs)])
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))         # the same bits every time
    for call, i in zip(calls, inputs):
        _check(call.plan.stream, *i, 20, call.plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side.torch_stream):
        calls[1].submit_for_plan()
    inputs[1][0].copy_(inputs[0][0])
    inputs[1][1].copy_(inputs[0][1])
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(calls[1].ids, calls[0].ids) and torch.equal(calls[1].logprobs, calls[0].logprobs)
    before = host.allocation_snapshot()
    calls[0].submit_for_plan()
    assert host.allocation_snapshot() == before
    del graph, calls, call
    side.close()


def test_refusals(stream):
    x, targets = _logits(4, 100, 1)
    plan = host.Plan(stream, host.logprobs_scratch_bytes(4, 8))
    for bad in ((x.half(), targets, 4), (x.T, targets, 4), (x, targets.long(), 4), (x, targets[:3], 4), (x, targets, 33), (x, targets, -1), (x, targets.cpu(), 4)):
        with pytest.raises(ValueError):
            host.TokenLogprobs.bind(plan, *bad)
    small, one = _logits(1, 3, 1)
    with pytest.raises(host.CudaRuntimeError):
        host.TokenLogprobs.bind(plan, small, one, 4)                    # more alternatives than tokens
    with pytest.raises(host.CudaRuntimeError):
        host.TokenLogprobs.bind(host.Plan(stream, 256), x, targets, 4)
