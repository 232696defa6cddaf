"""GPU tests of log probabilities of rows that hold a NaN or +infinity and else nothing but -infinity (every token masked, one logit not a number): the
answer is NaN wherever in the row that logit is, and however the row is dealt out."""
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


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("alternatives", [0, 5])
@pytest.mark.parametrize("rows,n", [(700, 40), (64, 1000), (1, 8192), (600, 8192), (1, 100003), (150, 100003), (600, 50000)])
def test_one_logit_that_is_no_number_among_masked_ones(stream, rows, n, alternatives, kind, value):
    # many rows: a CTA has several units of one row; one row: a unit each
    x = torch.full((rows, n), -math.inf, dtype=kind, device="cuda:0")
    places = [(row * 2654435761 % 4294967296) * n >> 32 for row in range(rows)]
    places[:3] = [0, n - 1, n // 2][:rows]
    place = torch.tensor(places, device="cuda:0")
    x.scatter_(1, place[:, None], value)
    plan = host.Plan(stream, host.logprobs_scratch_bytes(rows, alternatives))
    for targets in (place, (place + 1) % n):
        call = host.TokenLogprobs.bind(plan, x, targets.to(torch.int32), alternatives)
        call.submit_for_plan()
        stream.synchronize()
        assert bool(call.logprobs.isnan().all()) and bool(call.entropy.isnan().all()) and bool(call.alternative_logprobs.isnan().all())
        if alternatives:
            assert torch.equal(call.ids[:, 0].long(), place)
            # behind it the lowest indices: all equal
            order = torch.arange(alternatives, device="cuda:0")
            assert torch.equal(call.ids[:, 1:].long(), order[:-1] + (order[:-1] >= place[:, None]))
    assert plan.device_status() == 0


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1000, 8192, 100003])
def test_rows_around_stay_numbers(stream, n, kind):
    g = torch.Generator(device="cuda:0").manual_seed(n)
    x = (torch.randn((300, n), generator=g, device="cuda:0") * 3).to(kind)
    targets = torch.randint(n, (300,), generator=g, device="cuda:0", dtype=torch.int32)
    plan = host.Plan(stream, host.logprobs_scratch_bytes(300, 4))
    call = host.TokenLogprobs.bind(plan, x, targets, 4)
    call.submit_for_plan()
    stream.synchronize()
    results = call.logprobs, call.entropy, call.ids, call.alternative_logprobs
    clean = [t.clone() for t in results]
    bad = torch.arange(0, 300, 7, device="cuda:0")
    x[bad] = -math.inf
    x[bad, (bad * 97) % n] = math.nan
    call.submit_for_plan()
    stream.synchronize()
    good = torch.ones(300, dtype=torch.bool, device="cuda:0")
    good[bad] = False
    assert all(torch.equal(t[good], c[good]) for t, c in zip(results, clean))
    assert all(bool(t[bad].isnan().all()) for t in (call.logprobs, call.entropy, call.alternative_logprobs))
