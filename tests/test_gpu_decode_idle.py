"""GPU tests of steps without a live sequence, or with one among many idle slots: nothing is written, nothing reported, and the plan is as good as before."""
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


@pytest.mark.parametrize("slots", [1, 32, 33, 40, 1024])
@pytest.mark.parametrize("length", [0, 70])
def test_idle_slots(stream, slots, length):
    idle = Batch([(length, 0)] * slots, *LAYER, 16, seed=1, spare_rows=2)
    live = Batch([(length, 0)] * (slots - 1) + [(3000, 2)], *LAYER, 16, seed=2)
    plan = host.Plan(stream, kv.paged_attention_scratch_bytes(*LAYER, 2))
    bind = lambda b: kv.PagedAttention.bind(plan, kv.KvCache(b.k, b.v), 0, b.q, b.table, b.lengths, b.starts, 2,  # noqa: E731
                                            torch.full(b.q.shape, 77.0, dtype=torch.bfloat16, device="cuda:0"))
    nothing, something = bind(idle), bind(live)
    want, bound = attention_reference(live, 1 / 16)
    for _ in range(3):
        something.submit_for_plan()
        nothing.submit_for_plan()
    stream.synchronize()
    assert bool((nothing.out == 77.0).all()) and bool(((something.out.double() - want).abs() <= bound).all())
    assert plan.device_status() == 0
    g = torch.Generator(device="cuda:0").manual_seed(3)
    for batch in (idle, live):
        k, v = (torch.randn((batch.rows, 4, 256), generator=g, device="cuda:0").to(torch.bfloat16) for _ in range(2))
        keys, values = batch.k.clone(), batch.v.clone()
        call = kv.KvAppend.bind(stream, kv.KvCache(batch.k, batch.v), 0, batch.q, k, v, torch.zeros((3, batch.rows), dtype=torch.int32, device="cuda:0"),
                                torch.ones(32, device="cuda:0"), (11, 11, 10), batch.table, batch.lengths, batch.starts,
                                q_out=torch.full(batch.q.shape, 77.0, dtype=torch.bfloat16, device="cuda:0"))
        call.submit()
        stream.synchronize()
        if batch is idle:
            assert bool((call.q_out == 77.0).all()) and torch.equal(batch.k, keys) and torch.equal(batch.v, values)
        else:                                    # position 0 turns nothing
            assert torch.equal(call.q_out, batch.q)
            for token in range(2):
                at = 2998 + token
                page = batch.table[slots - 1, at // 16].long()
                assert torch.equal(batch.k[0, page, :, at % 16], k[token]) and torch.equal(batch.v[0, page, :, at % 16], v[token])
