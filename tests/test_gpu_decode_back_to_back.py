"""GPU tests of decoding calls behind one another on one plan, without a wait between them: each finds its own parts, records and arrivals in the scratch,
not those that the call before left there. All calls have other inputs, and each one's result is that of the call on its own, bit for bit."""
import pytest
import torch

from augur_v100_b200 import host, kv, synth
from decode_helpers import Batch

pytestmark = pytest.mark.gpu

LAYER = (24, 4, 256)


@pytest.fixture(scope="module")
def stream():
    torch.cuda.set_device(0)
    s = host.Stream(0, torch.cuda.Stream())
    yield s
    s.close()


def _alone_and_together(stream, calls, outputs, rounds):
    """`calls`: submits; `outputs`: tensors that each writes."""
    torch.cuda.synchronize()
    want = []
    for submit, tensors in zip(calls, outputs):
        submit()
        stream.synchronize()
        want.append([t.clone() for t in tensors])
    for tensors in outputs:
        for t in tensors:
            t.view(torch.uint8).fill_(0x55)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    for mode in range(2):
        for _ in range(rounds):
            if mode == 0:
                for submit in calls:
                    submit()
            else:
                with torch.cuda.stream(stream.torch_stream):
                    graph.replay()
        torch.cuda.synchronize()
        for tensors, good in zip(outputs, want):
            assert all(torch.equal(t.view(torch.uint8), g.view(torch.uint8)) for t, g in zip(tensors, good))
            for t in tensors:
                t.view(torch.uint8).fill_(0x55)
        torch.cuda.synchronize()
        if mode == 0:
            with torch.cuda.graph(graph, stream=stream.torch_stream):
                for submit in calls:
                    submit()
    del graph


@pytest.mark.parametrize("shape,tokens", [([(4100, 1)], 1), ([(4100, 4), (700, 2)], 8), ([(64 * b + 33, 1) for b in range(60)], 1)])
def test_layers(stream, shape, tokens):
    batch = Batch(shape, *LAYER, 64, seed=1, layers=6)
    plan = host.Plan(stream, kv.paged_attention_scratch_bytes(*LAYER, tokens))
    with torch.cuda.stream(stream.torch_stream):
        calls = [kv.PagedAttention.bind(plan, kv.KvCache(batch.k, batch.v), layer, batch.q, batch.table, batch.lengths, batch.starts, tokens) for layer in range(6)]
    _alone_and_together(stream, [c.submit_for_plan for c in calls], [[c.out] for c in calls], 20)
    assert plan.device_status() == 0


def test_all_operators_on_one_plan(stream):
    # attention of two lengths, log probabilities of two row counts and types, linears of two sizes, in turn on the same scratch
    a, b = Batch([(4100, 1)], *LAYER, 64, seed=2), Batch([(2000, 8), (9000, 3)], *LAYER, 16, seed=3)
    g = torch.Generator(device="cuda:0").manual_seed(4)
    logits = torch.randn((8, 100000), generator=g, device="cuda:0"), torch.randn((61, 50001), generator=g, device="cuda:0").to(torch.bfloat16)
    targets = [torch.randint(50000, (x.shape[0],), generator=g, device="cuda:0", dtype=torch.int32) for x in logits]
    linears = [host.Nvfp4Sm100Linear(stream, rows, cols, *synth.make_weight(3, 1, f"w{rows}", rows, cols)) for rows, cols in ((1024, 5120), (5120, 6144))]
    plan = host.Plan(stream, max(kv.paged_attention_scratch_bytes(*LAYER, 8), host.logprobs_scratch_bytes(61, 20), host.gemv_scratch_bytes(1024, 5120),
                                 host.gemv_scratch_bytes(5120, 6144)) + (1 << 20))
    x = [torch.randn((tokens, cols), generator=g, device="cuda:0").to(torch.bfloat16) for tokens, cols in ((8, 5120), (1, 6144))]
    attention = [kv.PagedAttention.bind(plan, kv.KvCache(t.k, t.v), 0, t.q, t.table, t.lengths, t.starts, n) for t, n in ((a, 1), (b, 8))]
    logprobs = [host.TokenLogprobs.bind(plan, l, t, k) for l, t, k in zip(logits, targets, (20, 5))]
    linear = [w.bind(plan, v) for w, v in zip(linears, x)]
    calls, outputs = [], []
    for i in range(2):
        for call, tensors in ((attention[i], [attention[i].out]), (linear[i], [linear[i].out]),
                              (logprobs[i], [logprobs[i].logprobs, logprobs[i].entropy, logprobs[i].ids, logprobs[i].alternative_logprobs])):
            calls.append(call.submit_for_plan)
            outputs.append(tensors)
    _alone_and_together(stream, calls, outputs, 20)
    assert plan.device_status() == 0
