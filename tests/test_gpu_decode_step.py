"""The decoding operators as they are used: projections, cache write, attention, output projection, vocabulary head, log probabilities, over several steps
of sequences that a pool forks, rolls back and compacts, enqueued behind one another and replayed from a graph.

Each stage is compared with its formula in 64 bits on the inputs that the stage before it really left, so the bounds are those of the
stages' own tests; the last check is that a graph of a whole step gives the same bits as its calls one by one."""
import numpy as np
import pytest
import torch

from augur_v100_b200 import abi, host, kv, synth
from decode_helpers import attention_reference, rotary_reference

pytestmark = pytest.mark.gpu

HIDDEN, QUERY, KEY, SIZE, PAGE, VOCABULARY, SECTIONS, ROWS = 512, 8, 2, 128, 16, 4096, (16, 24, 24), 8


class Model:
    """One layer's projections and the head on one stream, with the step's fixed tensors (what a captured step needs)."""

    def __init__(self, stream, slots):
        self.stream = stream
        device = torch.device("cuda:0")
        make = lambda name, rows, cols: host.Nvfp4Sm100Linear(stream, rows, cols, *synth.make_weight(11, 5, name, rows, cols))  # noqa: E731
        self.plan = host.Plan(stream, max(host.gemv_scratch_bytes(2 * QUERY * SIZE, HIDDEN), host.gemv_scratch_bytes(HIDDEN, QUERY * SIZE),
                                          kv.paged_attention_scratch_bytes(QUERY, KEY, SIZE), host.logprobs_scratch_bytes(ROWS, 5)) + (1 << 20))
        g = torch.Generator(device=device).manual_seed(3)
        self.x = torch.zeros((ROWS, HIDDEN), dtype=torch.bfloat16, device=device)
        self.table = torch.full((slots, 12), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(slots, dtype=torch.int32, device=device)
        self.starts = torch.zeros(slots + 1, dtype=torch.int32, device=device)
        self.positions = torch.zeros((3, ROWS), dtype=torch.int32, device=device)
        self.targets = torch.zeros(ROWS, dtype=torch.int32, device=device)
        self.frequencies = (1.0e7 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().to(device)
        self.cache = kv.KvCache.allocate(stream, 1, 24, KEY, PAGE, SIZE)
        self.cache.keys.fill_(float("nan"))
        self.cache.values.fill_(float("nan"))
        head = (torch.randn((VOCABULARY, HIDDEN), generator=g, device=device) * 0.05).to(torch.bfloat16)
        self.q = make("q", 2 * QUERY * SIZE, HIDDEN).bind(self.plan, self.x)            # a head's query and its gate side by side
        self.k = make("k", KEY * SIZE, HIDDEN).bind(self.plan, self.x)
        self.v = make("v", KEY * SIZE, HIDDEN).bind(self.plan, self.x)
        query = self.q.out.view(ROWS, QUERY, 2, SIZE)[:, :, 0]
        self.append = kv.KvAppend.bind(stream, self.cache, 0, query, self.k.out.view(ROWS, KEY, SIZE), self.v.out.view(ROWS, KEY, SIZE), self.positions,
                                       self.frequencies, SECTIONS, self.table, self.lengths, self.starts, interleaved=True)
        self.query = query
        self.attention = kv.PagedAttention.bind(self.plan, self.cache, 0, self.append.q_out, self.table, self.lengths, self.starts, tokens=4)
        self.o = make("o", HIDDEN, QUERY * SIZE).bind(self.plan, self.attention.out.view(ROWS, QUERY * SIZE))
        self.hidden = torch.zeros((ROWS, HIDDEN), dtype=torch.float32, device=device)
        self.head = host.Bf16Head.bind(stream, head, self.hidden)
        self.logprobs = host.TokenLogprobs.bind(self.plan, self.head.out, self.targets, 5)

    def submit(self):
        for stage in (self.q, self.k, self.v):
            stage.submit_for_plan()
        self.append.submit()
        self.attention.submit_for_plan()
        self.o.submit_for_plan()
        with torch.cuda.stream(self.stream.torch_stream):
            self.hidden.copy_(self.o.out)
        self.head.submit()
        self.logprobs.submit_for_plan()

    def fill(self, pool, step, seed):
        """A step's inputs: `step` is [(sequence or None, new tokens)], one entry a slot."""
        g = torch.Generator().manual_seed(seed)
        self.shape = [(pool.length(s), n) if s is not None else (0, 0) for s, n in step]
        starts = np.concatenate([[0], np.cumsum([n for _, n in self.shape])])
        self.table.fill_(-1)
        table = pool.table([s for s, _ in step])
        self.table[:, :table.shape[1]] = table.to("cuda:0")
        self.lengths.copy_(torch.tensor([length for length, _ in self.shape], dtype=torch.int32))
        self.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        self.x.copy_((torch.randn((ROWS, HIDDEN), generator=g) * 4).to(torch.bfloat16))
        self.targets.copy_(torch.randint(VOCABULARY, (ROWS,), generator=g, dtype=torch.int32))
        self.positions.copy_(torch.randint(100000, (3, ROWS), generator=g, dtype=torch.int32))
        torch.cuda.synchronize()

    def check(self):
        live = int(self.starts[-1])
        q = rotary_reference(self.query, None, self.positions, self.frequencies, SECTIONS, True, 0.0)
        assert bool(((self.append.q_out.double() - q).abs()[:live] <= 2.0 ** -8 * q.abs()[:live] + 2.0 ** -18 * q.abs().max()).all())
        batch = type("Step", (), dict(shape=self.shape, query_heads=QUERY, kv_heads=KEY, head_dim=SIZE, page_tokens=PAGE, starts=self.starts, q=self.append.q_out))()

        def cached(b, layer):
            length = self.shape[b][0]
            pages = self.table[b, :-(-length // PAGE)].long()
            take = lambda c: c[0, pages].double().transpose(0, 1).reshape(KEY, -1, SIZE)[:, :length]  # noqa: E731
            return take(self.cache.keys), take(self.cache.values)

        batch.cached = cached
        want, bound = attention_reference(batch, SIZE ** -0.5)
        assert bool(((self.attention.out.double() - want).abs() <= bound)[:live].all())
        logits = self.head.out.double()
        logs = torch.log_softmax(logits, -1)
        given = logs.gather(1, self.targets.long()[:, None])[:, 0]
        # F32 sums over 4096 logits below 2^6: log probabilities good to 2^-14 are far inside what their own test asks
        assert float((self.logprobs.logprobs.double() - given).abs().max()) <= 2.0 ** -14
        assert torch.equal(self.logprobs.ids.long(), torch.sort(self.head.out, dim=1, descending=True, stable=True).indices[:, :5])
        assert self.plan.device_status() == 0


def test_steps_forks_and_compaction():
    torch.cuda.set_device(0)
    stream = host.Stream(0, torch.cuda.Stream())
    model = Model(stream, 4)
    pool = kv.KvPagePool(24, PAGE)
    copy = kv.KvPageCopy.bind(stream, model.cache)
    a, b = pool.create(), pool.create()

    def step(entries, seed):
        for s, n in entries:
            if s is not None:
                copy.submit(*pool.extend(s, n))
        model.fill(pool, entries, seed)
        model.submit()
        stream.synchronize()
        model.check()

    for i in range(9):
        step([(a, 4), (None, 0), (b, 1 + i % 4), (None, 0)], i)
    c, copies = pool.fork(a)                       # 36 tokens: the third page is copied, two are shared
    copy.submit(*copies)
    step([(a, 2), (c, 1), (b, 1), (None, 0)], 20)
    pool.truncate(c, 30)                           # back into a page that both hold: the next token goes to a copy of it
    step([(a, 1), (c, 3), (None, 0), (b, 4)], 21)
    keys = model.attention.out.clone()
    pool.free(b)
    copy.submit(*pool.compact())
    assert all(page < pool.pages - pool.free_pages() for s in pool.sequences() for page in pool.page_list(s))
    step([(c, 1), (None, 0), (None, 0), (a, 4)], 22)
    assert not torch.equal(keys, model.attention.out)

    # the same step once more, from a graph: the same bits (its tokens are written to the same places again)
    outputs = lambda: [t.clone() for t in (model.append.q_out, model.attention.out, model.head.out, model.logprobs.logprobs, model.logprobs.ids)]  # noqa: E731
    want = outputs()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream.torch_stream):
        model.submit()
    for t in (model.attention.out, model.head.out, model.logprobs.logprobs):
        t.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    live = int(model.starts[-1])
    got = outputs()
    assert torch.equal(got[1][:live], want[1][:live]) and torch.equal(got[0], want[0])
    # and the next step from the same graph, with other tokens and tables
    for s, n in ((a, 1), (c, 2)):
        copy.submit(*pool.extend(s, n))
    model.fill(pool, [(a, 1), (c, 2), (None, 0), (None, 0)], 23)
    graph.replay()
    torch.cuda.synchronize()
    model.check()
    del graph
    launches = host.launch_count()
    abi.lib().augur_cuda_nvfp4_sm100_diagnostic_inject_submit_fault_v1(1)
    with pytest.raises(host.CudaRuntimeError):
        model.attention.submit_for_plan()
    assert host.launch_count() == launches
