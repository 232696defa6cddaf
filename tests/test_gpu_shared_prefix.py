"""Attention of sequences that share a prefix against 64-bit references, and beside the paged attention that reads it for each of them."""
import pytest
import torch
from kv8_helpers import PrefixBatch, check, prefix_attention_reference

from augur_v100_b200 import host, kv

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def _bind(batch, tokens, scale=None, stream=None, layer=0):
    stream = stream or host.Stream(0)
    plan = host.Plan(stream, kv.shared_prefix_attention_scratch_bytes(batch.query_heads, batch.kv_heads, batch.head_dim, batch.rows, tokens))
    return plan, kv.SharedPrefixAttention.bind(plan, kv.KvCache(batch.k, batch.v), layer, batch.q, batch.table, batch.lengths, batch.starts, batch.prefix_pages,
                                               batch.prefix_tokens, tokens=tokens, scale=scale)


def _attend(batch, tokens, scale=None, status=0):
    plan, bound = _bind(batch, tokens, scale)
    bound.submit_for_plan()
    torch.cuda.synchronize()
    assert plan.device_status() == status
    return bound.out


def _behind(prefix, shape):
    return [(prefix + length if length else 0, new) for length, new in shape]


SHAPES = {
    "one": (64, [(1, 1)]),
    "two": (1024, [(1, 1), (130, 2)]),
    "idle": (192, [(0, 0), (300, 1), (0, 0), (7, 1), (100, 0), (1, 1)]),
    "ragged": (4032, [(37 * b % 401 + 2, 1 + b % 2) for b in range(50)]),
    "many": (320, [(3 + b % 5, 1) for b in range(300)]),
    "none": (0, [(40, 1), (2, 2), (1, 1)]),
}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("heads,page", [((24, 4, 256), 64), ((6, 1, 256), 16), ((4, 4, 128), 16), ((8, 2, 128), 64), ((16, 1, 128), 32), ((24, 1, 128), 64),
                                        ((32, 2, 256), 32)])
def test_shared_prefix(shape, heads, page):
    prefix, sequences = SHAPES[shape]
    batch = PrefixBatch(_behind(prefix, sequences), *heads, page, prefix, seed=3, spare_rows=2, hide=True, spare_prefix=2, fill=float("nan"))
    check(_attend(batch, 2), *prefix_attention_reference(batch, batch.head_dim ** -0.5))


@pytest.mark.parametrize("heads,tokens", [((24, 4, 256), 8), ((8, 1, 128), 8), ((64, 1, 256), 1), ((64, 1, 128), 1), ((8, 8, 128), 8), ((10, 2, 256), 8), ((9, 3, 128), 7)])
@pytest.mark.parametrize("page", [16, 128, 512])
def test_several_tokens(heads, tokens, page):
    prefix = 1536
    shape = _behind(prefix, [(tokens, tokens), (1000, tokens), (70, max(tokens - 1, 1)), (257, 1), (129, tokens)])
    batch = PrefixBatch(shape, *heads, page, prefix, seed=tokens)
    check(_attend(batch, tokens), *prefix_attention_reference(batch, batch.head_dim ** -0.5))


@pytest.mark.parametrize("head_dim", [128, 256])
def test_sequences_that_end_in_the_prefix(head_dim):
    """A row sees the prefix up to its own token only; (0, 1) and the first row of (1, 2) see nothing."""
    batch = PrefixBatch([(1000, 2), (1, 1), (0, 1), (1, 2), (127, 1), (128, 1), (129, 2), (640, 2), (641, 2), (700, 1)], 12, 2, head_dim, 64, 640, seed=5, spare_rows=1)
    check(_attend(batch, 2), *prefix_attention_reference(batch, head_dim ** -0.5))


@pytest.mark.parametrize("head_dim", [128, 256])
def test_references_that_move(head_dim):
    """Scores that grow along the prefix, so that the running maximum moves often, and by far; the largest are the sequences' own, or the prefix's."""
    batch = PrefixBatch([(3200 + 40 * b, 1) for b in range(30)], 8, 2, head_dim, 32, 3200, seed=9)
    ramp = torch.ones(batch.pages, batch.page_tokens, device=DEVICE)
    for i in range(100):
        ramp[batch.prefix_pages[i].long()] = 2.0 ** (-4 + 9 * i / 100)
    batch.k = (batch.k.float() * ramp[None, :, None, :, None]).to(torch.bfloat16)
    check(_attend(batch, 1), *prefix_attention_reference(batch, batch.head_dim ** -0.5))
    check(_attend(batch, 1, scale=-1.0), *prefix_attention_reference(batch, -1.0))


def test_prefix_in_whole_pages():
    """What the count holds over whole pages is read from the sequences' own pages."""
    batch = PrefixBatch(_behind(256, [(100, 1), (33, 2)]), 24, 4, 256, 64, 256, seed=2)
    want, bound = prefix_attention_reference(batch, 0.0625)
    batch.prefix_tokens.fill_(256 + 63)
    batch.prefix_pages = torch.cat([batch.prefix_pages, torch.full((1,), -1, dtype=torch.int32, device=DEVICE)])
    check(_attend(batch, 2), want, bound)
    # a negative count is no prefix
    batch.table[:, :4] = batch.prefix_pages[:4]
    batch.prefix_tokens.fill_(-5)
    check(_attend(batch, 2), want, bound)


def test_as_the_paged_attention():
    """Far more keys than the tables of the other tests, two layers, against the paged attention over the same pages: both are within 2^-8 of the formula."""
    batch = PrefixBatch(_behind(40000, [(1 + 50 * b % 777, 1) for b in range(70)]), 24, 4, 256, 64, 40000 // 64 * 64, seed=7, layers=2)
    plan, bound = _bind(batch, 1, layer=1)
    bound.submit_for_plan()
    other = host.Plan(host.Stream(0), kv.paged_attention_scratch_bytes(24, 4, 256, 1))
    paged = kv.PagedAttention.bind(other, kv.KvCache(batch.k, batch.v), 1, batch.q, batch.table, batch.lengths, batch.starts)
    paged.submit_for_plan()
    torch.cuda.synchronize()
    assert plan.device_status() == 0 and other.device_status() == 0
    a, b = bound.out.double(), paged.out.double()
    assert float((a - b).norm() / b.norm()) < 2.0 ** -8


def test_not_finite():
    batch = PrefixBatch(_behind(640, [(30, 1), (5, 2), (200, 1), (64, 1)]), 8, 2, 128, 16, 640, seed=6)
    clean = _attend(batch, 2).clone()
    starts = batch.starts.tolist()
    own = batch.table[2, 40 + 3]
    batch.q[starts[0], 5, 2] = float("nan")
    batch.q[starts[1] + 1, 2, 9] = float("inf")
    batch.k[0, own, 1, 2, 7] = float("nan")
    got = _attend(batch, 2)
    want = torch.zeros_like(got, dtype=torch.bool)
    want[starts[0], 5] = want[starts[1] + 1, 2] = want[starts[2], 4:] = True
    assert torch.equal(got.isnan(), want) and torch.equal(got[~want], clean[~want])
    batch.k[0, batch.prefix_pages[17], 0, 5, 1] = float("nan")
    batch.v[0, batch.prefix_pages[3], 1, 15, 100] = float("nan")
    got = _attend(batch, 2)
    want[:, :4] = True
    want[:, 4:, 100] = True
    assert torch.equal(got.isnan(), want) and torch.equal(got[~want], clean[~want])


def test_scores_of_minus_infinity():
    """Keys of -infinity under positive queries weigh nothing; a row all of whose scores are -infinity gets zeros."""
    batch = PrefixBatch(_behind(256, [(9, 1), (70, 1)]), 8, 2, 128, 64, 256, seed=3)
    batch.q = batch.q.abs() + 0.5
    clean = batch.k.clone()
    batch.k[0, batch.prefix_pages[:2].long()] = -float("inf")
    shorter = PrefixBatch.__new__(PrefixBatch)
    shorter.__dict__.update(batch.__dict__)
    shorter.k = clean
    shorter.prefix_pages, shorter.table, shorter.prefix = batch.prefix_pages[2:].contiguous(), batch.table[:, 2:].contiguous(), 128
    shorter.lengths, shorter.prefix_tokens = batch.lengths - 128, batch.prefix_tokens - 128
    shorter.shape = [(length - 128, new) for length, new in batch.shape]
    check(_attend(batch, 1), *prefix_attention_reference(shorter, 128 ** -0.5))
    batch.k.fill_(-float("inf"))
    assert bool((_attend(batch, 1) == 0).all())


def test_bad_contents_are_told():
    batch = PrefixBatch(_behind(256, [(30, 1), (5, 2), (200, 1)]), 8, 2, 128, 16, 256, seed=6)
    good = _attend(batch, 2)

    def told(status):
        out = _attend(batch, 2, status=status)
        assert bool(out.isfinite().all())
        return out

    page = int(batch.prefix_pages[5])
    for bad in (-1, batch.pages, 2 ** 31 - 1):
        batch.prefix_pages[5] = bad
        told(0x401)
    batch.prefix_pages[5] = page
    batch.prefix_tokens.fill_(256 + 16)                # beyond the pages given: counts as those
    assert torch.equal(told(0x401), good)
    batch.prefix_tokens.fill_(2 ** 31 - 1)
    assert torch.equal(told(0x401), good)
    batch.prefix_tokens.fill_(256)
    batch.starts[1] = -4
    told(0x402)
    batch.starts[1] = 1
    held = int(batch.table[0, 17])
    batch.table[0, 17] = batch.pages
    assert torch.equal(told(0x401)[1:], good[1:])
    batch.table[0, 17] = held
    assert torch.equal(told(0), good)


def test_pages_beyond_the_cache_count_as_not_there():
    batch = PrefixBatch(_behind(256, [(30, 1), (64, 1)]), 8, 2, 128, 64, 256, seed=6)
    shorter = PrefixBatch.__new__(PrefixBatch)
    shorter.__dict__.update(batch.__dict__)
    keep = torch.tensor([0, 2, 3], device=DEVICE)
    shorter.prefix_pages, shorter.prefix = batch.prefix_pages[keep].contiguous(), 192
    shorter.table = batch.table[:, 1:].contiguous()
    shorter.shape = [(length - 64, new) for length, new in batch.shape]
    batch.prefix_pages = batch.prefix_pages.clone()
    batch.prefix_pages[1] = batch.pages
    batch.k[0, 0] = batch.k[0, 0]
    check(_attend(batch, 1, status=0x401), *prefix_attention_reference(shorter, 128 ** -0.5))


def test_results_do_not_depend_on_the_run():
    batch = PrefixBatch(_behind(8192, [(3 + 11 * b, 1) for b in range(40)]), 32, 8, 128, 64, 8192, seed=4)
    plan, bound = _bind(batch, 1)
    bound.submit_for_plan()
    first = bound.out.clone()
    for _ in range(10):
        bound.out.zero_()
        bound.submit_for_plan()
        assert torch.equal(bound.out, first)


def test_steps_with_the_pools_forks_in_a_graph():
    """Forks of one prompt, as the pool hands them out: cache write, attention behind the shared pages, replayed with other contents."""
    query, kv_heads, size, page = 12, 2, 256, 32
    stream_of = torch.cuda.Stream()
    with torch.cuda.stream(stream_of):
        stream = host.Stream(0)
        cache = kv.KvCache.allocate(stream, 1, 60, kv_heads, page, size)
        cache.keys.normal_(), cache.values.normal_()
        pool, copy = kv.KvPagePool(60, page), kv.KvPageCopy.bind(stream, cache)
        prompt = pool.create()
        pool.extend(prompt, 10 * page + 7)
        slots = [prompt]
        for _ in range(3):
            twin, copies = pool.fork(prompt)
            slots.append(twin)
            copy.submit(*copies)
        shared = pool.shared_prefix(slots)
        assert len(shared) == 10 and shared == pool.page_list(prompt)[:10]
        prefix_pages, prefix_tokens = torch.tensor(shared, dtype=torch.int32, device=DEVICE), torch.tensor([10 * page], dtype=torch.int32, device=DEVICE)
        table, lengths = torch.full((4, 20), -1, dtype=torch.int32, device=DEVICE), torch.zeros(4, dtype=torch.int32, device=DEVICE)
        starts = torch.arange(5, dtype=torch.int32, device=DEVICE)
        q = torch.zeros((4, query, size), dtype=torch.bfloat16, device=DEVICE)
        k, v = (torch.zeros((4, kv_heads, size), dtype=torch.bfloat16, device=DEVICE) for _ in range(2))
        positions, frequencies = torch.zeros((3, 4), dtype=torch.int32, device=DEVICE), torch.rand(32, device=DEVICE)
        append = kv.KvAppend.bind(stream, cache, 0, q, k, v, positions, frequencies, (32, 0, 0), table, lengths, starts)
        plan = host.Plan(stream, kv.shared_prefix_attention_scratch_bytes(query, kv_heads, size, 4, 1))
        attention = kv.SharedPrefixAttention.bind(plan, cache, 0, append.q_out, table, lengths, starts, prefix_pages, prefix_tokens)
        paged_plan = host.Plan(stream, kv.paged_attention_scratch_bytes(query, kv_heads, size, 1))
        paged = kv.PagedAttention.bind(paged_plan, cache, 0, append.q_out, table, lengths, starts)
        graph = None
        for step in range(30):
            for s in slots:
                copy.submit(*pool.extend(s, 1))
            for x in (q, k, v):
                x.normal_()
            table.copy_(pool.table(slots, 20)), lengths.copy_(torch.tensor([pool.length(s) for s in slots], dtype=torch.int32))
            positions.fill_(step + 327)
            if step == 1:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream_of):
                    append.submit(), attention.submit_for_plan(), paged.submit_for_plan()
            if graph is None:
                append.submit(), attention.submit_for_plan(), paged.submit_for_plan()
            else:
                graph.replay()
            stream.synchronize()
            assert plan.device_status() == 0
            a, b = attention.out.double(), paged.out.double()
            assert float((a - b).norm() / b.norm()) < 2.0 ** -8


def test_two_streams():
    batches = [PrefixBatch(_behind(2048, [(90 + 7 * i, 1), (37, 1), (300, 1)]), 24, 4, 256, 64, 2048, seed=20 + i) for i in range(2)]
    alone = [_attend(b, 1).clone() for b in batches]
    bound = [_bind(b, 1, stream=host.Stream(0, torch.cuda.Stream())) for b in batches]
    torch.cuda.synchronize()
    for _ in range(20):
        for _, x in bound:
            x.submit_for_plan()
    torch.cuda.synchronize()
    for (plan, x), want in zip(bound, alone):
        assert torch.equal(x.out, want) and plan.device_status() == 0


@pytest.mark.parametrize("seed", range(6))
def test_random_batches(seed):
    """Batches of any make-up: how the prefix and the own tokens are cut differs from seed to seed, and some sequences end in the prefix."""
    g = torch.Generator().manual_seed(200 + seed)
    pick = lambda *values: values[int(torch.randint(len(values), (1,), generator=g))]  # noqa: E731
    heads = pick((24, 4, 256), (16, 16, 128), (8, 1, 128), (16, 2, 256), (32, 8, 128), (4, 4, 256))
    tokens = int(torch.randint(1, min(8, 64 // (heads[0] // heads[1])) + 1, (1,), generator=g))
    page, count, longest = pick(16, 32, 64, 128), pick(2, 9, 40, 130), pick(20, 300, 2000)
    prefix = pick(1, 5, 30, 70) * page
    shape = []
    for _ in range(count):
        new = int(torch.randint(0, tokens + 1, (1,), generator=g))
        length = int(torch.randint(prefix // 2, prefix + longest, (1,), generator=g)) if seed % 2 else prefix + int(torch.randint(0, longest, (1,), generator=g)) + new
        shape.append((max(length, new), new))
    batch = PrefixBatch(shape, *heads, page, prefix, seed=seed, spare_rows=1, fill=float("nan"), spare_prefix=seed % 3)
    check(_attend(batch, tokens), *prefix_attention_reference(batch, batch.head_dim ** -0.5))


def test_long_own_tokens():
    batch = PrefixBatch(_behind(128, [(20000, 2), (3, 1), (7777, 1)]), 24, 4, 256, 128, 128, seed=8)
    check(_attend(batch, 2), *prefix_attention_reference(batch, 0.0625))


def test_a_page_more_than_once():
    """The prefix's list may name a page twice."""
    batch = PrefixBatch(_behind(512, [(30, 1), (64, 1)]), 8, 2, 128, 64, 512, seed=6)
    batch.prefix_pages[5] = batch.prefix_pages[2]
    batch.prefix_pages[6] = batch.prefix_pages[2]
    check(_attend(batch, 1), *prefix_attention_reference(batch, 128 ** -0.5))


def test_idle_slots_only():
    batch = PrefixBatch([(0, 0), (300, 0), (256, 0)], 8, 2, 128, 16, 256, spare_rows=3)
    assert bool((_attend(batch, 1) == 0).all())


def test_back_to_back_on_one_plan():
    batches = [PrefixBatch(_behind(640, [(700, 2), (33, 1)]), 24, 4, 256, 64, 640, seed=1), PrefixBatch(_behind(2048, [(400, 8)]), 8, 1, 128, 16, 2048, seed=2),
               PrefixBatch(_behind(96, [(9, 1)] * 150), 16, 16, 128, 32, 96, seed=3)]
    tokens = [2, 8, 1]
    alone = [_attend(b, t).clone() for b, t in zip(batches, tokens)]
    plan = host.Plan(host.Stream(0), max(kv.shared_prefix_attention_scratch_bytes(b.query_heads, b.kv_heads, b.head_dim, b.rows, t) for b, t in zip(batches, tokens)))
    bound = [kv.SharedPrefixAttention.bind(plan, kv.KvCache(b.k, b.v), 0, b.q, b.table, b.lengths, b.starts, b.prefix_pages, b.prefix_tokens, tokens=t)
             for b, t in zip(batches, tokens)]
    for _ in range(10):
        for x in bound:
            x.submit_for_plan()
    torch.cuda.synchronize()
    assert plan.device_status() == 0 and all(torch.equal(x.out, want) for x, want in zip(bound, alone))


def test_offsets_beyond_32_bits():
    """Pages whose elements lie behind 2^32 of the layer."""
    pages, kv_heads, page, size = 4200, 8, 512, 256
    batch = PrefixBatch(_behind(1536, [(700, 2), (1, 1)]), 16, kv_heads, size, page, 1536, seed=8, spare_pages=0)
    cache = kv.KvCache.allocate(host.Stream(0), 1, pages, kv_heads, page, size)
    count = batch.k.shape[1]
    cache.keys[0, -count:], cache.values[0, -count:] = batch.k[0], batch.v[0]
    batch.table = torch.where(batch.table >= 0, batch.table + (pages - count), -1)
    batch.prefix_pages = batch.prefix_pages + (pages - count)
    batch.k, batch.v = cache.keys, cache.values
    check(_attend(batch, 2), *prefix_attention_reference(batch, 0.0625))


def test_refusals():
    batch = PrefixBatch(_behind(256, [(30, 1)]), 8, 2, 128, 64, 256)
    plan = host.Plan(host.Stream(0), kv.shared_prefix_attention_scratch_bytes(8, 2, 128, batch.rows, 1))
    good = dict(plan=plan, cache=kv.KvCache(batch.k, batch.v), layer=0, q=batch.q, table=batch.table, lengths=batch.lengths, starts=batch.starts,
                prefix_pages=batch.prefix_pages, prefix_tokens=batch.prefix_tokens)
    kv.SharedPrefixAttention.bind(**good)
    for change, error in (({"layer": 1}, ValueError), ({"prefix_pages": batch.prefix_pages.long()}, ValueError), ({"prefix_pages": batch.prefix_pages[:0]}, ValueError),
                          ({"prefix_pages": batch.prefix_pages.cpu()}, ValueError), ({"prefix_tokens": batch.starts}, ValueError), ({"out": batch.q}, host.CudaRuntimeError),
                          ({"prefix_tokens": batch.lengths, "lengths": batch.lengths}, host.CudaRuntimeError), ({"tokens": 9}, host.CudaRuntimeError),
                          ({"scale": float("inf")}, host.CudaRuntimeError), ({"plan": host.Plan(host.Stream(0), 1 << 12)}, host.CudaRuntimeError)):
        with pytest.raises(error):
            kv.SharedPrefixAttention.bind(**{**good, **change})


def test_as_many_sequences_as_there_may_be():
    batch = PrefixBatch(_behind(256, [(1 + (37 * b) % 50, int(b % 5 != 3)) for b in range(1024)]), 8, 2, 128, 32, 256, seed=12, hide=True, fill=float("nan"))
    check(_attend(batch, 1), *prefix_attention_reference(batch, 128 ** -0.5))


@pytest.mark.parametrize("head_dim", [128, 256])
def test_a_scale_of_zero(head_dim):
    """Every key weighs the same; some rows end in the prefix."""
    batch = PrefixBatch([(300, 2), (40, 1), (193, 2), (500, 1)], 8, 2, head_dim, 64, 192, seed=13)
    check(_attend(batch, 2, scale=0.0), *prefix_attention_reference(batch, 0.0))


def test_another_prefix_in_a_captured_call():
    """A replay follows the prefix's count and pages, the lengths and the tables."""
    batch = PrefixBatch(_behind(2048, [(100 + 9 * b, 1) for b in range(24)]), 24, 4, 256, 64, 2048, seed=15)
    stream = torch.cuda.Stream()
    plan, bound = _bind(batch, 1, stream=host.Stream(0, stream))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        bound.submit_for_plan()
    pages, table, lengths = batch.prefix_pages.clone(), batch.table.clone(), batch.lengths.clone()
    for prefix in (2048, 640, 64, 0, 1984):
        # the first tokens of the prefix; what is left of it moves to the sequences' own pages
        held = prefix // 64
        batch.prefix, batch.shape = prefix, [(int(n), 1) for n in lengths]
        batch.table.copy_(torch.cat([pages.expand(24, -1), table[:, 32:]], 1))
        batch.prefix_tokens.fill_(prefix)
        want, error = prefix_attention_reference(batch, 0.0625)
        batch.table[:, :held] = -9
        graph.replay()
        torch.cuda.synchronize()
        assert plan.device_status() == 0
        check(bound.out, want, error)
    batch.prefix_pages.copy_(pages.flip(0))
    batch.prefix, batch.shape = 1024, [(int(n) - 1024, 1) for n in lengths]
    batch.prefix_tokens.fill_(1024)
    batch.table[:, 16:-16] = table[:, 32:][:, :batch.table.shape[1] - 32]
    batch.lengths.sub_(1024)
    want, error = prefix_attention_reference(batch, 0.0625)
    graph.replay()
    torch.cuda.synchronize()
    assert plan.device_status() == 0
    check(bound.out, want, error)
