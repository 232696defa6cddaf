"""GPU tests that every 64-token unit of a split cache counts once: what the spans leave as parts and the join adds up. Contents are chosen so that a part lost,
taken twice or taken from an earlier launch shows in some output, which is checked for the random ones with a span left out."""
import pytest
import torch

from augur_v100_b200 import host, kv
from decode_helpers import BF16_HALF_ULP, Batch

pytestmark = pytest.mark.gpu

UNIT = 64


@pytest.fixture(scope="module")
def stream():
    torch.cuda.set_device(0)
    s = host.Stream(0)
    yield s
    s.close()


class Plain:
    """Sequences [(length, new tokens), ...] over a cache of zeros, in pages dealt out at random."""

    def __init__(self, shape, heads, page, seed=0):
        self.shape, (query, key, size), device = shape, heads, "cuda:0"
        counts = [-(-length // page) for length, _ in shape]
        order = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(seed))
        self.table = torch.full((len(shape), max(counts)), -1, dtype=torch.int32)
        at = 0
        for b, count in enumerate(counts):
            self.table[b, :count] = order[at:at + count].to(torch.int32)
            at += count
        starts = [0]
        for _, new in shape:
            starts.append(starts[-1] + new)
        self.table, self.starts = self.table.to(device), torch.tensor(starts, dtype=torch.int32, device=device)
        self.lengths = torch.tensor([length for length, _ in shape], dtype=torch.int32, device=device)
        cache = (1, sum(counts), key, page, size)
        self.k, self.v = (torch.zeros(cache, dtype=torch.bfloat16, device=device) for _ in range(2))
        self.q = torch.zeros((starts[-1], query, size), dtype=torch.bfloat16, device=device)
        self.page = page

    def rows(self, b):
        """(page, row in the page) of every token of sequence b."""
        position = torch.arange(self.shape[b][0], device="cuda:0")
        return self.table[b, position // self.page].long(), position % self.page

    def bind(self, stream, heads, tokens, scale):
        plan = host.Plan(stream, kv.paged_attention_scratch_bytes(*heads, tokens))
        return kv.PagedAttention.bind(plan, kv.KvCache(self.k, self.v), 0, self.q, self.table, self.lengths, self.starts, tokens, scale=scale)


SPLIT = [((24, 4, 256), [(40001, 1)], 64), ((24, 4, 256), [(20017, 8), (9000, 8), (1, 1), (16385, 8)], 16), ((8, 1, 128), [(40001, 1)], 128),
         ((16, 2, 256), [(30000, 5)], 32), ((64, 8, 128), [(10000, 8), (4097, 3)], 64), ((32, 8, 128), [(131071, 1), (131068, 1)], 128),
         ((24, 4, 256), [(300 + 67 * b, 1 + b % 3) for b in range(40)], 64), ((5, 5, 128), [(129, 8)], 1024)]


@pytest.mark.parametrize("heads,shape,page", SPLIT)
def test_every_unit_counts_once(stream, heads, shape, page):
    # All scores are zero, so every token weighs the same, exactly. Element d of a value is 1 in the units u with u = d + 5 head (mod head size), else 0: an output is
    # the number of such tokens that the row sees over the number of all that it sees. Both sums are whole numbers below 2^24, so what
    # is off is the reciprocal (2^-23), the product (2^-24) and the output's rounding.
    query, key, size = heads
    batch = Plain(shape, heads, page)
    batch.q.normal_(generator=torch.Generator(device="cuda:0").manual_seed(1))
    code = lambda n: ((torch.arange(n, device="cuda:0") // UNIT)[:, None, None] - 5 * torch.arange(key, device="cuda:0")[:, None] - torch.arange(size, device="cuda:0")) % size == 0  # noqa: E731
    for b, (length, _) in enumerate(shape):
        pages, rows = batch.rows(b)
        batch.v[0, pages, :, rows] = code(length).to(torch.bfloat16)
    call = batch.bind(stream, heads, max(new for _, new in shape), None)
    for _ in range(3):
        call.out.fill_(77)
        call.submit_for_plan()
        stream.synchronize()
        for b, (length, new) in enumerate(shape):
            marks = code(length)
            for i in range(new):
                seen = length - new + i + 1
                want = (marks[:seen].sum(0).double() / seen).repeat_interleave(query // key, 0)
                got = call.out[int(batch.starts[b]) + i].double()
                assert bool(((got - want).abs() <= want * (BF16_HALF_ULP + 2.0 ** -21)).all()), (b, i)
    assert call.plan.device_status() == 0


@pytest.mark.parametrize("heads,length,page", [((24, 4, 256), 40001, 64), ((8, 1, 128), 9000, 16), ((32, 8, 128), 65537, 128)])
def test_one_key_of_every_unit_in_turn(stream, heads, length, page):
    # A query's score is 256 at its own key and 0 at all others, which then weigh 2^-369, nothing in F32: the output is that key's value, bit for bit.
    query, key, size = heads
    group = query // key
    batch = Plain([(length, 1)], heads, page)
    batch.v.normal_(generator=torch.Generator(device="cuda:0").manual_seed(2))
    for r in range(group):
        batch.q[0, torch.arange(key) * group + r, r] = 16
    pages, rows = batch.rows(0)
    units = -(-length // UNIT)
    call = batch.bind(stream, heads, 1, 1.0)
    positions = [min(u * UNIT + u * 37 % UNIT, length - 1) for u in range(units)] + [0, length - 1]
    for first in range(0, len(positions), group):
        mine = [positions[(first + r) % len(positions)] for r in range(group)]
        at = pages[mine], rows[mine]
        for r in range(group):
            batch.k[0, at[0][r], :, at[1][r], r] = 16
        call.submit_for_plan()
        want = batch.v[0, at[0], :, at[1]].transpose(0, 1).reshape(query, size)      # [group, key, size] by head
        assert torch.equal(call.out[0], want), first
        batch.k[0, at[0], :, at[1]] = 0
    assert call.plan.device_status() == 0


def _chain_reference(batch, scale, drop=None):
    """(output, bound) of the one row of a batch of one sequence in 64 bits, with the bound's sums by the chains that there are.

    The output is rounded once (2^-8 |o|). The weights' two BF16 terms and the scores' sums: as in `attention_reference`. A sum in F32 runs over the tokens of a span (and
    over a rescaling for each of its 128-token tiles at most), then over the pair's parts, of which each is scaled by a power good to 2^-22; with truncation and in any order
    that is (tokens of a span + tiles + parts + 16) 2^-23 of sum w |v|, in numerator and denominator. `drop`: tokens left out."""
    query, key, size, length = batch.query_heads, batch.kv_heads, batch.head_dim, batch.shape[0][0]
    k, v = batch.cached(0)
    x = batch.q[0].double().reshape(key, query // key, size)
    scores = torch.einsum("hgd,hjd->hgj", x, k) * scale
    if drop is not None:
        scores[..., drop] = -float("inf")
    w = torch.softmax(scores, -1)
    value, spread = torch.einsum("hgj,hjd->hgd", w, v), torch.einsum("hgj,hjd->hgd", w, v.abs())
    size_of = torch.einsum("hgd,hjd->hgj", x.abs(), k.abs()).amax(-1, keepdim=True) * abs(scale)
    span = _span_tokens(length, key)
    chain = span + span / 128 + -(-length // span) + 1 + 16
    relative = 2 * BF16_HALF_ULP ** 2 + 2 * (size_of * size * 2.0 ** -23 + 2.0 ** -22) + 2 * chain * 2.0 ** -23
    bound = BF16_HALF_ULP * value.abs() + relative * spread * (1 + BF16_HALF_ULP)
    return value.reshape(query, size), bound.reshape(query, size)


def _span_tokens(length, key):
    return -(-(-(-length // UNIT) * key) // host.sm_count()) * UNIT


@pytest.mark.parametrize("heads", [(24, 4, 256), (8, 1, 128)])
def test_random_contents_within_the_bound_of_a_span(stream, heads):
    length = 40001
    batch = Batch([(length, 1)], *heads, 64, seed=12)
    plan = host.Plan(stream, kv.paged_attention_scratch_bytes(*heads, 1))
    call = kv.PagedAttention.bind(plan, kv.KvCache(batch.k, batch.v), 0, batch.q, batch.table, batch.lengths, batch.starts, 1)
    call.submit_for_plan()
    stream.synchronize()
    scale = heads[2] ** -0.5
    want, bound = _chain_reference(batch, scale)
    assert bool(((call.out[0].double() - want).abs() <= bound).all()), float(((call.out[0].double() - want).abs() - bound).max())
    # and the bound is one: with any span of the shorter length left out, some output of every key-value head lies outside
    units, spans = -(-length // UNIT) * heads[1], host.sm_count()
    span = units // spans * UNIT
    for first in range(0, length - span, 5 * span):
        without, _ = _chain_reference(batch, scale, slice(first, first + span))
        outside = ((without - want).abs() > bound).reshape(heads[1], -1).any(1)
        assert bool(outside.all()), first
