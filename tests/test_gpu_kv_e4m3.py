"""The cache in 8 bits: the quantising cache write, attention over it and its page copies, against 64-bit references."""
import pytest
import torch
from decode_helpers import rotary_reference
from kv8_helpers import BatchE4m3, check, decoded_scales, e4m3_attention_reference

from augur_v100_b200 import host, kv

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def _cache(batch):
    return kv.KvCacheE4m3(batch.k, batch.v, batch.scales)


# ---- the cache write ------------------------------------------------------------------------------

def _append(batch, cache, x, norm, interleaved, rotary, positions, epsilon=1e-6, stream=None):
    sections = (rotary // 2 - 2 * (rotary // 6), rotary // 6, rotary // 6)
    frequencies = (1.0e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float().to(DEVICE)
    bound = kv.KvAppend.bind(stream or host.Stream(0), cache, 0, batch.q, x[0], x[1], positions, frequencies, sections, batch.table, batch.lengths, batch.starts,
                             interleaved=interleaved, q_norm=norm, k_norm=norm, epsilon=epsilon)
    bound.submit()
    return bound, frequencies, sections


def _slots(batch):
    """(row, page, place in it) of every new token."""
    table, starts = batch.table.cpu(), batch.starts.tolist()
    out = []
    for b, (length, new) in enumerate(batch.shape):
        for i in range(new):
            at = length - new + i
            if at >= 0:
                out.append((starts[b] + i, int(table[b, at // batch.page_tokens]), at % batch.page_tokens))
    return [torch.tensor(x, device=DEVICE) for x in zip(*out)]


def _check_codes(codes, scales, x, error):
    """Codes [..., head_dim] and scale bytes [...] of x in 64 bits, itself known to `error`."""
    most = x.abs().amax(-1)
    def exponent(a):                             # the smallest e with a <= 448 * 2^e = 0.875 * 2^(9 + e)
        fraction, e = torch.frexp(a.clamp(min=2.0 ** -100))
        return (e - 9 + (fraction > 0.875).int()).clamp(-60, 60)

    power = scales.double() - 127
    assert bool(((power == exponent(most)) | (power == exponent(most + error)) | (power == exponent(most - error))).all())
    unit = torch.exp2(power)[..., None]
    step = torch.exp2(torch.floor(torch.log2(((x.abs() + error[..., None]) / unit).clamp(min=2.0 ** -6))) - 3) * unit      # between two codes
    assert bool(((codes.double() * unit - x).abs() <= step / 2 * (1 + 2.0 ** -20) + error[..., None]).all())


@pytest.mark.parametrize("heads,shape,page,rotary,norm,interleaved", [
    ((24, 4, 256), [(9, 8)], 64, 64, True, True),
    ((24, 4, 256), [(1, 1), (0, 0), (17, 5), (130, 3)], 16, 256, False, False),
    ((8, 8, 128), [(33, 33), (2, 1)], 32, 128, True, False),
    ((3, 1, 128), [(700, 650), (5, 5)], 128, 16, True, True),          # rows by fours
    ((5, 5, 256), [(2600, 2593)], 1024, 48, False, True),
])
def test_append(heads, shape, page, rotary, norm, interleaved):
    query, kv_heads, size = heads
    batch = BatchE4m3(shape, query, kv_heads, size, page, seed=len(shape) + size, spare_rows=2)
    g = torch.Generator().manual_seed(5)
    k, v = ((torch.randn((batch.rows, kv_heads, size), generator=g) * torch.exp2(torch.randint(-9, 10, (batch.rows, kv_heads, 1), generator=g).float())).to(torch.bfloat16).to(DEVICE)
            for _ in range(2))
    positions = torch.randint(0, 1 << 20, (3, batch.rows), generator=g, dtype=torch.int32).to(DEVICE)
    weight = (1 + 0.1 * torch.randn(size, generator=g)).to(DEVICE) if norm else None
    before = [x.view(torch.uint8).clone() for x in (batch.k, batch.v, batch.scales)]
    bound, frequencies, sections = _append(batch, _cache(batch), (k, v), weight, interleaved, rotary, positions)
    torch.cuda.synchronize()
    row, at, offset = _slots(batch)
    keys = rotary_reference(k, weight, positions, frequencies, sections, interleaved, 1e-6)[row]
    values = v.double()[row]
    # F32: the squares' sum, root and weight, the rotation's two products and a sine good to a few 2^-23
    largest = keys.abs().amax(-1) * 2.0 ** -19
    for x, cache, which, error in ((keys, batch.k, 0, largest), (values, batch.v, 1, largest * 0)):
        codes = cache.view(torch.uint8)[0, at, :, offset].view(torch.float8_e4m3fn)
        _check_codes(codes, batch.scales.view(torch.uint8)[0, at, :, offset, which], x, error)
    # nothing else was written
    for old, new in zip(before, (batch.k, batch.v, batch.scales)):
        new = new.view(torch.uint8).clone()
        old[0, at, :, offset] = 0
        new[0, at, :, offset] = 0
        assert torch.equal(old, new)
    # the queries are those of the BF16 cache's write
    twin = kv.KvCache(torch.zeros(batch.k.shape, dtype=torch.bfloat16, device=DEVICE), torch.zeros(batch.k.shape, dtype=torch.bfloat16, device=DEVICE))
    other = _append(batch, twin, (k, v), weight, interleaved, rotary, positions)[0]
    torch.cuda.synchronize()
    used = torch.arange(int(batch.starts[-1]), device=DEVICE)
    assert torch.equal(bound.q_out[used].view(torch.int16), other.q_out[used].view(torch.int16))


def test_append_values_at_the_borders():
    """Zeros, powers of two at either end of the scales, 448 and just above, halfway cases, NaN and infinities: the codes that the rule gives, bit by bit."""
    size, inf, nan = 128, float("inf"), float("nan")
    rows = [([0.0], 67), ([448.0], 127), ([450.0], 128), ([1.75, -1.0], 119), ([1.7578125], 120), ([2.0 ** -52 * 1.75], 67), ([2.0 ** -70, 2.0 ** -69], 67),
            ([448 * 2.0 ** 60], 187), ([2.0 ** 70, 2.0 ** 69, 2.0 ** 68], 187), ([inf, 448.0, 17.0, 18.0, 19.0], 127), ([nan, -inf, 0.5], 118), ([nan], 67),
            ([448.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 1.0625, 1.1875], 127), ([2.0 ** -130], 67), ([3.0e38], 187)]
    x = torch.zeros((len(rows), 1, size))
    for i, (values, _) in enumerate(rows):
        x[i, 0, :len(values)] = torch.tensor(values)
    x = x.to(torch.bfloat16)
    batch = BatchE4m3([(len(rows), len(rows))], 1, 1, size, 16)
    value = x.to(DEVICE)
    _append(batch, _cache(batch), (value, value), None, False, 16, torch.zeros((3, batch.rows), dtype=torch.int32, device=DEVICE))   # (no turn)
    torch.cuda.synchronize()
    _, at, offset = _slots(batch)
    scales = batch.scales.view(torch.uint8)[0, at, 0, offset].cpu()
    want = torch.tensor([byte for _, byte in rows])
    assert torch.equal(scales[:, 0].long(), want) and torch.equal(scales[:, 1].long(), want)
    scaled = x[:, 0].double() * torch.exp2(127 - want.double())[:, None]
    scaled = torch.where(scaled.abs() <= 448, scaled, nan)
    turned = scaled.clone()
    turned[:, 8:16] = torch.where(x[:, 0, :8].isfinite(), scaled[:, 8:16], nan)      # an infinity's partner gets 0 times infinity
    for cache, codes in ((batch.k, turned.float().to(torch.float8_e4m3fn)), (batch.v, scaled.float().to(torch.float8_e4m3fn))):
        got = cache.view(torch.uint8)[0, at, 0, offset].view(torch.float8_e4m3fn).float().cpu()
        assert torch.equal(got.isnan(), codes.float().isnan()) and torch.equal(got[~got.isnan()], codes.float()[~got.isnan()])


def test_append_leaves_what_has_no_page():
    batch = BatchE4m3([(40, 3), (2, 4), (20, 2)], 4, 2, 128, 16, spare_rows=3)
    batch.table[0, 2] = batch.pages + 5          # of the first sequence's tokens 37..39
    batch.table[2, 1] = -1
    before = [x.view(torch.uint8).clone() for x in (batch.k, batch.v, batch.scales)]
    x = torch.randn((batch.rows, 2, 128), device=DEVICE).to(torch.bfloat16)
    _append(batch, _cache(batch), (x, x), None, False, 64, torch.zeros((3, batch.rows), dtype=torch.int32, device=DEVICE))
    torch.cuda.synchronize()
    changed = (before[2] != batch.scales.view(torch.uint8)).any(-1)[0].any(1)      # [pages, tokens]
    allowed = torch.zeros_like(changed)
    allowed[int(batch.table[1, 0]), :2] = True   # two of the four rows lie before the cache's first token
    assert not bool((changed & ~allowed).any())
    assert bool((before[0] == batch.k.view(torch.uint8))[0].transpose(1, 2)[~allowed].all())


# ---- attention --------------------------------------------------------------------------------------

def _attend(batch, tokens, scale=None, stream=None, plan=None, layer=0):
    plan = plan or host.Plan(stream or host.Stream(0), kv.paged_attention_scratch_bytes(batch.query_heads, batch.kv_heads, batch.head_dim, tokens))
    bound = kv.PagedAttention.bind(plan, _cache(batch), layer, batch.q, batch.table, batch.lengths, batch.starts, tokens=tokens, scale=scale)
    bound.submit_for_plan()
    torch.cuda.synchronize()
    assert plan.device_status() == 0
    return bound.out


SHAPES = {
    "one": [(1, 1)],
    "short": [(2, 2), (1, 1), (5, 2)],
    "tile_ends": [(127, 1), (128, 1), (129, 1), (64, 1), (65, 1), (63, 1), (256, 1), (257, 1), (15, 1), (16, 1), (17, 1)],
    "idle": [(0, 0), (300, 1), (0, 0), (7, 1), (100, 0)],
    "sees_nothing": [(0, 1), (1, 2), (200, 1)],
    "ragged": [(37 * b + 5, 1 + b % 2) for b in range(40)],
    "long": [(20000, 1), (3, 2), (12345, 2)],
}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("heads,page", [((24, 4, 256), 64), ((6, 1, 256), 16), ((4, 4, 128), 128), ((8, 2, 128), 16), ((16, 1, 128), 32), ((24, 1, 128), 1024),
                                        ((32, 2, 256), 256)])
def test_attention(shape, heads, page):
    batch = BatchE4m3(SHAPES[shape], *heads, page, seed=3, spare_rows=2, fill=0x7f)
    check(_attend(batch, 2), *e4m3_attention_reference(batch, batch.head_dim ** -0.5))


@pytest.mark.parametrize("heads,tokens", [((24, 4, 256), 8), ((8, 1, 128), 8), ((64, 1, 256), 1), ((64, 1, 128), 1), ((8, 8, 128), 8), ((10, 2, 256), 8), ((9, 3, 128), 7),
                                          ((40, 1, 256), 1), ((36, 1, 128), 1)])
def test_attention_of_several_tokens(heads, tokens):
    shape = [(tokens, tokens), (1000, tokens), (70, max(tokens - 1, 1)), (4097, 1), (129, tokens)]
    batch = BatchE4m3(shape, *heads, 64, seed=tokens)
    check(_attend(batch, tokens), *e4m3_attention_reference(batch, batch.head_dim ** -0.5))


@pytest.mark.parametrize("head_dim", [128, 256])
def test_references_that_move(head_dim):
    """Scores that grow along the sequence, so that the running maximum moves often, and by far."""
    batch = BatchE4m3([(3000, 2), (700, 1)], 8, 2, head_dim, 32, seed=9)
    ramp = torch.zeros((batch.pages, batch.page_tokens), dtype=torch.long)
    table = batch.table.cpu()
    for b, (length, _) in enumerate(batch.shape):
        for j in range(length):
            ramp[table[b, j // 32], j % 32] = j * (6 if b == 0 else 9) // length
    scales = batch.scales.view(torch.uint8).clone()
    scales[0, :, :, :, 0] = (118 + ramp).to(torch.uint8).to(DEVICE)[:, None]
    batch.scales = scales.view(torch.float8_e8m0fnu)
    check(_attend(batch, 2), *e4m3_attention_reference(batch, batch.head_dim ** -0.5))


@pytest.mark.parametrize("head_dim", [128, 256])
def test_value_scales_far_apart(head_dim):
    """Values whose scales lie 2^40 apart: the weight that counts is that of the product."""
    batch = BatchE4m3([(500, 1), (4000, 2), (129, 1)], 12, 2, head_dim, 16, seed=11)
    g = torch.Generator().manual_seed(1)
    scales = batch.scales.view(torch.uint8).clone()
    scales[..., 1] = torch.randint(100, 141, scales.shape[:-1], generator=g, dtype=torch.uint8).to(DEVICE)
    scales[:, :, :, ::7, 1] = 67
    scales[:, :, 0, ::5, 1] = 3                       # counts as 67
    scales[:, :, 1, 3, 1] = 200                       # counts as 187
    batch.scales = scales.view(torch.float8_e8m0fnu)
    check(_attend(batch, 2), *e4m3_attention_reference(batch, batch.head_dim ** -0.5))


@pytest.mark.parametrize("amplitude", [2.0 ** -30, 1.0, 2.0 ** 20])
def test_query_sizes(amplitude):
    batch = BatchE4m3([(777, 2)], 12, 4, 256, 64, seed=4)
    batch.q = (batch.q.float() * torch.exp2(-torch.arange(12, device=DEVICE).float())[:, None] * amplitude).to(torch.bfloat16)
    batch.q[1, 3] = 0
    batch.q[0, 5, 17] = 3.0 * amplitude                # one element far above the others
    scale = 0.05 / amplitude
    check(_attend(batch, 2, scale=scale), *e4m3_attention_reference(batch, scale))
    assert float(_attend(batch, 2, scale=-scale).abs().max()) > 0
    check(_attend(batch, 2, scale=-scale), *e4m3_attention_reference(batch, -scale))


def test_not_finite():
    """A NaN key, value, scale or query element gives NaN in the rows that see it and nowhere else; an infinite query element likewise."""
    shape = [(300, 1), (5, 2), (400, 1), (130, 1), (140, 1), (2000, 1), (90, 1), (33, 1)]
    batch = BatchE4m3(shape, 8, 2, 128, 16, seed=6)
    clean = _attend(batch, 2).clone()
    starts = batch.starts.tolist()
    slot = lambda b, j: (0, int(batch.table[b, j // 16]), slice(None), j % 16)  # noqa: E731
    k, v, s = (x.view(torch.uint8) for x in (batch.k, batch.v, batch.scales))
    k[slot(0, 7)][0, 3] = 0x7f                         # sequence 0, head 0: all outputs
    v[slot(1, 4)][1, 9] = 0xff                         # the last token of sequence 1: its second row, and it may reach the first
    s[slot(2, 399)][0, 0] = 255
    s[slot(3, 0)][1, 1] = 255
    batch.q[starts[4], 5, 2] = float("nan")
    batch.q[starts[5], 1, 0] = float("inf")
    batch.q[starts[6], 1, 0] = -float("inf")
    got = _attend(batch, 2)
    nan = got.isnan()
    want = torch.zeros_like(nan)
    want[starts[0], :4] = True
    want[starts[1] + 1, 4:, 9] = True
    want[starts[2], :4] = True
    want[starts[3], 4:] = True
    want[starts[4], 5] = True
    want[starts[5], 1] = True
    want[starts[6], 1] = True
    maybe = torch.zeros_like(nan)
    maybe[starts[1], 4:, 9] = True
    assert bool((nan == want)[~maybe].all())
    assert torch.equal(got[~want & ~maybe], clean[~want & ~maybe])


def test_bad_contents_are_told():
    batch = BatchE4m3([(300, 1), (40, 1), (100, 1)], 8, 2, 128, 16, seed=6)
    good = _attend(batch, 2)

    def told(status):
        plan = host.Plan(host.Stream(0), kv.paged_attention_scratch_bytes(8, 2, 128, 2))
        bound = kv.PagedAttention.bind(plan, _cache(batch), 0, batch.q, batch.table, batch.lengths, batch.starts, tokens=2)
        bound.submit_for_plan()
        assert plan.device_status() == status and bool(bound.out.isfinite().all())
        return bound.out

    for bad in (-1, batch.pages, 2 ** 31 - 1):
        batch.table[1, 1] = bad
        out = told(0x401)
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    batch.table[1, 1] = 0
    batch.lengths[2] = 16 * batch.table.shape[1] + 1
    told(0x401)
    batch.lengths[2] = -3
    assert bool((told(0)[2] == 0).all())
    batch.lengths[2] = 100
    for place, bad in ((3, 7), (3, 5), (3, -1), (1, -4)):
        held = int(batch.starts[place])
        batch.starts[place] = bad
        told(0x402)
        batch.starts[place] = held
    out = told(0)
    assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])


def test_offsets_beyond_32_bits():
    """Codes behind 2^32 of a layer, in a second layer."""
    pages, kv_heads, page, size = 4200, 8, 512, 256      # 4.4e9 bytes a layer
    batch = BatchE4m3([(1500, 1), (700, 2)], 16, kv_heads, size, page, seed=8, spare_pages=0)
    small_k, small_v, small_s = batch.k, batch.v, batch.scales
    cache = kv.KvCacheE4m3.allocate(host.Stream(0), 1, pages, kv_heads, page, size)
    count = small_k.shape[1]
    for big, little in ((cache.keys, small_k), (cache.values, small_v), (cache.scales, small_s)):
        big.view(torch.uint8)[0, -count:] = little.view(torch.uint8)[0]
    batch.table = torch.where(batch.table >= 0, batch.table + (pages - count), -1)
    want = e4m3_attention_reference
    plan = host.Plan(host.Stream(0), kv.paged_attention_scratch_bytes(16, kv_heads, size, 2))
    bound = kv.PagedAttention.bind(plan, cache, 0, batch.q, batch.table, batch.lengths, batch.starts, tokens=2)
    bound.submit_for_plan()
    torch.cuda.synchronize()
    assert plan.device_status() == 0
    batch.k, batch.v, batch.scales = cache.keys, cache.values, cache.scales
    check(bound.out, *want(batch, size ** -0.5))
    # and written there
    x = torch.randn((batch.rows, kv_heads, size), device=DEVICE).to(torch.bfloat16)
    _append(batch, cache, (x, x), None, False, 64, torch.zeros((3, batch.rows), dtype=torch.int32, device=DEVICE))
    torch.cuda.synchronize()
    row, at, offset = _slots(batch)
    _check_codes(cache.values.view(torch.uint8)[0, at, :, offset].view(torch.float8_e4m3fn), cache.scales.view(torch.uint8)[0, at, :, offset, 1], x.double()[row],
                 torch.zeros((len(row), kv_heads), dtype=torch.float64, device=DEVICE))


# ---- page copies -------------------------------------------------------------------------------------

@pytest.mark.parametrize("layers,pages,kv_heads,page,size,pairs", [(1, 2, 1, 16, 128, 1), (3, 40, 4, 64, 256, 13), (2, 2500, 1, 16, 128, 1100), (1, 5, 8, 1024, 256, 2)])
def test_page_copy(layers, pages, kv_heads, page, size, pairs):
    g = torch.Generator().manual_seed(pages)
    cache = kv.KvCacheE4m3.allocate(host.Stream(0), layers, pages, kv_heads, page, size)
    want = []
    order = torch.randperm(pages, generator=g).tolist()
    sources, destinations = order[:pairs], order[pairs:2 * pairs]
    for x in (cache.keys, cache.values, cache.scales):
        x.view(torch.uint8).copy_(torch.randint(0, 256, x.shape, generator=g, dtype=torch.uint8))
        w = x.view(torch.uint8).clone()
        w[:, destinations] = w[:, sources]
        want.append(w)
    kv.KvPageCopy.bind(host.Stream(0), cache).submit(sources, destinations)
    torch.cuda.synchronize()
    for x, w in zip((cache.keys, cache.values, cache.scales), want):
        assert torch.equal(x.view(torch.uint8), w)


# ---- as they are used together -----------------------------------------------------------------------

def test_decoding_steps_with_a_fork_and_a_graph():
    """Steps of two sequences and a fork: cache write, attention, page copies, the later steps as replays of one captured graph."""
    query, kv_heads, size, page, layers = 12, 2, 128, 16, 2
    device, stream_of = torch.device(DEVICE), torch.cuda.Stream()
    with torch.cuda.stream(stream_of):
        stream = host.Stream(0)
        cache = kv.KvCacheE4m3.allocate(stream, layers, 24, kv_heads, page, size)
        for x in (cache.keys, cache.values, cache.scales):
            x.view(torch.uint8).fill_(0x7f)
        pool, copy = kv.KvPagePool(24, page), kv.KvPageCopy.bind(stream, cache)
        slots = [pool.create(), pool.create(), None]
        tables = torch.full((3, 6), -1, dtype=torch.int32, device=device)
        lengths, starts = torch.zeros(3, dtype=torch.int32, device=device), torch.zeros(4, dtype=torch.int32, device=device)
        q = torch.zeros((3, query, 2, size), dtype=torch.bfloat16, device=device)
        k, v = (torch.zeros((3, kv_heads, size), dtype=torch.bfloat16, device=device) for _ in range(2))
        positions = torch.zeros((3, 3), dtype=torch.int32, device=device)
        frequencies = (1.0e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float().to(device)
        plan = host.Plan(stream, kv.paged_attention_scratch_bytes(query, kv_heads, size, 1))
        steps = []
        for layer in range(layers):
            append = kv.KvAppend.bind(stream, cache, layer, q[:, :, 0], k, v, positions, frequencies, (12, 10, 10), tables, lengths, starts, interleaved=True)
            steps.append((append, kv.PagedAttention.bind(plan, cache, layer, append.q_out, tables, lengths, starts)))
        history = {}                            # by sequence: the keys and values as the cache must hold them, in 64 bits
        g, graph = torch.Generator().manual_seed(2), None
        for step in range(40):
            if step == 21:
                twin, copies = pool.fork(slots[0])
                slots[2] = twin
                history[twin] = list(history[slots[0]])
                copy.submit(*copies)
            live = [s for s in slots if s is not None]
            for s in live:
                copies = pool.extend(s, 1)
                copy.submit(*copies)
            fresh = lambda *shape: torch.randn(shape, generator=g).to(torch.bfloat16)  # noqa: E731
            q.copy_(fresh(3, query, 2, size)), k.copy_(fresh(3, kv_heads, size)), v.copy_(fresh(3, kv_heads, size))
            tables.copy_(pool.table(slots, 6))
            lengths.copy_(torch.tensor([0 if s is None else pool.length(s) for s in slots], dtype=torch.int32))
            starts.copy_(torch.tensor([0, *torch.tensor([s is not None for s in slots]).long().cumsum(0).tolist()], dtype=torch.int32))
            positions[:, :len(live)] = torch.tensor([pool.length(s) - 1 for s in live], dtype=torch.int32, device=device)
            if step == 22:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream_of):
                    for append, attention in steps:
                        append.submit()
                        attention.submit_for_plan()
            if graph is None:
                for append, attention in steps:
                    append.submit()
                    attention.submit_for_plan()
            else:
                graph.replay()
            stream.synchronize()
            assert plan.device_status() == 0
            for row, s in enumerate(live):
                at = pool.length(s) - 1
                pg = pool.page_list(s)[at // page]
                held = []
                for cached, which in ((cache.keys, 0), (cache.values, 1)):
                    codes = cached.view(torch.uint8)[0, pg, :, at % page].view(torch.float8_e4m3fn).double()
                    held.append(codes * decoded_scales(cache.scales.view(torch.uint8)[0, pg, :, at % page, which])[:, None])
                assert float((held[1] - v[row].double()).abs().max()) <= float(v[row].abs().max()) * 2.0 ** -4
                history.setdefault(s, []).append(held)
                keys, values = (torch.stack([h[i] for h in history[s]], 1) for i in range(2))
                for append, attention in steps:            # both layers hold the same
                    x = append.q_out[row].double().reshape(kv_heads, -1, size)
                    w = torch.softmax(torch.einsum("hgd,hjd->hgj", x, keys) * size ** -0.5, -1)
                    want = torch.einsum("hgj,hjd->hgd", w, values).reshape(query, size)
                    spread = torch.einsum("hgj,hjd->hgd", w, values.abs()).reshape(query, size)
                    assert bool(((attention.out[row].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread).all())


def test_two_streams_and_graphs():
    """Two plans on two streams at once, and two captured graphs of them in turn: the same results as alone."""
    batches = [BatchE4m3([(900 + 70 * i, 1), (37, 1), (3000, 1)], 24, 4, 256, 64, seed=20 + i) for i in range(2)]
    alone = [_attend(b, 1).clone() for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    bound, graphs = [], []
    for b, s in zip(batches, streams):
        plan = host.Plan(host.Stream(0, s), kv.paged_attention_scratch_bytes(24, 4, 256, 1))
        bound.append(kv.PagedAttention.bind(plan, _cache(b), 0, b.q, b.table, b.lengths, b.starts))
    torch.cuda.synchronize()
    for _ in range(20):
        for x in bound:
            x.submit_for_plan()
    torch.cuda.synchronize()
    for x, want in zip(bound, alone):
        assert torch.equal(x.out, want)
        x.out.zero_()
    torch.cuda.synchronize()
    for x, s in zip(bound, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            x.submit_for_plan()
        graphs.append(graph)
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for x, want in zip(bound, alone):
        assert torch.equal(x.out, want) and x.plan.device_status() == 0


@pytest.mark.parametrize("seed", range(6))
def test_random_batches(seed):
    """Batches of any make-up: where the spans are cut, which pairs share one, and which lie in several differs from seed to seed."""
    g = torch.Generator().manual_seed(100 + seed)
    pick = lambda *values: values[int(torch.randint(len(values), (1,), generator=g))]  # noqa: E731
    heads = pick((24, 4, 256), (16, 16, 128), (8, 1, 128), (16, 2, 256), (32, 8, 128), (4, 4, 256))
    tokens = int(torch.randint(1, min(8, 64 // (heads[0] // heads[1])) + 1, (1,), generator=g))
    count, longest = pick(1, 7, 33, 150), pick(20, 300, 3000)
    shape = []
    for _ in range(count):
        new = int(torch.randint(0, tokens + 1, (1,), generator=g))
        shape.append((max(int(torch.randint(0, longest, (1,), generator=g)), new), new))
    batch = BatchE4m3(shape, *heads, pick(16, 32, 64, 128), seed=seed, spare_rows=1, fill=0xff)
    check(_attend(batch, tokens), *e4m3_attention_reference(batch, batch.head_dim ** -0.5))


def test_idle_slots_only():
    batch = BatchE4m3([(0, 0), (300, 0), (5, 0)], 8, 2, 128, 16, spare_rows=3)
    assert bool((_attend(batch, 1) == 0).all())
    before = [x.view(torch.uint8).clone() for x in (batch.k, batch.v, batch.scales)]
    x = torch.randn((batch.rows, 2, 128), device=DEVICE).to(torch.bfloat16)
    _append(batch, _cache(batch), (x, x), None, False, 64, torch.zeros((3, batch.rows), dtype=torch.int32, device=DEVICE))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, (batch.k, batch.v, batch.scales)))


def test_back_to_back_on_one_plan():
    """Calls of other shapes right behind one another on one plan, which is as large as the largest wants: the same results as alone."""
    batches = [BatchE4m3([(700, 2), (33, 1)], 24, 4, 256, 64, seed=1), BatchE4m3([(4000, 8)], 8, 1, 128, 16, seed=2), BatchE4m3([(9, 1)] * 50, 16, 16, 128, 32, seed=3)]
    alone = [_attend(b, 8 if i == 1 else 2).clone() for i, b in enumerate(batches)]
    plan = host.Plan(host.Stream(0), max(kv.paged_attention_scratch_bytes(b.query_heads, b.kv_heads, b.head_dim, 8 if i == 1 else 2) for i, b in enumerate(batches)))
    bound = [kv.PagedAttention.bind(plan, _cache(b), 0, b.q, b.table, b.lengths, b.starts, tokens=8 if i == 1 else 2) for i, b in enumerate(batches)]
    for _ in range(10):
        for x in bound:
            x.submit_for_plan()
    torch.cuda.synchronize()
    assert plan.device_status() == 0 and all(torch.equal(x.out, want) for x, want in zip(bound, alone))


def test_refusals():
    batch = BatchE4m3([(40, 1)], 8, 2, 128, 16)
    cache, plan = _cache(batch), host.Plan(host.Stream(0), kv.paged_attention_scratch_bytes(8, 2, 128, 1))
    good = dict(plan=plan, cache=cache, layer=0, q=batch.q, table=batch.table, lengths=batch.lengths, starts=batch.starts)
    kv.PagedAttention.bind(**good)
    for change, error in (({"layer": 1}, ValueError), ({"q": batch.q.float()}, ValueError), ({"table": batch.table.long()}, ValueError), ({"out": batch.q}, host.CudaRuntimeError),
                          ({"tokens": 9}, host.CudaRuntimeError), ({"scale": float("nan")}, host.CudaRuntimeError), ({"lengths": batch.lengths.cpu()}, ValueError),
                          ({"cache": object()}, (ValueError, AttributeError)), ({"plan": host.Plan(host.Stream(0), 1 << 12)}, host.CudaRuntimeError)):
        with pytest.raises(error):
            kv.PagedAttention.bind(**{**good, **change})


def test_as_many_sequences_as_there_may_be():
    batch = BatchE4m3([(1 + (37 * b) % 90, int(b % 5 != 3)) for b in range(1024)], 8, 2, 128, 32, seed=12, fill=0x7f)
    check(_attend(batch, 1), *e4m3_attention_reference(batch, 128 ** -0.5))


def test_a_scale_of_zero():
    """Every key weighs the same."""
    batch = BatchE4m3([(300, 2), (40, 1)], 24, 4, 256, 64, seed=13)
    check(_attend(batch, 2, scale=0.0), *e4m3_attention_reference(batch, 0.0))
