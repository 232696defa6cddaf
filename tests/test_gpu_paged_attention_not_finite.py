"""GPU tests of the attention over a paged cache with NaN and infinities in live queries, keys and values: the output is what the formula gives, however
the (sequence, key-value head) pairs fall into spans. A pair of one unit of 64 tokens lies in one span; longer ones, of a sequence on its own, in several."""
import math

import pytest
import torch

from augur_v100_b200 import host, kv
from decode_helpers import BF16_HALF_ULP, Batch, attention_reference

pytestmark = pytest.mark.gpu

LAYER = (24, 4, 256)
GROUP = LAYER[0] // LAYER[1]
# one span; spans whose last unit holds the newest token alone; dozens of parts
LENGTHS = [1, 50, 129, 4097, 20011]


@pytest.fixture(scope="module")
def stream():
    torch.cuda.set_device(0)
    s = host.Stream(0)
    yield s
    s.close()


def _run(stream, batch, tokens):
    plan = host.Plan(stream, kv.paged_attention_scratch_bytes(*LAYER, tokens))
    out = torch.full(batch.q.shape, 77.0, dtype=torch.bfloat16, device="cuda:0")
    call = kv.PagedAttention.bind(plan, kv.KvCache(batch.k, batch.v), 0, batch.q, batch.table, batch.lengths, batch.starts, tokens, out)
    call.submit_for_plan()
    stream.synchronize()
    assert plan.device_status() == 0
    return out


def _slot(batch, position, head, b=0):
    """Index of a key or value of sequence b: [page, head, row]."""
    return 0, int(batch.table[b, position // batch.page_tokens]), head, position % batch.page_tokens


def _heads(head):
    return slice(head * GROUP, (head + 1) * GROUP)


def _within(got, want, bound):
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() - bound).max())


@pytest.mark.parametrize("tokens", [1, 4])
@pytest.mark.parametrize("length", LENGTHS)
def test_nan_in_a_query(stream, length, tokens):
    length = max(length, tokens)
    batch = Batch([(length, tokens)], *LAYER, 64, seed=length)
    clean = _run(stream, batch, tokens)
    want, bound = attention_reference(batch, 1 / 16)
    token, head = tokens // 2, 8
    for value in (math.nan, -math.nan):
        q = batch.q.clone()
        q[token, head, 17] = value
        batch.q, kept = q, batch.q
        out = _run(stream, batch, tokens)
        batch.q = kept
        assert bool(out[token, head].isnan().all())
        alone = torch.zeros(out.shape, dtype=torch.bool, device="cuda:0")
        alone[token, head] = True
        _within(out[~alone], want[~alone], bound[~alone])
        other = torch.ones(LAYER[0], dtype=torch.bool, device="cuda:0")
        other[_heads(head // GROUP)] = False
        assert torch.equal(out[:, other], clean[:, other])         # other pairs: not a bit


@pytest.mark.parametrize("tokens", [1, 4])
@pytest.mark.parametrize("length", LENGTHS)
def test_nan_in_a_key(stream, length, tokens):
    length = max(length, tokens)
    batch = Batch([(length, tokens)], *LAYER, 64, seed=length)
    clean = _run(stream, batch, tokens)
    want, bound = attention_reference(batch, 1 / 16)
    for position in sorted({0, length // 2, length - 1, max(length - 2, 0)}):
        k = batch.k.clone()
        k[_slot(batch, position, 2)][5] = math.nan
        batch.k, kept = k, batch.k
        out = _run(stream, batch, tokens)
        batch.k = kept
        for token in range(tokens):
            mine = out[token, _heads(2)]
            if position < length - tokens + token + 1:
                assert bool(mine.isnan().all()), (position, token)
            else:
                _within(mine, want[token, _heads(2)], bound[token, _heads(2)])
        for head in (0, 1, 3):
            assert torch.equal(out[:, _heads(head)], clean[:, _heads(head)])


@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("length", LENGTHS[1:])
def test_nan_beside_a_key_that_outweighs_it(stream, length, what):
    # The first key's score is above all others by more than F32 powers of two reach (12 |q|^2 / 16 log2(e), some 270): every other weight is
    # zero in F32, and the formula is NaN all the same.
    batch = Batch([(length, 1)], *LAYER, 64, seed=3)
    head = 7
    batch.k[_slot(batch, 0, 1)] = (12 * batch.q[0, head].float()).to(torch.bfloat16)
    out = _run(stream, batch, 1)
    assert torch.equal(out[0, head], batch.v[_slot(batch, 0, 1)])
    for position in sorted({length // 2, length - 1}):
        tensor = batch.k if what == "key" else batch.v
        kept = tensor.clone()
        tensor[_slot(batch, position, 1)][5] = math.nan
        out = _run(stream, batch, 1)
        tensor.copy_(kept)
        lost = out[0, head].isnan()
        assert bool(lost.all()) if what == "key" else bool(lost[5]) and int(lost.sum()) == 1


@pytest.mark.parametrize("length", LENGTHS)
def test_infinity_in_a_key(stream, length):
    # A score of +infinity makes the formula NaN (infinity less infinity); one of -infinity takes the key out.
    batch = Batch([(length, 1)], *LAYER, 64, seed=length + 1)
    want, bound = attention_reference(batch, 1 / 16)
    for position in sorted({0, length // 2, length - 1}):
        for value in (math.inf, -math.inf):
            kept = batch.k.clone()
            batch.k[_slot(batch, position, 0)][9] = value
            out = _run(stream, batch, 1)
            batch.k.copy_(kept)
            up = (batch.q[0, :GROUP, 9] > 0) == (value > 0)
            assert bool(out[0, :GROUP][up].isnan().all())
            if bool((~up).any()):
                k, v = batch.cached(0)
                rest = torch.arange(length, device="cuda:0") != position
                x = batch.q[0, :GROUP].double()[~up]
                w = torch.softmax(x @ k[0, rest].T / 16, -1) if length > 1 else torch.zeros((len(x), 0), dtype=torch.float64, device="cuda:0")
                one_less = (w @ v[0, rest])
                # the bound of all keys, its output term for the other output (2^-8 of it), and weights that one key less makes larger: at most by the ratio
                # of the denominators
                more = bound[0, :GROUP][~up] * (1 / (1 - _weight(batch, position)[~up]))[:, None] if length > 1 else 0
                _within(out[0, :GROUP][~up], one_less, more + BF16_HALF_ULP * one_less.abs())
            _within(out[0, GROUP:], want[0, GROUP:], bound[0, GROUP:])


def _weight(batch, position):
    """The weight of one key of the first key-value head for each of its queries."""
    k, _ = batch.cached(0)
    return torch.softmax(batch.q[0, :GROUP].double() @ k[0].T / 16, -1)[:, position]


@pytest.mark.parametrize("length", LENGTHS)
def test_a_row_whose_scores_are_all_minus_infinity(stream, length):
    # Documented: zeros, as where a row sees no token at all.
    batch = Batch([(length, 1)], *LAYER, 64, seed=length + 2)
    want, bound = attention_reference(batch, 1 / 16)
    q, k = batch.q.clone(), batch.k.clone()
    k[0, :, 3, :, 30] = -k[0, :, 3, :, 30].abs() - 1
    q[0, 20, 30] = math.inf
    batch.q, batch.k = q, k
    out = _run(stream, batch, 1)
    assert bool((out[0, 20] == 0).all())
    _within(out[0, :18], want[0, :18], bound[0, :18])
    batch.k = -k                                     # and all of +infinity: NaN
    out = _run(stream, batch, 1)
    assert bool(out[0, 20].isnan().all())


@pytest.mark.parametrize("length", LENGTHS[1:])
def test_lowest_scores_beside_minus_infinity(stream, length):
    # The first half's scores are all -1.3 2^127, in powers of two -1.87 2^127, among the lowest that F32 holds; the second half's are -infinity. The first half weighs
    # the same, and the row gets its mean: as good as sums of fewer than 2^15 terms, each rounded by 2^-23 of what is summed, and the output's rounding.
    batch = Batch([(length, 1)], *LAYER, 64, seed=length + 4)
    batch.k.zero_()
    batch.q.zero_()
    batch.q[0, :, 7] = 1.296875 * 2.0 ** 63
    half = (length + 1) // 2
    position = torch.arange(length, device="cuda:0")
    batch.k[0, batch.table[0, position // 64].long(), :, position % 64, 7] = torch.where(position < half, -2.0 ** 64, -math.inf).to(torch.bfloat16)[:, None]
    plan = host.Plan(stream, kv.paged_attention_scratch_bytes(*LAYER, 1))
    call = kv.PagedAttention.bind(plan, kv.KvCache(batch.k, batch.v), 0, batch.q, batch.table, batch.lengths, batch.starts, 1, scale=1.0)
    call.submit_for_plan()
    stream.synchronize()
    _, v = batch.cached(0)
    want, spread = v[:, :half].mean(1), v[:, :half].abs().mean(1)
    _within(call.out[0].reshape(4, 6, 256), want[:, None], (BF16_HALF_ULP * want.abs() + half * 2.0 ** -22 * spread)[:, None])


@pytest.mark.parametrize("length", LENGTHS)
def test_infinity_and_nan_in_a_value(stream, length):
    # Documented: an infinity that a row sees gives an infinity or NaN, in its own element of the head only.
    batch = Batch([(length, 1)], *LAYER, 64, seed=length + 3)
    want, bound = attention_reference(batch, 1 / 16)
    for position in sorted({0, length // 2, length - 1}):
        for value in (math.inf, -math.inf, math.nan):
            kept = batch.v.clone()
            batch.v[_slot(batch, position, 3)][200] = value
            out = _run(stream, batch, 1)
            batch.v.copy_(kept)
            hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda:0")
            hit[0, _heads(3), 200] = True
            assert not bool(out[hit].isfinite().any()) and (math.isinf(value) or bool(out[hit].isnan().all()))
            _within(out[~hit], want[~hit], bound[~hit])


def test_nan_stays_in_its_sequence(stream):
    # A batch with pairs of both kinds: sequences without a NaN keep every bit.
    batch = Batch([(30, 1), (3000, 1), (64, 1), (1025, 1)], *LAYER, 16, seed=6)
    clean = _run(stream, batch, 1)
    for b, (length, _) in enumerate(batch.shape):
        q = batch.q.clone()
        q[b, :, 0] = math.nan
        batch.q, kept = q, batch.q
        out = _run(stream, batch, 1)
        batch.q = kept
        assert bool(out[b].isnan().all())
        rest = [i for i in range(4) if i != b]
        assert torch.equal(out[rest], clean[rest])
