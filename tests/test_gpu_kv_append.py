"""GPU tests of the rotary positions and the cache write, against 64 bits.

Bound of an element's error: one rounding to BF16 (2^-8 of the value) and F32 before it. The rotation adds two products of values below the pair's
norm r with a sine and a cosine that are good to 2^-22 (their angle to 2^-24 of a half turn, the functions to 2 units in the last place), each
product and the sum rounded: 2^-20 r is above all of it. The head norm's factor is good to (head_dim + 4) 2^-24, less than 2^-15 of the value."""
import pytest
import torch

from augur_v100_b200 import host, kv
from decode_helpers import BF16_HALF_ULP, Batch, rotary_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def stream():
    torch.cuda.set_device(0)
    s = host.Stream(0)
    yield s
    s.close()


class Step:
    """A step's tensors: q as the query half of a query|gate projection, k and v side by side in one."""

    def __init__(self, shape, heads, page_tokens, sections, seed=0, norm=False, far=1 << 20, spare_rows=0):
        g = torch.Generator().manual_seed(seed)
        self.batch = Batch(shape, *heads, page_tokens, seed=seed, spare_rows=spare_rows)
        rows, (query, key, size) = self.batch.rows, heads
        cuda = lambda t: t.to("cuda:0")  # noqa: E731
        self.q = cuda(torch.randn((rows, query, 2, size), generator=g).to(torch.bfloat16))[:, :, 0]
        pair = cuda(torch.randn((rows, 2 * key, size), generator=g).to(torch.bfloat16) * 3)
        self.k, self.v = pair[:, :key], pair[:, key:]
        self.positions = cuda(torch.randint(far, (3, rows), generator=g, dtype=torch.int32))
        self.sections, half = sections, sum(sections)
        self.frequencies = cuda((1.0e7 ** (-torch.arange(half, dtype=torch.float64) / half)).float())
        self.q_norm = cuda(1 + 0.2 * torch.randn(size, generator=g)) if norm else None
        self.k_norm = cuda(1 + 0.2 * torch.randn(size, generator=g)) if norm else None

    def bind(self, stream, interleaved=False, **changes):
        b = self.batch
        self.q_out = torch.full(self.q.shape, 77.0, dtype=torch.bfloat16, device="cuda:0")
        values = dict(q=self.q, k=self.k, v=self.v, positions=self.positions, frequencies=self.frequencies, sections=self.sections, table=b.table,
                      lengths=b.lengths, starts=b.starts, q_out=self.q_out, q_norm=self.q_norm, k_norm=self.k_norm)
        return kv.KvAppend.bind(stream, kv.KvCache(b.k, b.v), 0, interleaved=interleaved, **{**values, **changes})

    def check(self, stream, interleaved, skip=()):
        """Submits, and compares everything that the call may write with what it should; rows in `skip` are not written to the cache."""
        b = self.batch
        keys, values = b.k.clone(), b.v.clone()
        self.bind(stream, interleaved).submit()
        stream.synchronize()
        epsilon = 1e-6
        q = rotary_reference(self.q, self.q_norm, self.positions, self.frequencies, self.sections, interleaved, epsilon)
        k = rotary_reference(self.k, self.k_norm, self.positions, self.frequencies, self.sections, interleaved, epsilon)
        live = [row for s, (_, new) in enumerate(b.shape) for row in range(int(b.starts[s]), int(b.starts[s]) + new)]
        self.close(self.q_out[live], q[live])
        rest = [row for row in range(b.rows) if row not in live]
        assert bool((self.q_out[rest] == 77.0).all())
        for s, (length, new) in enumerate(b.shape):
            for i in range(new):
                row, at = int(b.starts[s]) + i, length - new + i
                if row in skip:
                    continue
                page = int(b.table[s, at // b.page_tokens])
                self.close(b.k[0, page, :, at % b.page_tokens], k[row])
                assert torch.equal(b.v[0, page, :, at % b.page_tokens], self.v[row])
                keys[0, page, :, at % b.page_tokens] = b.k[0, page, :, at % b.page_tokens]
                values[0, page, :, at % b.page_tokens] = b.v[0, page, :, at % b.page_tokens]
        assert torch.equal(b.k, keys) and torch.equal(b.v, values)          # nothing else was written

    def close(self, got, want):
        half = sum(self.sections)
        size = want.abs()
        pair = torch.sqrt(want[..., :half] ** 2 + want[..., half:2 * half] ** 2)
        size[..., :half], size[..., half:2 * half] = pair, pair
        bound = BF16_HALF_ULP * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -20 * size + 2.0 ** -15 * size * (self.q_norm is not None) * 2
        assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() - bound).max())


LAYER = (24, 4, 256)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,sections", [(LAYER, (11, 11, 10)), ((32, 8, 128), (16, 24, 24)), ((1, 1, 128), (8, 0, 0)), ((3, 1, 256), (0, 64, 64)),
                                            ((5, 5, 128), (1, 3, 20))])
def test_heads_norms_and_sections(stream, heads, sections, norm, interleaved):
    Step([(8, 8), (100, 1), (0, 0), (17, 3), (64, 0), (33, 33)], heads, 16, sections, seed=sum(sections), norm=norm, spare_rows=2).check(stream, interleaved)


@pytest.mark.parametrize("page_tokens", [16, 64, 1024])
@pytest.mark.parametrize("shape", [[(1, 1)], [(5, 1)] * 700, [(1030, 1030)], [(64, 8), (65, 8), (66, 8)]])
def test_steps_of_all_sizes(stream, shape, page_tokens):
    Step(shape, (4, 2, 128), page_tokens, (16, 24, 24), seed=len(shape)).check(stream, False)


def test_far_positions_lose_nothing(stream):
    step = Step([(6, 6)], LAYER, 16, (11, 11, 10), seed=2)
    step.positions[:] = torch.tensor([2 ** 31 - 1, 2 ** 24 + 1, -2 ** 31, -1, 0, 123456789], dtype=torch.int32)
    # an angle of 2^31 radians is good to 2^-20 of a radian in 64 bits here and in the reference: inside the bound only from there
    step.check(stream, True)


def test_pages_that_are_not_there(stream):
    for bad in (-1, -7, 10 ** 9):
        step = Step([(20, 2), (40, 3)], LAYER, 16, (11, 11, 10), seed=3)
        step.batch.table[1, 2] = bad                                          # tokens 37..39 of the second sequence
        step.check(stream, False, skip=(2, 3, 4))
    step = Step([(20, 2), (40, 3)], LAYER, 16, (11, 11, 10), seed=3)
    step.batch.lengths[1] = 16 * step.batch.table.shape[1] + 3               # behind the table
    step.check(stream, False, skip=(2, 3, 4))
    step.batch.lengths[1] = 2                                                 # fewer tokens than rows: the first row has no place
    keys = step.batch.k.clone()
    step.bind(stream).submit()
    stream.synchronize()
    page = int(step.batch.table[1, 0])
    changed = (keys != step.batch.k).any(-1).any(2)[0]                        # [pages, page_tokens]
    assert sorted(map(tuple, changed.nonzero().tolist())) == [(page, 0), (page, 1)]


def test_replay_side_stream_and_refusals(stream):
    step = Step([(30, 2)], LAYER, 16, (11, 11, 10), seed=8, norm=True)
    side = host.Stream(0, torch.cuda.Stream())
    call = step.bind(side)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side.torch_stream):
        call.submit()
    step.batch.lengths.fill_(29)
    step.batch.shape = [(29, 2)]
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    first = call.q_out.clone(), step.batch.k.clone()
    step.check(side, False)
    assert torch.equal(first[0], step.q_out) and torch.equal(first[1], step.batch.k)
    del graph
    for bad in (dict(q=step.q.float()), dict(k=step.k[:, :2]), dict(positions=step.positions.long()), dict(frequencies=step.frequencies[:4]),
                dict(q_out=step.q_out[:, :, ::2]), dict(sections=(11, 11)), dict(lengths=step.batch.lengths.cpu()), dict(q_norm=step.q_norm.half())):
        with pytest.raises(ValueError):
            step.bind(stream, **bad)
    with pytest.raises(host.CudaRuntimeError):
        step.bind(stream, q_out=step.batch.k[0, :2 * 24 * 256 // (4 * 16 * 256) + 1].reshape(-1)[:2 * 24 * 256].reshape(2, 24, 256))
    side.close()
