"""Attention over the E4M3 cache where weights lie far apart: one key that outweighs a long tail, against a 64-bit reference with a bound
that counts the tail's keys at 2^-32 of the largest weight each."""
import math

import pytest
import torch
from decode_helpers import BF16_HALF_ULP
from kv8_helpers import BatchE4m3

from augur_v100_b200 import host, kv

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def _batch(length, sequences, group, head_dim, seed):
    """As many sequences of one key-value head on the same pages: with one for each SM, every one is a span of its own."""
    batch = BatchE4m3([(length, 1)], group, 1, head_dim, 256, seed=seed)
    batch.shape, batch.rows = batch.shape * sequences, sequences
    batch.table = batch.table.expand(sequences, -1).contiguous()
    batch.lengths = torch.full((sequences,), length, dtype=torch.int32, device=DEVICE)
    batch.starts = torch.arange(sequences + 1, dtype=torch.int32, device=DEVICE)
    g = torch.Generator().manual_seed(seed)
    batch.q = (torch.randint(0, 2, (sequences, group, head_dim), generator=g) * 2 - 1).to(torch.bfloat16).to(DEVICE)
    return batch


def _slot(batch, key):
    return 0, int(batch.table[0, key // 256]), 0, key % 256


def _reference(batch, scale):
    """(output, bound of the error) in 64 bits.

    The bound: the result is rounded to BF16 once. A weight times its value's scale enters the product in half precision (2^-11 of it; below 2^-21 of the one that
    set the reference, which the largest is at least, to 2^-32 of that), met exactly by three terms. Queries are met exactly too (no element below 2^-9 of its head's largest). A
    score is off by 2 head_dim 2^-23 sum |q_i k_ji| (F32 sums of either term) and, below 128 and rounded three times on its way into the exponential, by 3 * 2^-18; with 2^-22 for the
    exponential that is a relative error of its weight, in numerator and denominator. The products of 32 keys are added to the F32 sum at a time, and a
    thread adds every 128th weight to a denominator: 2^-23 of the sum for each."""
    k, ks, v, vs = (x[0] for x in batch.codes(0))
    k, length = k * ks, batch.shape[0][0]
    out, bound = (torch.empty(batch.q.shape, dtype=torch.float64, device=DEVICE) for _ in range(2))
    for b in range(len(batch.shape)):
        x = batch.q[b].double()
        assert bool((x.abs() >= x.abs().amax(-1, keepdim=True) * 2.0 ** -9).all())
        scores = x @ k.T * scale
        assert float(scores.abs().max()) / math.log(2) + float(vs.log2().abs().max()) < 128
        w = torch.softmax(scores, -1)
        error = (x.abs() @ k.abs().T * abs(scale)).amax(-1) * 2 * batch.head_dim * 2.0 ** -23 + 3 * 2.0 ** -18 + 2.0 ** -22
        relative = 2.0 ** -11 + 2 * error + length * (1 / 32 + 1 / 128) * 2.0 ** -23
        out[b] = w @ (v * vs)
        floor = (w * vs[:, 0]).amax(-1, keepdim=True) * v.abs().sum(0) * 2.0 ** -32
        bound[b] = BF16_HALF_ULP * out[b].abs() + (relative[:, None] * (w @ (v * vs).abs()) + floor) * (1 + BF16_HALF_ULP)
    return out, bound


def _check(batch, scale):
    plan = host.Plan(host.Stream(0), kv.paged_attention_scratch_bytes(batch.query_heads, 1, batch.head_dim, 1))
    bound = kv.PagedAttention.bind(plan, kv.KvCacheE4m3(batch.k, batch.v, batch.scales), 0, batch.q, batch.table, batch.lengths, batch.starts, scale=scale)
    bound.submit_for_plan()
    torch.cuda.synchronize()
    assert plan.device_status() == 0
    want, allowed = _reference(batch, scale)
    worst = ((bound.out.double() - want).abs() / allowed).max().item()
    assert worst <= 1, f"off by {worst:.3g} of the bound"


@pytest.mark.parametrize("length,where", [(4100, 0.0), (32769, 0.0), (32769, 0.6), (131072, 0.0), (131072, 0.3), (131072, 1.0)])
@pytest.mark.parametrize("group,head_dim", [(8, 128), (16, 256), (40, 128), (64, 256)])
def test_a_key_that_outweighs_a_long_tail(length, where, group, head_dim):
    """The tail's keys weigh 2^-20 of one key, or 2^-17, or 2^-12, with a spread of a factor e: together from next to nothing to nearly all. Values of one sign, the first dim's 1."""
    batch = _batch(length, host.sm_count(0), group, head_dim, seed=length % 97)
    scale, unit = head_dim ** -0.5, 2.0 ** -7
    # the dims behind the first: scores with a spread of 1 (codes of spread 90, head_dim - 1 products); the first: the one key's
    batch.k.view(torch.uint8)[..., 0] = 0
    batch.scales.view(torch.uint8)[..., 0] = 120
    batch.scales.view(torch.uint8)[..., 1] = 127
    batch.v = batch.v.float().abs().clamp(min=1.0).to(torch.float8_e4m3fn)
    batch.v.view(torch.uint8)[..., 0] = 0x38                            # 1
    key = min(int(where * length), length - 1)
    batch.k.view(torch.uint8)[_slot(batch, key)] = 0
    batch.k.view(torch.uint8)[_slot(batch, key)][0] = 0x7e              # 448
    q = batch.q.float()
    q[..., 1:] /= 90 * unit * scale * math.sqrt(head_dim - 1)
    q[..., 0] = torch.tensor([20.0, 17.0, 12.0], device=DEVICE)[torch.arange(group, device=DEVICE) % 3] * math.log(2) / (448 * unit * scale)
    batch.q = q.to(torch.bfloat16)
    _check(batch, scale)


@pytest.mark.parametrize("where", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("parts", [True, False])
@pytest.mark.parametrize("group,head_dim", [(8, 128), (16, 256), (40, 128), (64, 256)])
def test_value_scales_at_either_end(parts, where, group, head_dim):
    """Values of the least scale under one of the largest, in other parts of the sequence than that one's or in other tiles of the one part: the key with
    the largest has 2^7 times their weight, or 2^3, and 16384 others nearly all of the denominator; their references lie 2^127 apart, or 2^123."""
    length, scale, unit = 16385, head_dim ** -0.5, 2.0 ** -7
    batch = _batch(length, 1 if parts else host.sm_count(0), group, head_dim, seed=7)
    batch.k.view(torch.uint8).zero_()
    batch.scales.view(torch.uint8)[..., 0] = 120
    batch.scales.view(torch.uint8)[..., 1] = 67
    slot = _slot(batch, min(int(where * length), length - 1))
    batch.k.view(torch.uint8)[slot][0] = 0x7e                           # 448
    batch.scales.view(torch.uint8)[slot][1] = 187
    q = batch.q.float()
    q[..., 0] = torch.tensor([7.0, 3.0], device=DEVICE)[torch.arange(group, device=DEVICE) % 2] * math.log(2) / (448 * unit * scale)
    batch.q = q.to(torch.bfloat16)
    _check(batch, scale)
