"""Batches over a paged cache and 64-bit references for the tests of the decoding operators."""
import numpy as np
import torch

BF16_HALF_ULP = torch.finfo(torch.bfloat16).eps / 2      # 2^-8: a rounding to BF16 is off by at most this, relative to the value


class Batch:
    """Sequences over a paged cache with random contents: `shape` is [(cached tokens with the new ones, new tokens), ...]."""

    def __init__(self, shape, query_heads, kv_heads, head_dim, page_tokens, seed=0, device="cuda:0", spare_pages=3, spare_rows=0, table_spare=1,
                 layers=1, fill=None):
        g = torch.Generator(device="cpu").manual_seed(seed)
        counts = [-(-length // page_tokens) for length, _ in shape]
        self.shape, self.query_heads, self.kv_heads, self.head_dim, self.page_tokens = shape, query_heads, kv_heads, head_dim, page_tokens
        self.pages = sum(counts) + spare_pages
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(shape), max(max(counts), 1) + table_spare), -1, dtype=torch.int32)
        at = 0
        for b, count in enumerate(counts):
            self.table[b, :count] = order[at:at + count]
            at += count
        starts = np.concatenate([[0], np.cumsum([new for _, new in shape])])
        self.rows = int(starts[-1]) + spare_rows
        self.starts = torch.tensor(starts, dtype=torch.int32)
        self.lengths = torch.tensor([length for length, _ in shape], dtype=torch.int32)
        normal = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16)  # noqa: E731
        cache = (layers, self.pages, kv_heads, page_tokens, head_dim)
        self.k, self.v = normal(*cache), normal(*cache)
        if fill is not None:                     # what no sequence may see holds this value
            seen = torch.zeros((self.pages, page_tokens), dtype=torch.bool)
            for b, (length, _) in enumerate(shape):
                for i in range(counts[b]):
                    seen[self.table[b, i], :min(page_tokens, length - i * page_tokens)] = True
            self.k.masked_fill_(~seen[None, :, None, :, None], fill)
            self.v.masked_fill_(~seen[None, :, None, :, None], fill)
        self.q = normal(max(self.rows, 1), query_heads, head_dim)
        self.rows = max(self.rows, 1)
        for name in ("table", "starts", "lengths", "k", "v", "q"):
            setattr(self, name, getattr(self, name).to(device))

    def cached(self, b, layer=0):
        """Keys and values of sequence b in 64 bits: [kv_heads, length, head_dim]."""
        length = self.shape[b][0]
        pages = self.table[b, :-(-length // self.page_tokens)].long()
        take = lambda c: c[layer, pages].double().transpose(0, 1).reshape(self.kv_heads, -1, self.head_dim)[:, :length]  # noqa: E731
        return take(self.k), take(self.v)


def attention_reference(batch, scale, layer=0, q=None):
    """(output, bound of the error) of every row in 64 bits, NaN where a row belongs to no sequence.

    The bound, for outputs o = sum w_j v_j: the result is rounded to BF16 once (2^-8 |o|). Every weight is the sum of two BF16 terms, off by 2^-8 of
    the first one's rounding error, 2^-8 of it again, in the product and in the denominator: sum w_j |v_j| takes 2^-16 from either. A score's F32 sum of
    head_dim exact products, added in any order and with truncation, is off by head_dim 2^-23 sum |q_i k_ji| at most; scaled to
    a power of two and taken to it, with another 2^-22 for the exponential, that is a relative error of w_j, in numerator and denominator.
    Sums of the weights and of the products in F32, with truncation: the number of tokens times 2^-23."""
    q = batch.q if q is None else q
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    group, starts = batch.query_heads // batch.kv_heads, batch.starts.tolist()
    for b, (length, new) in enumerate(batch.shape):
        if not new:
            continue
        k, v = batch.cached(b, layer)
        rows = slice(starts[b], starts[b] + new)
        x = q[rows].double().reshape(new, batch.kv_heads, group, -1)
        scores = torch.einsum("nhgd,hjd->nhgj", x, k) * scale
        size = torch.einsum("nhgd,hjd->nhgj", x.abs(), k.abs()) * abs(scale)
        hidden = torch.arange(length, device=q.device) > torch.arange(length - new, length, device=q.device)[:, None]
        scores = scores.masked_fill(hidden[:, None, None], -float("inf"))
        w = torch.softmax(scores, -1)
        score_error = (w * size).amax(-1) * 0 + size.masked_fill(hidden[:, None, None], 0).amax(-1) * batch.head_dim * 2.0 ** -23 + 2.0 ** -22
        value = torch.einsum("nhgj,hjd->nhgd", w, v)
        spread = torch.einsum("nhgj,hjd->nhgd", w, v.abs())
        relative = 2 * BF16_HALF_ULP ** 2 + 2 * score_error[..., None] + 2 * length * 2.0 ** -23
        out[rows] = value.reshape(new, batch.query_heads, -1)
        bound[rows] = (BF16_HALF_ULP * value.abs() + relative * spread * (1 + BF16_HALF_ULP)).reshape(new, batch.query_heads, -1)
    return out, bound


def axis_of_pairs(sections, interleaved):
    total = sum(sections)
    if not interleaved:
        return [0] * sections[0] + [1] * sections[1] + [2] * sections[2]
    return [i % 3 if i < 3 * sections[i % 3] else 0 for i in range(total)]


def rotary_reference(x, norm, positions, frequencies, sections, interleaved, epsilon):
    """[rows, heads, head_dim] in 64 bits: optional head norm, then the rotation. `positions` [3, rows]."""
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + epsilon) * norm.double()
    half = sum(sections)
    angle = positions[axis_of_pairs(sections, interleaved)].double().T * frequencies.double()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1)
