"""Batches over an E4M3 cache and over a BF16 cache with a shared prefix, with 64-bit references, for the tests of those operators."""
import torch
from decode_helpers import BF16_HALF_ULP, Batch

LEAST, LARGEST = 2.0 ** -60, 2.0 ** 60


def decoded_scales(scales):
    """The values of scale bytes in 64 bits: bytes below 67 and above 187 count as these, 255 as NaN."""
    byte = scales.view(torch.uint8).double()
    return torch.where(byte == 255, float("nan"), torch.exp2(byte.clamp(67, 187) - 127))


class BatchE4m3(Batch):
    """A `Batch` whose cache holds E4M3 codes, a head's largest around 300, and scales between 2^-9 and 2^-5."""

    def __init__(self, *args, seed=0, device="cuda:0", fill=None, **kwargs):
        super().__init__(*args, seed=seed, device="cpu", **kwargs)
        g = torch.Generator().manual_seed(seed + 1000)
        shape = self.k.shape
        self.k, self.v = ((x.float() * 90).clamp(-448, 448).to(torch.float8_e4m3fn) for x in (self.k, self.v))
        self.scales = torch.randint(118, 123, (*shape[:4], 2), generator=g, dtype=torch.uint8)
        if fill is not None:                     # what no sequence may see holds this byte
            seen = torch.zeros((self.pages, self.page_tokens), dtype=torch.bool)
            for b, (length, _) in enumerate(self.shape):
                for i in range(-(-length // self.page_tokens)):
                    seen[self.table[b, i].long(), :min(self.page_tokens, length - i * self.page_tokens)] = True
            hidden = ~seen[None, :, None, :, None]
            self.k, self.v = (x.view(torch.uint8).masked_fill(hidden, fill).view(torch.float8_e4m3fn) for x in (self.k, self.v))
            self.scales.masked_fill_(hidden, 255)
        self.scales = self.scales.view(torch.float8_e8m0fnu)
        self.to(device)

    def to(self, device):
        for name in ("table", "starts", "lengths", "k", "v", "q", "scales"):
            setattr(self, name, getattr(self, name).to(device))

    def codes(self, b, layer=0):
        """Codes and scales of sequence b's keys and values in 64 bits: [kv_heads, length, head_dim] and [kv_heads, length, 1]."""
        length = self.shape[b][0]
        pages = self.table[b, :-(-length // self.page_tokens)].long()
        out = []
        for which, cache in enumerate((self.k, self.v)):
            x = cache.view(torch.uint8)[layer, pages].view(torch.float8_e4m3fn).double()
            s = decoded_scales(self.scales.view(torch.uint8)[layer, pages])[..., which:which + 1]
            out += [y.transpose(0, 1).reshape(self.kv_heads, -1, y.shape[-1])[:, :length] for y in (x, s)]
        return out


def e4m3_attention_reference(batch, scale, layer=0, q=None):
    """(output, bound of the error) of every row in 64 bits, NaN where a row belongs to no sequence.

    The bound, for outputs o = sum w_j v_j: the result is rounded to BF16 once (2^-8 |o|). A query enters as two E4M3 terms in units in which its largest
    element is 224 at least: together they are off by 2^-10 of a unit at most, below 2^-17 of the largest element. A score's F32 sums of
    head_dim products for either term, in any order and with truncation, are off by 2 head_dim 2^-23 sum |q_i k_ji|. What a score is off by is a
    relative error of its weight, in numerator and denominator, with 2^-22 for the exponential and 2^-18 for its argument, which is up to 56. A weight times its value's scale enters the product in
    half precision (2^-11 of it) as three E4M3 terms, exact above their units: the last one's is 2^-9 / 16^2 = 2^-17, half of it the error, where the
    largest weight is 1 or more (the one that set the reference): 2^-18 of the largest, for every code. Sums in F32, with truncation: the number of tokens times 2^-23."""
    q = batch.q if q is None else q
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    group, starts = batch.query_heads // batch.kv_heads, batch.starts.tolist()
    for b, (length, new) in enumerate(batch.shape):
        if not new:
            continue
        if not length:
            out[starts[b]:starts[b] + new] = 0
            continue
        k, ks, v, vs = batch.codes(b, layer)
        rows = slice(starts[b], starts[b] + new)
        x = q[rows].double().reshape(new, batch.kv_heads, group, -1)
        scores = torch.einsum("nhgd,hjd->nhgj", x, k * ks) * scale
        size = torch.einsum("nhgd,hjd->nhgj", x.abs(), (k * ks).abs()) * abs(scale)
        rough = x.abs().amax(-1, keepdim=True) * (k * ks).abs().sum(-1) [None, :, None, :] * abs(scale) * 2.0 ** -17
        hidden = (torch.arange(length, device=q.device) > torch.arange(length - new, length, device=q.device)[:, None])[:, None, None]
        scores = scores.masked_fill(hidden, -float("inf"))
        w = torch.softmax(scores, -1).masked_fill(hidden.all(-1, keepdim=True), 0)      # a row that sees nothing gets zeros
        score_error = (size * 2 * batch.head_dim * 2.0 ** -23 + rough).masked_fill(hidden, 0).amax(-1) + 2.0 ** -22 + 2.0 ** -18
        value = torch.einsum("nhgj,hjd->nhgd", w, v * vs)
        spread = torch.einsum("nhgj,hjd->nhgd", w, (v * vs).abs())
        units = (w * vs[None, :, None, :, 0]).amax(-1, keepdim=True) * v.abs().sum(1)[None, :, None] * 2.0 ** -18
        relative = 2.0 ** -11 + 2 * score_error[..., None] + 2 * length * 2.0 ** -23
        out[rows] = value.reshape(new, batch.query_heads, -1)
        bound[rows] = (BF16_HALF_ULP * value.abs() + (relative * spread + units) * (1 + BF16_HALF_ULP)).reshape(new, batch.query_heads, -1)
    return out, bound


class PrefixBatch(Batch):
    """A `Batch` whose sequences begin with the same `prefix` tokens (whole pages) in pages of their own; `shape` counts them too. A sequence may be shorter."""

    def __init__(self, shape, query_heads, kv_heads, head_dim, page_tokens, prefix, seed=0, device="cuda:0", hide=False, spare_prefix=0, **kwargs):
        super().__init__([(max(length - prefix, 0), new) for length, new in shape], query_heads, kv_heads, head_dim, page_tokens, seed=seed, device="cpu", **kwargs)
        held = prefix // page_tokens
        own, self.shape, self.prefix = self.table, list(shape), prefix
        g = torch.Generator().manual_seed(seed + 2000)
        normal = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16)  # noqa: E731
        more = (self.k.shape[0], held + spare_prefix, *self.k.shape[2:])
        order = torch.randperm(self.pages + held + spare_prefix, generator=g)        # the prefix's pages lie among the others
        self.k, self.v = (torch.cat([x, normal(*more)], 1)[:, torch.argsort(order)] for x in (self.k, self.v))
        where = order.to(torch.int32)
        own = torch.where(own >= 0, where[own.clamp(min=0).long()], -1)
        first = self.pages
        self.pages += held + spare_prefix
        self.prefix_pages = where[first:first + held + spare_prefix] if held + spare_prefix else torch.zeros(1, dtype=torch.int32)
        shared = where[first:first + held].expand(len(shape), -1) if not hide else torch.full((len(shape), held), -7, dtype=torch.int32)
        self.table = torch.cat([shared, own], 1).contiguous()
        self.lengths = torch.tensor([length for length, _ in shape], dtype=torch.int32)
        self.prefix_tokens = torch.tensor([prefix], dtype=torch.int32)
        for name in ("table", "starts", "lengths", "k", "v", "q", "prefix_pages", "prefix_tokens"):
            setattr(self, name, getattr(self, name).to(device))

    def cached(self, b, layer=0):
        length, held = self.shape[b][0], self.prefix // self.page_tokens
        pages = torch.cat([self.prefix_pages[:held], self.table[b, held:]])[:-(-length // self.page_tokens)].long()
        take = lambda c: c[layer, pages].double().transpose(0, 1).reshape(self.kv_heads, -1, self.head_dim)[:, :length]  # noqa: E731
        return take(self.k), take(self.v)


def prefix_attention_reference(batch, scale, layer=0, q=None):
    """As `decode_helpers.attention_reference`, with weights of one BF16 term: o = sum w_j (1 + d_j) v_j / sum w_j (1 + d_j) with |d_j| <= 2^-8
    is off by 2^-8 sum w_j |v_j - o| / (1 - 2^-8) at most."""
    q = batch.q if q is None else q
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    group, starts = batch.query_heads // batch.kv_heads, batch.starts.tolist()
    for b, (length, new) in enumerate(batch.shape):
        if not new:
            continue
        if not length:
            out[starts[b]:starts[b] + new] = 0
            continue
        k, v = batch.cached(b, layer)
        rows = slice(starts[b], starts[b] + new)
        x = q[rows].double().reshape(new, batch.kv_heads, group, -1)
        scores = torch.einsum("nhgd,hjd->nhgj", x, k) * scale
        size = torch.einsum("nhgd,hjd->nhgj", x.abs(), k.abs()) * abs(scale)
        hidden = (torch.arange(length, device=q.device) > torch.arange(length - new, length, device=q.device)[:, None])[:, None, None]
        w = torch.softmax(scores.masked_fill(hidden, -float("inf")), -1).masked_fill(hidden.all(-1, keepdim=True), 0)
        score_error = size.masked_fill(hidden, 0).amax(-1) * batch.head_dim * 2.0 ** -23 + 2.0 ** -22
        value = torch.einsum("nhgj,hjd->nhgd", w, v)
        spread = torch.einsum("nhgj,hjd->nhgd", w, v.abs())
        relative = 2 * score_error[..., None] + 2 * length * 2.0 ** -23
        rounded = (spread + value.abs()) * BF16_HALF_ULP / (1 - BF16_HALF_ULP)
        out[rows] = value.reshape(new, batch.query_heads, -1)
        bound[rows] = (BF16_HALF_ULP * value.abs() + (relative * spread + rounded) * (1 + BF16_HALF_ULP)).reshape(new, batch.query_heads, -1)
    return out, bound


def check(got, want, bound):
    """Rows of sequences within the bound, the others as they were (zeros)."""
    live = ~want.isnan()
    off = (got.double() - want).abs()
    assert bool((off <= bound)[live].all()), f"off by {(off / bound.clamp(min=1e-300))[live].max().item():.3g} of the bound"
    assert bool((got[~live] == 0).all())
