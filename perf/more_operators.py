"""Cases of the operators around an 8-bit key-value cache and a shared prefix: the cache write that quantises to E4M3, attention over
that cache, and attention of a batch whose sequences share a long prefix, each with a plain form in elementary torch operations.

``own`` selects what ``run`` computes with: the plain form, or the library's entry points through the package.
"""
import math

import torch

own = False

DEVICE = "cuda:0"

# (query heads, key-value heads, head size). The first is the full-attention layer of the model this library serves; the others are generic.
HEADS = ((24, 4, 256), (32, 8, 128), (16, 16, 128), (8, 1, 128), (16, 2, 256))
ROTARY = {256: (64, (11, 11, 10)), 128: (128, (16, 24, 24))}    # rotary size and sections (time, height, width) by head size
EPSILON = 1e-6


def listed():
    return [
        # the cache write of the batch of eight rows that verifies speculated tokens, with head norms
        {"name": "append_8", "op": "append", "heads": 0, "sequences": 1, "tokens": 8, "page": 64, "norm": True, "interleaved": True, "far": 262143},
        # a full server's, text and image positions, small pages
        {"name": "append_96x5", "op": "append", "heads": 1, "sequences": 96, "tokens": 5, "page": 16, "norm": False, "interleaved": False, "far": 1000003},
        # a chunk of two prompts
        {"name": "append_prompt", "op": "append", "heads": 0, "sequences": 2, "tokens": 2047, "page": 64, "norm": True, "interleaved": True, "far": 131072},
        # one user's decoding step, a few thousand tokens in
        {"name": "attention_one_4k", "op": "attention", "heads": 0, "sequences": 1, "length": 4100, "tokens": 1, "page": 64, "ragged": False},
        # a server's decoding step: 64 users, contexts from a few hundred tokens to 8 thousand, some slots idle
        {"name": "attention_64_ragged", "op": "attention", "heads": 0, "sequences": 64, "length": 8191, "tokens": 1, "page": 64, "ragged": True},
        # eight speculated tokens of four users, 16 thousand tokens in, small pages
        {"name": "attention_verify_8", "op": "attention", "heads": 0, "sequences": 4, "length": 16385, "tokens": 8, "page": 16, "ragged": False},
        # two long documents
        {"name": "attention_long_128", "op": "attention", "heads": 1, "sequences": 2, "length": 131071, "tokens": 1, "page": 128, "ragged": False},
        # four answers sampled from one prompt
        {"name": "prefix_4x2k", "op": "prefix", "heads": 0, "sequences": 4, "prefix": 2048, "length": 130, "tokens": 1, "page": 64, "ragged": False},
        # a server whose users share a long system prompt and tools, some slots idle
        {"name": "prefix_64x32k", "op": "prefix", "heads": 0, "sequences": 64, "prefix": 32768, "length": 1021, "tokens": 1, "page": 64, "ragged": True},
        # many short questions on one document, small heads
        {"name": "prefix_192x16k", "op": "prefix", "heads": 1, "sequences": 192, "prefix": 16000, "length": 77, "tokens": 1, "page": 16, "ragged": True},
        # eight speculated tokens of 12 branches of one long conversation
        {"name": "prefix_verify_12x64k", "op": "prefix", "heads": 0, "sequences": 12, "prefix": 65536, "length": 300, "tokens": 8, "page": 128, "ragged": False},
    ]


def draw(rng):
    def spread(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    op = rng.choice(("attention", "attention", "append", "prefix", "prefix"))
    heads = rng.randrange(len(HEADS))
    query, kv, size = HEADS[heads]
    page = rng.choice((16, 32, 64, 128))
    if op == "append":
        sequences = spread(1, 128)
        return {"op": op, "heads": heads, "sequences": sequences, "tokens": spread(1, max(8, 4096 // sequences)), "page": page, "norm": rng.random() < 0.5,
                "interleaved": rng.random() < 0.5, "far": spread(64, 1 << 20)}
    tokens = rng.randint(1, min(8, 64 // (query // kv)))
    if op == "attention":
        sequences = spread(1, 96)
        most = min(131072, int(0.5e9 / (sequences * kv * size * 2)))
        return {"op": op, "heads": heads, "sequences": sequences, "length": spread(tokens, most), "tokens": tokens, "page": page, "ragged": rng.random() < 0.5}
    sequences = spread(2, 256)
    most = min(65536, int(1.5e11 / (4 * sequences * tokens * query * size)))
    length = spread(tokens, max(tokens, min(2048, int(1.0e9 / (sequences * kv * size * 4)))))
    return {"op": op, "heads": heads, "sequences": sequences, "prefix": spread(page, max(page, most)) // page * page, "length": length, "tokens": tokens,
            "page": page, "ragged": rng.random() < 0.5}


def _sequences(case):
    """(tokens behind the prefix with the new ones, new tokens) of every sequence: a function of the case, not of the seed. A ragged batch has idle slots."""
    out = []
    for b in range(case["sequences"]):
        if not case["ragged"]:
            out.append((max(case["length"] - 3 * b, case["tokens"]), case["tokens"]))
            continue
        if b % 9 == 4:
            out.append((0, 0))
            continue
        part = (b * 0.6180339887498949 + 0.37) % 1.0
        new = 1 + (b * 5 + 2) % case["tokens"]
        out.append((max(int(case["length"] * (0.03 + 0.97 * part)), new), new))
    return out


def work(case):
    query, kv, size = HEADS[case["heads"]]
    if case["op"] == "append":
        rows = case["sequences"] * case["tokens"]
        return {"bytes": rows * (2 * (2 * query + 2 * kv) * size + 2 * kv * (size + 1) + 16), "flops": rows * (query + 2 * kv) * size * 10}
    sequences = _sequences(case)
    cached, rows = sum(n for n, _ in sequences), sum(n for _, n in sequences)
    pairs = sum(length * new - new * (new - 1) // 2 for length, new in sequences)
    tables = sum(-(-n // case["page"]) * 4 for n, _ in sequences) + rows * query * size * 4
    if case["op"] == "attention":
        return {"bytes": cached * kv * 2 * (size + 1) + tables, "flops": 4 * pairs * query * size}
    return {"bytes": (case["prefix"] + cached) * kv * size * 4 + tables, "flops": 4 * (pairs + case["prefix"] * rows) * query * size}


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, *shape, type=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(type)


def _codes(g, *shape):
    """E4M3 codes as the cache write leaves them: the largest of a head's elements between 224 and 448."""
    return (torch.randn(shape, generator=g, device=DEVICE) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)


def _scales(g, *shape):
    """Powers of two around 2^-7, as E8M0."""
    return torch.randint(119, 122, shape, generator=g, device=DEVICE, dtype=torch.uint8).view(torch.float8_e8m0fnu)


def _table(g, counts, spare=0, shared=()):
    """Page table [sequences, most] with every sequence's pages anywhere in the cache behind the shared ones; unused entries are -1."""
    total = max(sum(counts), 1) + spare + len(shared)
    order = torch.tensor(sorted(set(range(total)) - set(shared)))
    order = order[torch.randperm(len(order), generator=g, device=DEVICE).cpu()].to(torch.int32)
    table = torch.full((len(counts), len(shared) + max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        if n and shared:
            table[b, :len(shared)] = torch.tensor(shared, dtype=torch.int32)
        table[b, len(shared):len(shared) + n] = order[at:at + n]
        at += n
    return table.to(DEVICE), total


def _starts(sequences):
    starts = [0]
    for _, new in sequences:
        starts.append(starts[-1] + new)
    return torch.tensor(starts, dtype=torch.int32, device=DEVICE)


def _inputs(case, seed):
    g = _generator(seed)
    query, kv, size = HEADS[case["heads"]]
    page = case["page"]
    if case["op"] == "append":
        new = case["tokens"]
        sequences = [(new + 1 + (37 * b + 11) % (4 * page), new) for b in range(case["sequences"])]
        rows = case["sequences"] * new
        table, pages = _table(g, [-(-n // page) for n, _ in sequences], spare=1)
        rotary, sections = ROTARY[size]
        query_gate = _normal(g, rows, query, 2, size)     # the projection's rows hold a head's query and its gate
        first = torch.randint(max(case["far"] - new, 1), (3, case["sequences"], 1), generator=g, device=DEVICE)
        positions = (first + torch.arange(new, device=DEVICE)).reshape(3, rows).to(torch.int32)
        frequencies = (1.0e7 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).to(torch.float32).to(DEVICE)
        state = {"q": query_gate[:, :, 0], "k": _normal(g, rows, kv, size), "v": _normal(g, rows, kv, size, scale=0.7), "positions": positions,
                 "frequencies": frequencies, "sections": sections, "table": table, "starts": _starts(sequences),
                 "lengths": torch.tensor([n for n, _ in sequences], dtype=torch.int32, device=DEVICE),
                 "k_cache": _codes(g, 1, pages, kv, page, size), "v_cache": _codes(g, 1, pages, kv, page, size), "scales": _scales(g, 1, pages, kv, page, 2),
                 "q_out": torch.zeros((rows, query, size), dtype=torch.bfloat16, device=DEVICE), "q_norm": None, "k_norm": None}
        if case["norm"]:
            state["q_norm"] = 1 + _normal(g, size, type=torch.float32, scale=0.1)
            state["k_norm"] = 1 + _normal(g, size, type=torch.float32, scale=0.1)
        return state
    sequences = _sequences(case)
    rows = max(sum(n for _, n in sequences), 1)
    counts = [-(-n // page) for n, _ in sequences]
    state = {"q": _normal(g, rows, query, size, scale=1.5), "starts": _starts(sequences),
             "out": torch.zeros((rows, query, size), dtype=torch.bfloat16, device=DEVICE)}
    if case["op"] == "attention":
        state["table"], pages = _table(g, counts)
        state |= {"k_cache": _codes(g, 1, pages, kv, page, size), "v_cache": _codes(g, 1, pages, kv, page, size), "scales": _scales(g, 1, pages, kv, page, 2)}
        lengths = [n for n, _ in sequences]
    else:
        held = case["prefix"] // page
        everywhere = torch.randperm(held + sum(counts) + 1, generator=g, device=DEVICE).cpu().tolist()
        shared = everywhere[:held]
        state["table"], pages = _table(g, counts, spare=1, shared=shared)
        state |= {"k_cache": _normal(g, 1, pages, kv, page, size), "v_cache": _normal(g, 1, pages, kv, page, size),
                  "prefix_pages": torch.tensor(shared, dtype=torch.int32, device=DEVICE),
                  "prefix_tokens": torch.tensor([case["prefix"]], dtype=torch.int32, device=DEVICE)}
        lengths = [case["prefix"] + n if n else 0 for n, _ in sequences]
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        from augur_v100_b200 import host, kv

        op = case["op"]
        stream = state["stream"] = host.Stream(0)
        query, heads, size = HEADS[case["heads"]]
        if op == "append":
            state["bound"] = kv.KvAppend.bind(
                stream, kv.KvCacheE4m3(state["k_cache"], state["v_cache"], state["scales"]), 0, state["q"], state["k"], state["v"], state["positions"],
                state["frequencies"], state["sections"], state["table"], state["lengths"], state["starts"], interleaved=case["interleaved"],
                q_out=state["q_out"], q_norm=state["q_norm"], k_norm=state["k_norm"], epsilon=EPSILON)
        elif op == "attention":
            plan = state["plan"] = host.Plan(stream, kv.paged_attention_scratch_bytes(query, heads, size, case["tokens"]))
            state["bound"] = kv.PagedAttention.bind(
                plan, kv.KvCacheE4m3(state["k_cache"], state["v_cache"], state["scales"]), 0, state["q"], state["table"], state["lengths"], state["starts"],
                tokens=case["tokens"], out=state["out"])
        else:
            plan = state["plan"] = host.Plan(stream, kv.shared_prefix_attention_scratch_bytes(query, heads, size, state["q"].shape[0], case["tokens"]))
            state["bound"] = kv.SharedPrefixAttention.bind(
                plan, kv.KvCache(state["k_cache"], state["v_cache"]), 0, state["q"], state["table"], state["lengths"], state["starts"],
                state["prefix_pages"], state["prefix_tokens"], tokens=case["tokens"], out=state["out"])
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        bound = state["bound"]
        if op == "append":
            bound.submit()
            return {"q": state["q_out"], "k": state["k_cache"], "v": state["v_cache"], "scales": state["scales"]}
        bound.submit_for_plan()
        return state["out"]
    return {"append": _plain_append, "attention": _plain_attention, "prefix": _plain_prefix}[op](state)


# ---- plain forms -----------------------------------------------------------------------

def _axes(sections, interleaved, device):
    """The axis of every rotary pair: sections one behind the other, or interleaved with the first axis where the others end."""
    pair = torch.arange(sum(sections), device=device)
    if interleaved:
        return torch.where((pair % 3 == 1) & (pair < 3 * sections[1]), 1, torch.where((pair % 3 == 2) & (pair < 3 * sections[2]), 2, 0))
    return (pair >= sections[0]).long() + (pair >= sections[0] + sections[1]).long()


def _slots(state, rows, page):
    """(page, row in the page) of every new token."""
    starts, lengths = state["starts"].long(), state["lengths"].long()
    row = torch.arange(rows, device=starts.device)
    sequence = torch.searchsorted(starts[1:], row, right=True)
    position = lengths[sequence] - (starts[sequence + 1] - row)
    return state["table"][sequence, position // page].long(), position % page


def _quantised(x):
    """Codes and scale byte of every head: the smallest power of two with which the largest element is at most 448."""
    fraction, exponent = torch.frexp(x.abs().amax(-1))
    exponent = (exponent - 9 + (fraction > 0.875).int()).clamp(-60, 60)      # 448 = 0.875 * 2^9
    return torch.ldexp(x, -exponent.unsqueeze(-1)).to(torch.float8_e4m3fn), (exponent + 127).to(torch.uint8)


def _plain_append(state):
    case = state["case"]
    rows = state["q"].shape[0]
    half = sum(state["sections"])
    axes = _axes(state["sections"], case["interleaved"], DEVICE)
    angle = state["positions"][axes].double().T * state["frequencies"].double()
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)

    def rotated(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON) * weight
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1)

    state["q_out"].copy_(rotated(state["q"], state["q_norm"]).to(torch.bfloat16))
    page, offset = _slots(state, rows, case["page"])
    scales = state["scales"].view(torch.uint8)
    keys, key_scales = _quantised(rotated(state["k"], state["k_norm"]))
    values, value_scales = _quantised(state["v"].float())
    state["k_cache"].view(torch.uint8)[0, page, :, offset] = keys.view(torch.uint8)
    state["v_cache"].view(torch.uint8)[0, page, :, offset] = values.view(torch.uint8)
    scales[0, page, :, offset, 0] = key_scales
    scales[0, page, :, offset, 1] = value_scales
    return {"q": state["q_out"], "k": state["k_cache"], "v": state["v_cache"], "scales": state["scales"]}


def _plain_rows(state):
    """(token row of every sequence's i-th new token, whether there is one)."""
    starts = state["starts"].long()
    index = torch.arange(state["case"]["tokens"], device=starts.device)
    live = index < (starts[1:] - starts[:-1])[:, None]
    return torch.where(live, starts[:-1, None] + index, 0), live


def _plain_seen(state, first, keys):
    """Which of `keys` cached tokens from `first` on each new token sees: [sequences, tokens, keys]."""
    starts, lengths = state["starts"].long(), state["lengths"].long()
    index = torch.arange(state["case"]["tokens"], device=starts.device)
    last = lengths[:, None] - (starts[1:] - starts[:-1])[:, None] + index
    return first + torch.arange(keys, device=starts.device) <= last[..., None]


def _plain_attention(state):
    query, kv, size = HEADS[state["case"]["heads"]]
    most = state["case"]["tokens"]
    sequences = state["table"].shape[0]
    pages = state["table"].clamp(min=0).long()
    scales = state["scales"][0].float()
    # (whole bytes are gathered: indexing knows them)
    k = state["k_cache"].view(torch.uint8)[0][pages].view(torch.float8_e4m3fn).float() * scales[pages][..., 0:1]
    v = state["v_cache"].view(torch.uint8)[0][pages].view(torch.float8_e4m3fn).float() * scales[pages][..., 1:2]
    k, v = (x.transpose(1, 2).reshape(sequences, kv, -1, size) for x in (k, v))
    row, live = _plain_rows(state)
    q = state["q"].float()[row].reshape(sequences, most, kv, query // kv, size).permute(0, 2, 1, 3, 4).reshape(sequences, kv, -1, size)
    scores = (q @ k.transpose(-1, -2)) * size ** -0.5
    seen = _plain_seen(state, 0, k.shape[2]).repeat_interleave(query // kv, 1)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    weight = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3.0e38))
    out = (weight @ v) / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = out.reshape(sequences, kv, most, query // kv, size).permute(0, 2, 1, 3, 4).reshape(sequences, most, query, size)
    state["out"][row[live]] = out[live].to(torch.bfloat16)
    return state["out"]


def _plain_prefix(state):
    """The prefix once for all sequences, then every sequence's own tokens, under one softmax."""
    case = state["case"]
    query, kv, size = HEADS[case["heads"]]
    most, group = case["tokens"], query // kv
    sequences = state["table"].shape[0]
    shared = state["prefix_pages"].long()
    row, live = _plain_rows(state)
    q = state["q"].float()[row].reshape(sequences, most, kv, group, size).permute(0, 2, 1, 3, 4).reshape(sequences, kv, -1, size)
    k, v = (state[name][0][shared].float().transpose(0, 1).reshape(kv, -1, size) for name in ("k_cache", "v_cache"))
    together = q.transpose(0, 1).reshape(kv, -1, size)
    scores = ((together @ k.transpose(-1, -2)) * size ** -0.5).reshape(kv, sequences, most * group, -1).transpose(0, 1)
    pages = state["table"][:, shared.shape[0]:].clamp(min=0).long()
    own_k, own_v = (state[name][0][pages].float().transpose(1, 2).reshape(sequences, kv, -1, size) for name in ("k_cache", "v_cache"))
    own_scores = (q @ own_k.transpose(-1, -2)) * size ** -0.5
    seen = _plain_seen(state, case["prefix"], own_k.shape[2]).repeat_interleave(group, 1)[:, None]
    own_scores = own_scores.masked_fill(~seen, -math.inf)
    top = torch.maximum(scores.amax(-1, keepdim=True), own_scores.amax(-1, keepdim=True))
    weight, own_weight = torch.exp(scores - top), torch.exp(own_scores - top)
    total = weight.sum(-1, keepdim=True) + own_weight.sum(-1, keepdim=True)
    out = (weight.transpose(0, 1).reshape(kv, sequences * most * group, -1) @ v).reshape(kv, sequences, most * group, size).transpose(0, 1)
    out = (out + own_weight @ own_v) / total
    out = out.reshape(sequences, kv, most, group, size).permute(0, 2, 1, 3, 4).reshape(sequences, most, query, size)
    state["out"][row[live]] = out[live].to(torch.bfloat16)
    return state["out"]


# ---- definitions in 64 bits --------------------------------------------------------------

def _nearest_e4m3(x):
    """The nearest multiple of 2^(binade - 3), ties to the even one; below 2^-6 of 2^-9."""
    binade = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6) * (1 + 1e-15)))
    step = torch.exp2(binade - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    state = _inputs(case, seed)
    query, kv, size = HEADS[case["heads"]]
    page = case["page"]
    table, lengths, starts = state["table"].tolist(), state["lengths"].tolist(), state["starts"].tolist()
    if case["op"] == "append":
        time, height, width = state["sections"]
        half = time + height + width
        axis = [0] * time + [1] * height + [2] * width
        if case["interleaved"]:
            axis = [1 if i % 3 == 1 and i // 3 < height else 2 if i % 3 == 2 and i // 3 < width else 0 for i in range(half)]
        position = torch.stack([state["positions"][a] for a in axis], 1).double()
        turn = torch.polar(torch.ones_like(position), position * state["frequencies"].double())

        def rotated(x, weight):
            x = x.double()
            if weight is not None:
                x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / size + EPSILON) * weight.double()
            z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn[:, None]
            return torch.cat((z.real, z.imag, x[..., 2 * half:]), -1)

        k, v, scales = state["k_cache"].double(), state["v_cache"].double(), state["scales"].float().double()
        slots = [(table[b][(lengths[b] - starts[b + 1] + row) // page], (lengths[b] - starts[b + 1] + row) % page)
                 for b in range(len(lengths)) for row in range(starts[b], starts[b + 1])]
        at, offset = (torch.tensor(x, device=DEVICE) for x in zip(*slots))
        for held, x, which in ((k, rotated(state["k"], state["k_norm"]), 0), (v, state["v"].double(), 1)):
            power = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 448) - 1e-9).clamp(-60, 60))   # (log2 of a power of two may be an ulp off)
            held[0, at, :, offset] = _nearest_e4m3(x / power)
            scales[0, at, :, offset, which] = power[..., 0]
        return {"q": rotated(state["q"], state["q_norm"]), "k": k, "v": v, "scales": scales}
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device=DEVICE)
    group = query // kv
    for h in range(kv):
        if case["op"] == "prefix":
            first = [state[name][0, state["prefix_pages"].long(), h].reshape(-1, size).double() for name in ("k_cache", "v_cache")]
            skip = state["prefix_pages"].shape[0]
        else:
            first, skip = [torch.zeros((0, size), dtype=torch.float64, device=DEVICE)] * 2, 0
        for b, length in enumerate(lengths):
            new = starts[b + 1] - starts[b]
            if not new:
                continue
            rest = []
            for which, name in enumerate(("k_cache", "v_cache")):
                pages = torch.tensor(table[b][skip:-(-length // page)], device=DEVICE)
                if case["op"] == "attention":
                    x = state[name].view(torch.uint8)[0, pages, h].view(torch.float8_e4m3fn).double()
                    x = x * state["scales"].view(torch.uint8)[0, pages, h, :, which:which + 1].double().sub(127).exp2()
                else:
                    x = state[name][0, pages, h].double()
                rest.append(x.reshape(-1, size)[:length - skip * page])
            rows = slice(starts[b], starts[b + 1])
            q = state["q"][rows, h * group:(h + 1) * group].double()
            s = torch.cat([q @ first[0].T, q @ rest[0].T], -1) / math.sqrt(size)
            seen = torch.arange(length, device=DEVICE) < (length - new + 1 + torch.arange(new, device=DEVICE))[:, None]
            p = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1)
            out[rows, h * group:(h + 1) * group] = p[..., :skip * page] @ first[1] + p[..., skip * page:] @ rest[1]
    return out
