"""Cases of the decoding operators beside the linears: the cache write with rotary positions, attention over the paged cache,
page copies, and log probabilities behind the vocabulary head, each with a plain form in elementary torch operations.

``own`` selects what ``run`` computes with: the plain form, or the library's entry points through the package.
"""
import math

import torch

own = False

DEVICE = "cuda:0"

# (query heads, key-value heads, head size). The first is the full-attention layer of the model this library serves (projections of
# 12288, 1024, 1024 and 6144 rows); the others are generic.
HEADS = ((24, 4, 256), (32, 8, 128), (16, 16, 128), (8, 1, 128), (16, 2, 256))
VOCABULARY = 248320
ROTARY = {256: (64, (11, 11, 10)), 128: (128, (16, 24, 24))}    # rotary size and sections (time, height, width) by head size


def listed():
    return [
        # one user's decoding step, a few thousand tokens in
        {"name": "attention_one_4k", "op": "attention", "heads": 0, "sequences": 1, "length": 4100, "tokens": 1, "page": 64, "ragged": False},
        # a server's decoding step: 64 users, contexts from a few hundred tokens to 8 thousand, some slots idle
        {"name": "attention_64_ragged", "op": "attention", "heads": 0, "sequences": 64, "length": 8191, "tokens": 1, "page": 64, "ragged": True},
        # the fixed batch of eight rows that verifies speculated tokens, 16 thousand tokens in, small pages
        {"name": "attention_verify_8", "op": "attention", "heads": 0, "sequences": 4, "length": 16385, "tokens": 8, "page": 16, "ragged": False},
        # two long documents
        {"name": "attention_long_128", "op": "attention", "heads": 1, "sequences": 2, "length": 131071, "tokens": 1, "page": 128, "ragged": False},
        # the cache write of the verify batch, with head norms
        {"name": "append_8", "op": "append", "heads": 0, "sequences": 1, "tokens": 8, "page": 64, "norm": True, "interleaved": True, "far": 262143},
        # the same for a full server, text and image positions
        {"name": "append_96x5", "op": "append", "heads": 1, "sequences": 96, "tokens": 5, "page": 16, "norm": False, "interleaved": False, "far": 1000003},
        # fork of one conversation: its last page in every full-attention layer
        {"name": "pages_fork", "op": "pages", "heads": 0, "layers": 16, "pages": 64, "pairs": 1, "page": 64},
        # compaction of a cache
        {"name": "pages_compact", "op": "pages", "heads": 0, "layers": 16, "pages": 1024, "pairs": 301, "page": 64},
        # one decoded token with the 20 best alternatives
        {"name": "logprobs_1", "op": "logprobs", "rows": 1, "vocabulary": VOCABULARY, "alternatives": 20, "type": "f32"},
        # the verify batch
        {"name": "logprobs_8", "op": "logprobs", "rows": 8, "vocabulary": VOCABULARY, "alternatives": 20, "type": "f32"},
        # scoring a prompt's chunk
        {"name": "logprobs_509", "op": "logprobs", "rows": 509, "vocabulary": VOCABULARY, "alternatives": 5, "type": "f32"},
        # the same from a BF16 linear with a smaller vocabulary
        {"name": "logprobs_bf16_301", "op": "logprobs", "rows": 301, "vocabulary": 151936, "alternatives": 0, "type": "bf16"},
    ]


def draw(rng):
    def spread(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    op = rng.choice(("attention", "attention", "append", "pages", "logprobs"))
    heads = rng.randrange(len(HEADS))
    query, kv, size = HEADS[heads]
    page = rng.choice((16, 32, 64, 128))
    if op == "attention":
        sequences = spread(1, 96)
        tokens = rng.randint(1, min(8, 64 // (query // kv)))
        most = min(131072, int(1.0e9 / (sequences * kv * size * 4)))
        return {"op": op, "heads": heads, "sequences": sequences, "length": spread(max(tokens, 1), most), "tokens": tokens, "page": page,
                "ragged": rng.random() < 0.5}
    if op == "append":
        return {"op": op, "heads": heads, "sequences": spread(1, 128), "tokens": rng.randint(1, 8), "page": page, "norm": rng.random() < 0.5,
                "interleaved": rng.random() < 0.5, "far": spread(64, 1 << 20)}
    if op == "pages":
        layers = spread(1, 24)
        pages = spread(2, max(2, int(2.0e9 / (layers * kv * page * size * 4))))
        return {"op": op, "heads": heads, "layers": layers, "pages": pages, "pairs": spread(1, max(1, pages // 3)), "page": page}
    vocabulary = spread(17, 262144)
    return {"op": op, "rows": spread(1, max(1, min(4096, int(1.2e8 / vocabulary)))), "vocabulary": vocabulary,
            "alternatives": rng.randint(0, min(32, vocabulary)), "type": rng.choice(("f32", "bf16"))}


def _sequences(case):
    """(cached length with the new tokens, new tokens) of every sequence: a function of the case, not of the seed. A ragged batch has idle slots."""
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
    op = case["op"]
    if op == "logprobs":
        size = case["rows"] * case["vocabulary"]
        return {"bytes": size * (4 if case["type"] == "f32" else 2) + case["rows"] * (12 + 8 * case["alternatives"]), "flops": 8 * size}
    query, kv, size = HEADS[case["heads"]]
    if op == "pages":
        return {"bytes": 2 * 2 * case["layers"] * case["pairs"] * kv * case["page"] * size * 2, "flops": 0}
    if op == "append":
        rows = case["sequences"] * case["tokens"]
        return {"bytes": rows * (2 * 2 * (query + 2 * kv) * size + 16), "flops": rows * (query + kv) * size * 10}
    sequences = _sequences(case)
    cached, rows = sum(n for n, _ in sequences), sum(n for _, n in sequences)
    pairs = sum(length * new - new * (new - 1) // 2 for length, new in sequences)
    return {"bytes": cached * kv * size * 4 + rows * query * size * 4 + sum(-(-n // case["page"]) * 4 for n, _ in sequences), "flops": 4 * pairs * query * size}


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, *shape, type=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(type)


def _table(g, sequences, page, spare=0):
    """Page table [sequences, most] with every sequence's pages anywhere in the cache; unused entries are -1."""
    counts = [-(-n // page) for n, _ in sequences]
    total = max(sum(counts), 1) + spare
    order = torch.randperm(total, generator=g, device=DEVICE).to(torch.int32).cpu()
    table = torch.full((len(sequences), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(DEVICE), total


def _starts(sequences):
    starts = [0]
    for _, new in sequences:
        starts.append(starts[-1] + new)
    return torch.tensor(starts, dtype=torch.int32, device=DEVICE)


def _inputs(case, seed):
    g = _generator(seed)
    if case["op"] == "logprobs":
        kind = torch.float32 if case["type"] == "f32" else torch.bfloat16
        rows, vocabulary = case["rows"], case["vocabulary"]
        logits = _normal(g, rows, vocabulary, type=torch.float32, scale=2.5)
        best = torch.randint(vocabulary, (rows, 3), generator=g, device=DEVICE)
        logits.scatter_add_(1, best, torch.rand((rows, 3), generator=g, device=DEVICE) * 12)
        banned = torch.randint(vocabulary, (max(vocabulary // 64, 1),), generator=g, device=DEVICE)   # tokens that a grammar forbids
        logits[:, banned] = -math.inf
        other = torch.randint(vocabulary, (rows,), generator=g, device=DEVICE)
        pick = torch.rand(rows, generator=g, device=DEVICE) < 0.7
        return {"logits": logits.to(kind), "targets": torch.where(pick, best[:, 0], other).to(torch.int32)}
    query, kv, size = HEADS[case["heads"]]
    page = case["page"]
    if case["op"] == "pages":
        shape = (case["layers"], case["pages"], kv, page, size)
        order = torch.randperm(case["pages"], generator=g, device=DEVICE).cpu().tolist()
        pairs = min(case["pairs"], case["pages"] // 2)
        return {"k": _normal(g, *shape), "v": _normal(g, *shape), "sources": order[:pairs], "destinations": order[pairs:2 * pairs]}
    if case["op"] == "append":
        new = case["tokens"]
        sequences = [(new + 1 + (37 * b + 11) % (4 * page), new) for b in range(case["sequences"])]
        rows = case["sequences"] * new
        table, pages = _table(g, sequences, page, spare=1)
        rotary, sections = ROTARY[size]
        query_gate = _normal(g, rows, query, 2, size)     # the projection's rows hold a head's query and its gate
        first = torch.randint(max(case["far"] - new, 1), (3, case["sequences"], 1), generator=g, device=DEVICE)
        positions = (first + torch.arange(new, device=DEVICE)).reshape(3, rows).to(torch.int32)
        frequencies = (1.0e7 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).to(torch.float32).to(DEVICE)
        state = {"q": query_gate[:, :, 0], "k": _normal(g, rows, kv, size), "v": _normal(g, rows, kv, size), "positions": positions,
                 "frequencies": frequencies, "sections": sections, "table": table, "starts": _starts(sequences),
                 "lengths": torch.tensor([n for n, _ in sequences], dtype=torch.int32, device=DEVICE),
                 "k_cache": _normal(g, 1, pages, kv, page, size), "v_cache": _normal(g, 1, pages, kv, page, size),
                 "q_out": torch.zeros((rows, query, size), dtype=torch.bfloat16, device=DEVICE), "q_norm": None, "k_norm": None}
        if case["norm"]:
            state["q_norm"] = 1 + _normal(g, size, type=torch.float32, scale=0.1)
            state["k_norm"] = 1 + _normal(g, size, type=torch.float32, scale=0.1)
        return state
    sequences = _sequences(case)
    rows = sum(n for _, n in sequences)
    table, pages = _table(g, sequences, page)
    return {"q": _normal(g, max(rows, 1), query, size, scale=1.5), "k_cache": _normal(g, 1, pages, kv, page, size),
            "v_cache": _normal(g, 1, pages, kv, page, size), "table": table, "starts": _starts(sequences),
            "lengths": torch.tensor([n for n, _ in sequences], dtype=torch.int32, device=DEVICE),
            "out": torch.zeros((max(rows, 1), query, size), dtype=torch.bfloat16, device=DEVICE)}


EPSILON = 1e-6


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        from augur_v100_b200 import host, kv

        op = case["op"]
        stream = state["stream"] = host.Stream(0)
        if op == "logprobs":
            plan = state["plan"] = host.Plan(stream, host.logprobs_scratch_bytes(case["rows"], case["alternatives"]))
            state["bound"] = host.TokenLogprobs.bind(plan, state["logits"], state["targets"], case["alternatives"])
        elif op == "pages":
            state["bound"] = kv.KvPageCopy.bind(stream, kv.KvCache(state["k"], state["v"]))
        elif op == "append":
            state["bound"] = kv.KvAppend.bind(
                stream, kv.KvCache(state["k_cache"], state["v_cache"]), 0, state["q"], state["k"], state["v"], state["positions"],
                state["frequencies"], state["sections"], state["table"], state["lengths"], state["starts"], interleaved=case["interleaved"],
                q_out=state["q_out"], q_norm=state["q_norm"], k_norm=state["k_norm"], epsilon=EPSILON)
        else:
            query, heads, size = HEADS[case["heads"]]
            plan = state["plan"] = host.Plan(stream, kv.paged_attention_scratch_bytes(query, heads, size, case["tokens"]))
            state["bound"] = kv.PagedAttention.bind(
                plan, kv.KvCache(state["k_cache"], state["v_cache"]), 0, state["q"], state["table"], state["lengths"], state["starts"],
                tokens=case["tokens"], out=state["out"])
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        bound = state["bound"]
        if op == "logprobs":
            bound.submit_for_plan()
            return {"logprobs": bound.logprobs, "entropy": bound.entropy, "ids": bound.ids, "alternatives": bound.alternative_logprobs}
        if op == "pages":
            bound.submit(state["sources"], state["destinations"])
            return {"k": state["k"].view(torch.int16), "v": state["v"].view(torch.int16)}
        if op == "append":
            bound.submit()
            return {"q": state["q_out"], "k": state["k_cache"], "v": state["v_cache"]}
        bound.submit_for_plan()
        return state["out"]
    return {"logprobs": _plain_logprobs, "pages": _plain_pages, "append": _plain_append, "attention": _plain_attention}[op](state)


# ---- plain forms -----------------------------------------------------------------------

def _plain_logprobs(state):
    x = state["logits"].float()
    k = state["case"]["alternatives"]
    most = x.amax(1, keepdim=True)
    below = x - most
    weight = torch.exp(below)
    total = weight.sum(1, keepdim=True)
    log_total = torch.log(total)
    moment = (weight * torch.where(weight > 0, below, 0.0)).sum(1, keepdim=True)
    entropy = (log_total - moment / total).squeeze(1)
    given = below.gather(1, state["targets"].long().unsqueeze(1))
    # the best, the lowest index first where values are equal: whole numbers that order as (value, -index)
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) - torch.arange(x.shape[1], device=x.device)
    ids = order.topk(k, dim=1).indices
    return {"logprobs": (given - log_total).squeeze(1), "entropy": entropy, "ids": ids.to(torch.int32),
            "alternatives": below.gather(1, ids) - log_total}


def _plain_pages(state):
    k, v = state["k"], state["v"]
    sources = torch.tensor(state["sources"], device=k.device)
    destinations = torch.tensor(state["destinations"], device=k.device)
    k[:, destinations] = k[:, sources]
    v[:, destinations] = v[:, sources]
    return {"k": k.view(torch.int16), "v": v.view(torch.int16)}


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
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1).to(torch.bfloat16)

    state["q_out"].copy_(rotated(state["q"], state["q_norm"]))
    page, offset = _slots(state, rows, case["page"])
    state["k_cache"][0, page, :, offset] = rotated(state["k"], state["k_norm"])
    state["v_cache"][0, page, :, offset] = state["v"]
    return {"q": state["q_out"], "k": state["k_cache"], "v": state["v_cache"]}


def _plain_attention(state):
    query, kv, size = HEADS[state["case"]["heads"]]
    most = state["case"]["tokens"]
    table, lengths, starts = state["table"], state["lengths"].long(), state["starts"].long()
    sequences = table.shape[0]
    pages = table.clamp(min=0).long()
    k = state["k_cache"][0][pages].float().transpose(1, 2).reshape(sequences, kv, -1, size)
    v = state["v_cache"][0][pages].float().transpose(1, 2).reshape(sequences, kv, -1, size)
    new = starts[1:] - starts[:-1]
    index = torch.arange(most, device=table.device)
    live = index < new[:, None]
    row = torch.where(live, starts[:-1, None] + index, 0)
    q = state["q"].float()[row].reshape(sequences, most, kv, query // kv, size).permute(0, 2, 1, 3, 4).reshape(sequences, kv, -1, size)
    scores = (q @ k.transpose(-1, -2)) * size ** -0.5
    key = torch.arange(k.shape[2], device=table.device)
    seen = key < (lengths[:, None, None] - new[:, None, None] + index[:, None] + 1)
    seen = seen.repeat_interleave(query // kv, 1)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3.0e38)
    weight = torch.exp(scores - top)
    v = torch.where((key < lengths[:, None])[:, None, :, None], v, 0.0)
    out = (weight @ v) / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = out.reshape(sequences, kv, most, query // kv, size).permute(0, 2, 1, 3, 4).reshape(sequences, most, query, size)
    state["out"][row[live]] = out[live].to(torch.bfloat16)
    return state["out"]


# ---- definitions in 64 bits --------------------------------------------------------------

def exact(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    op = case["op"]
    if op == "pages":
        return None
    if op == "logprobs":
        out = {"logprobs": [], "entropy": [], "ids": None, "alternatives": []}
        for row, target in zip(state["logits"], state["targets"].tolist()):
            x = row.double()
            logs = x - torch.logsumexp(x, 0)
            p = logs.exp()
            out["logprobs"].append(logs[target])
            out["entropy"].append(-torch.xlogy(p, p).sum())
            out["alternatives"].append(logs.sort(descending=True).values[:case["alternatives"]])
        return {name: None if values is None else torch.stack(values) for name, values in out.items()}
    query, kv, size = HEADS[case["heads"]]
    page = case["page"]
    table, lengths, starts = state["table"].tolist(), state["lengths"].tolist(), state["starts"].tolist()
    if op == "append":
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

        k, v = state["k_cache"].double(), state["v_cache"].double()
        new_k = rotated(state["k"], state["k_norm"])
        for b in range(len(lengths)):
            for row in range(starts[b], starts[b + 1]):
                at = lengths[b] - starts[b + 1] + row
                k[0, table[b][at // page], :, at % page] = new_k[row]
                v[0, table[b][at // page], :, at % page] = state["v"][row].double()
        return {"q": rotated(state["q"], state["q_norm"]), "k": k, "v": v}
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device=DEVICE)
    group = query // kv
    for b, length in enumerate(lengths):
        new = starts[b + 1] - starts[b]
        if not new:
            continue
        pages = torch.tensor(table[b][:-(-length // page)], device=DEVICE)
        for h in range(kv):
            keys = state["k_cache"][0, pages, h].reshape(-1, size)[:length].double()
            values = state["v_cache"][0, pages, h].reshape(-1, size)[:length].double()
            for i in range(new):
                last = length - new + i + 1
                row = starts[b] + i
                q = state["q"][row, h * group:(h + 1) * group].double()
                out[row, h * group:(h + 1) * group] = torch.softmax(q @ keys[:last].T / math.sqrt(size), -1) @ values[:last]
    return out
