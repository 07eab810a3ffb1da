"""The operators of drafted decoding and of latent caches, as measured cases.

Each case is one pass through one operator:

- "layout": where the tokens of drafted trees stand, from their parents, once a step.
- "tree":   attention of a run of new tokens per sequence (a tree of drafted
            tokens, or a prompt's) over paged key/value caches.
- "enter":  one shared latent and rotated key per new token into a paged cache.
- "latent": attention of such runs over paged latents.
- "settle": the accepted path of each tree, and its rows moved together in every
            layer's caches.

The run of sequence s is tokens starts[s] .. starts[s + 1] - 1 of the batch.  Its
token i is cached behind the sequence's lengths[s] tokens, at lengths[s] + i, and
parents[t] is the token of the run that it follows (-1: the context alone).  A page
buffer is [pages, kv_heads, page_size, width]; a sequence's tokens lie in the pages
that its table row names, in order.
"""
import math

import numpy as np
import torch

own = False

EPSILON = 1.0e-5
THETA = 1.0e6
VOCAB = 65536


def listed():
    return [
        # One conversation's drafted tree, laid out once for all layers of a step.
        {"name": "layout_1x16", "kind": "layout", "sequences": 1, "run_low": 16, "run_high": 16},
        # A server's trees of many sizes.
        {"name": "layout_96x8-64", "kind": "layout", "sequences": 96, "run_low": 8,
         "run_high": 64},
        # One conversation's tree over its cache: latency.
        {"name": "tree_1x2047+16_32x8x64_f32", "kind": "tree", "sequences": 1, "shortest": 2047,
         "longest": 2047, "run_low": 16, "run_high": 16, "chain": False, "heads": 32,
         "kv_heads": 8, "dim": 64, "page": 16, "half": False},
        # A server's step over wide heads, conversations of all ages.
        {"name": "tree_48x17-8191+4-32_32x8x128_f16", "kind": "tree", "sequences": 48,
         "shortest": 17, "longest": 8191, "run_low": 4, "run_high": 32, "chain": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "half": True},
        # The second half of a long prompt.
        {"name": "prompt_1x2048+2048_32x8x64_f16", "kind": "tree", "sequences": 1,
         "shortest": 2048, "longest": 2048, "run_low": 2048, "run_high": 2048, "chain": True,
         "heads": 32, "kv_heads": 8, "dim": 64, "page": 16, "half": True},
        # One conversation's next token enters its latent cache.
        {"name": "enter_1x16x512+64_f32", "kind": "enter", "tokens": 1, "prompt": False,
         "heads": 16, "rank": 512, "rope": 64, "interleaved": True, "page": 16, "half": False,
         "context": 2048},
        # A ragged prompt enters.
        {"name": "enter_prompt_4099x32x512+64_f16", "kind": "enter", "tokens": 4099,
         "prompt": True, "heads": 32, "rank": 512, "rope": 64, "interleaved": False, "page": 64,
         "half": True, "context": 8192},
        # One conversation's next token over its latents: latency.
        {"name": "latent_1x2047+1_16x512+64_f32", "kind": "latent", "sequences": 1,
         "shortest": 2047, "longest": 2047, "run_low": 1, "run_high": 1, "chain": True,
         "heads": 16, "rank": 512, "rope": 64, "page": 16, "half": False},
        # A server's decode step.
        {"name": "latent_64x100-8191+1_16x512+64_f16", "kind": "latent", "sequences": 64,
         "shortest": 100, "longest": 8191, "run_low": 1, "run_high": 1, "chain": True,
         "heads": 16, "rank": 512, "rope": 64, "page": 64, "half": True},
        # The second half of a prompt, absorbed.
        {"name": "latent_1x1024+1024_32x512+64_f16", "kind": "latent", "sequences": 1,
         "shortest": 1024, "longest": 1024, "run_low": 1024, "run_high": 1024, "chain": True,
         "heads": 32, "rank": 512, "rope": 64, "page": 64, "half": True},
        # A conversation's tree is settled in the key and value pages of six layers.
        {"name": "settle_1x16x12_16x8x64_f32", "kind": "settle", "sequences": 1, "run_low": 16,
         "run_high": 16, "chain": False, "columns": 16, "buffers": 12, "kv_heads": 8, "dim": 64,
         "page": 16, "half": False},
        # A server's.
        {"name": "settle_96x4-32x12_16x8x64_f16", "kind": "settle", "sequences": 96,
         "run_low": 4, "run_high": 32, "chain": False, "columns": 32, "buffers": 12,
         "kv_heads": 8, "dim": 64, "page": 16, "half": True},
    ]


def _spread(rng, low, high):
    """An integer of [low, high], uniform over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["layout", "tree", "tree", "tree", "enter", "latent", "latent", "latent",
                       "settle"])
    page, half = 1 << rng.randint(3, 8), rng.random() < 0.5
    if kind == "layout":
        low = _spread(rng, 1, 64)
        return {"kind": kind, "sequences": _spread(rng, 1, 96), "run_low": low,
                "run_high": rng.randint(low, 64)}
    if kind == "settle":
        low = _spread(rng, 1, 32)
        return {"kind": kind, "sequences": _spread(rng, 1, 96), "run_low": low,
                "run_high": rng.randint(low, 32), "chain": rng.random() < 0.2,
                "columns": rng.choice([4, 8, 32]), "buffers": rng.randint(1, 12),
                "kv_heads": rng.choice([1, 2, 3, 5, 8]), "dim": rng.choice([36, 64, 64]),
                "page": min(page, 32), "half": half}
    rank, rope = rng.choice([128, 256, 512, 512]), rng.choice([32, 64, 64])
    if kind == "enter":
        heads = rng.choice([5, 8, 16, 32])
        prompt = rng.random() < 0.5
        most = 4099 if prompt else int(60e6) // (page * 4 * (rank + rope))
        return {"kind": kind, "tokens": _spread(rng, 1, min(4099, most)), "prompt": prompt,
                "heads": heads, "rank": rank, "rope": rope, "interleaved": rng.random() < 0.5,
                "page": page, "half": half, "context": 8192}
    sequences = _spread(rng, 1, 64)
    if kind == "tree":
        kv_heads, dim = rng.choice([1, 2, 4, 5, 8]), rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        row, most_pairs = 2 * kv_heads * dim * (2 if half else 4), int(12e9) // (heads * dim)
    else:
        heads = rng.choice([5, 8, 16, 16, 20, 32, 64, 128])
        row, most_pairs = (rank + rope) * (2 if half else 4), int(24e9) // (heads * (2 * rank + rope))
    # Tokens of context a sequence may have, by bytes, and by (token, key) pairs.
    longest = _spread(rng, 16, max(16, min(65535, int(120e6) // (row * sequences))))
    chain = rng.random() < 0.5
    most_run = max(1, min(2048 if chain else 64, most_pairs // (sequences * (longest + 2048)),
                          int(120e6) // (row * sequences), 4096 // sequences))
    high = _spread(rng, 1, most_run)
    page = 1 << min(page, max(16, longest // 2)).bit_length() - 1
    case = {"kind": kind, "sequences": sequences, "shortest": _spread(rng, 1, longest),
            "longest": longest, "run_low": _spread(rng, 1, high), "run_high": high,
            "chain": chain, "heads": heads}
    if kind == "tree":
        return {**case, "kv_heads": kv_heads, "dim": dim, "page": page, "half": half}
    return {**case, "rank": rank, "rope": rope, "page": page, "half": half}


# ---- inputs ----------------------------------------------------------------

class _Source:
    """Seeded values, made on the GPU."""

    def __init__(self, seed):
        self.device = torch.device("cuda")
        self.generator = torch.Generator(self.device)
        self.generator.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.generator, device=self.device)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.generator, device=self.device)

    def whole(self, low, high, *shape):
        return torch.randint(low, high, shape, generator=self.generator, device=self.device)

    def order(self, count):
        return torch.randperm(count, generator=self.generator, device=self.device)

    def pages(self, count, heads, page, width, half, gain=1.0):
        values = gain * self.normal(count, heads, page, width)
        return values.half() if half else values


def _even(count, low, high):
    """`count` whole numbers from low to high, evenly spread over the logarithm."""
    if count == 1:
        return [high]
    return [round(low * (high / low) ** (i / (count - 1))) for i in range(count)]


def _tables(s, lengths, page):
    """(page count, table rows): distinct pages in random order; the entries
    behind a sequence's last page name page 0."""
    counts = torch.div(lengths + page - 1, page, rounding_mode="floor")
    total, columns = int(counts.sum()), int(counts.max())
    order = s.order(total + 1)
    first = torch.cumsum(counts, 0) - counts
    column = torch.arange(columns, device=order.device)
    inside = column[None, :] < counts[:, None]
    return total + 1, torch.where(inside, order[torch.where(inside, first[:, None] + column, 0)], 0)


def _runs(s, v, case):
    """The batch's runs: starts, and each token's sequence and number in its run."""
    runs = torch.tensor(_even(case["sequences"], case["run_low"], case["run_high"]),
                        device=s.device)[s.order(case["sequences"])]
    v["starts"] = torch.cat([torch.zeros(1, dtype=torch.long, device=s.device),
                             torch.cumsum(runs, 0)])
    v["runs"], tokens = runs, int(runs.sum())
    v["sequence"] = torch.repeat_interleave(torch.arange(len(runs), device=s.device), runs)
    v["number"] = torch.arange(tokens, device=s.device) - v["starts"][v["sequence"]]
    return tokens


def _parents(s, v, tokens):
    """Trees as drafts grow: a token follows the last one, or any before it."""
    number = v["number"]
    any_of = torch.floor(s.uniform(tokens) * number).long()
    v["parents"] = torch.where(number == 0, -1,
                               torch.where(s.uniform(tokens) < 0.4, number - 1, any_of))


def _ancestors(v, most):
    """[tokens, most]: whether a run's token is the row's own or one of its ancestors."""
    sequences, tokens = len(v["runs"]), len(v["parents"])
    reach = torch.zeros(sequences, most, most, device=v["parents"].device)
    reach[:, torch.arange(most), torch.arange(most)] = 1.0
    child = v["parents"] >= 0
    reach[v["sequence"][child], v["number"][child], v["parents"][child]] = 1.0
    for _ in range(max(1, math.ceil(math.log2(most)))):  # paths of 1, 2, 4, ... steps
        reach = (torch.bmm(reach, reach) > 0).float()
    return reach[v["sequence"], v["number"]] > 0


def _packed(bits):
    """Bit i % 8 of byte i / 8."""
    tokens, count = bits.shape
    wide = torch.zeros(tokens, -(-count // 8) * 8, dtype=torch.uint8, device=bits.device)
    wide[:, :count] = bits
    weight = 2 ** torch.arange(8, device=bits.device)
    return (wide.reshape(tokens, -1, 8) * weight).sum(dim=2).to(torch.uint8)


def _values(case, seed):
    """The case's inputs as torch tensors, by name."""
    s, v, kind = _Source(seed), {}, case["kind"]
    if kind == "enter":
        tokens, page, width = case["tokens"], case["page"], case["rank"] + case["rope"]
        v["query"] = s.normal(tokens, case["heads"] * case["rope"])
        v["latent"] = s.normal(tokens, case["rank"]) * torch.exp(0.5 * s.normal(case["rank"]))
        v["key"] = s.normal(tokens, case["rope"])
        v["weight"] = 1.0 + 0.1 * s.normal(case["rank"])
        if case["prompt"]:
            # One sequence's next tokens, behind what it holds already.
            start = int(s.whole(0, case["context"] - tokens + 1, 1))
            v["positions"] = torch.arange(start, start + tokens, device=s.device)
            v["rows"] = torch.zeros(tokens, dtype=torch.long, device=s.device)
            count, v["table"] = _tables(s, torch.tensor([case["context"]], device=s.device), page)
        else:
            # One token of each sequence; the table names its last page alone.
            v["positions"] = s.whole(0, case["context"], tokens)
            v["rows"] = torch.arange(tokens, device=s.device)
            count = tokens + 1
            v["table"] = torch.zeros(tokens, -(-case["context"] // page), dtype=torch.long,
                                     device=s.device)
            v["table"][v["rows"], v["positions"] // page] = s.order(count)[:tokens]
        angle = (torch.arange(case["context"], device=s.device).double()[:, None] *
                 torch.pow(THETA, -2.0 * torch.arange(case["rope"] // 2, device=s.device).double()
                           / case["rope"]))
        v["rotation"] = torch.cat([torch.cos(angle), torch.sin(angle)], dim=1).float()
        v["pages"] = s.pages(count, 1, page, width, case["half"])
        return v
    tokens = _runs(s, v, case)
    if kind == "layout":
        _parents(s, v, tokens)
        v["lengths"] = s.whole(0, 100000, case["sequences"])
        return v
    if kind == "settle":
        if not case["chain"]:
            _parents(s, v, tokens)
        parents = v["number"] - 1 if case["chain"] else v["parents"]
        v["tokens"] = s.whole(0, VOCAB, tokens)
        # The model goes on to a drafted token most of the time, else to another.
        child = torch.zeros(tokens, dtype=torch.long, device=s.device)
        follows = parents >= 0
        child.scatter_reduce_(0, (v["starts"][v["sequence"]] + parents)[follows],
                              torch.arange(tokens, device=s.device)[follows], "amax")
        drafted = (child > 0) & (s.uniform(tokens) < 0.8)
        v["choices"] = torch.where(drafted, v["tokens"][child], s.whole(0, VOCAB, tokens))
        v["lengths"] = s.whole(0, 2000, case["sequences"])
        # The pages that the runs lie in; the tables' other entries name page 0.
        page = case["page"]
        first = v["lengths"] // page
        need = (v["lengths"] + v["runs"] - 1) // page - first + 1
        _, table = _tables(s, need * page, page)
        count = 1 + sum((n - 1) // page + 2 for n in v["runs"].tolist())  # at most
        columns = (2000 + case["run_high"]) // page + 2
        column = torch.arange(columns, device=s.device)[None, :] - first[:, None]
        inside = (column >= 0) & (column < need[:, None])
        v["table"] = torch.where(inside, table.gather(1, column.clamp(0, table.shape[1] - 1)), 0)
        v["pages"] = [s.pages(count, case["kv_heads"], page, case["dim"], case["half"])
                      for _ in range(case["buffers"])]
        return v
    v["lengths"] = torch.tensor(_even(case["sequences"], case["shortest"], case["longest"]),
                                device=s.device)[s.order(case["sequences"])]
    count, v["table"] = _tables(s, v["lengths"] + v["runs"], case["page"])
    if not case["chain"]:
        _parents(s, v, tokens)
        v["mask"] = _packed(_ancestors(v, case["run_high"]))
    if kind == "tree":
        v["query"] = 1.5 * s.normal(tokens, case["heads"] * case["dim"])
        shape = (count, case["kv_heads"], case["page"], case["dim"], case["half"])
        v["key_pages"], v["value_pages"] = s.pages(*shape, 1.2), s.pages(*shape)
    else:
        v["latent_query"] = s.normal(tokens, case["heads"] * case["rank"])
        v["query"] = 1.5 * s.normal(tokens, case["heads"] * case["rope"])
        v["pages"] = s.pages(count, 1, case["page"], case["rank"] + case["rope"], case["half"])
        v["scale"] = float(np.float32(1.0 / math.sqrt(128 + case["rope"])))
    return v


_SHARED = []


def _backend():
    """The process's one backend instance (and stream)."""
    if not _SHARED:
        from runtime_amd.backend import HipBackend

        _SHARED.append(HipBackend(0))
    return _SHARED[0]


def _upload(tensor):
    from runtime_amd.backend import CACHE

    array = tensor.cpu().numpy()
    if array.dtype == np.uint8:
        return _backend().upload_u8_classified(array.shape, array, CACHE)
    if array.dtype == np.float16:
        shape = array.shape[:-1] + (2 * array.shape[-1],)
        return _backend().upload_u8_classified(shape, array.view(np.uint8), CACHE)
    return _backend().upload_f32_classified(array.shape, array.astype(np.float32), CACHE)


class Outputs(dict):
    """A pass's results by name.  They stay in the backend's buffers, where a
    program's next operation would read them; looking one up reads it back
    (binary16 pages through an f32 copy of them, as their own values)."""

    def __init__(self, state, names):
        super().__init__((name, state[name]) for name in names)

    def __getitem__(self, name):
        buffer, backend = super().__getitem__(name), _backend()
        if buffer.dtype == 0:
            return backend.read(buffer)
        if len(buffer.shape) == 2:
            return backend.read_u8(buffer)
        pages, heads, size, width = buffer.shape
        wide = backend.alloc_pages(pages, heads, size, width // 2)
        every = range(pages)
        backend.copy_pages([wide], [buffer], every, every)
        return backend.read(wide).astype(np.float16)


def prepare(case, seed):
    state = {"case": case, **_values(case, seed)}
    if own:
        state["own"] = _prepare_own(state)
    return state


INPUTS = {"layout": ("starts", "parents", "lengths"),
          "tree": ("query", "key_pages", "value_pages", "table", "starts", "lengths", "mask"),
          "enter": ("query", "latent", "key", "weight", "rotation", "table", "rows", "positions",
                    "pages"),
          "latent": ("latent_query", "query", "pages", "table", "starts", "lengths", "mask"),
          "settle": ("tokens", "choices", "starts", "parents", "lengths", "table")}


def _prepare_own(v):
    """The same inputs in the backend's buffers, with the outputs' own."""
    backend, case = _backend(), v["case"]
    kind, sequences = case["kind"], case.get("sequences")
    s = {name: _upload(v[name]) if name in v else None for name in INPUTS[kind]}
    if kind == "layout":
        tokens = len(v["parents"])
        for name in ("sequences", "positions", "places"):
            s[name] = backend.allocate_f32((tokens,))
        s["mask"] = _upload(torch.zeros(tokens, -(-case["run_high"] // 8), dtype=torch.uint8))
    elif kind == "settle":
        for i, pages in enumerate(v["pages"]):
            s["pages%d" % i] = _upload(pages)
        s["pages"] = [s["pages%d" % i] for i in range(case["buffers"])]
        s["emitted"] = backend.allocate_f32((sequences, case["columns"]))
        s["counts"], s["next"] = (backend.allocate_f32((sequences,)) for _ in range(2))
    else:
        s["out"] = backend.allocate_f32(s["latent_query" if kind == "latent" else "query"].shape)
        if kind == "tree":
            from runtime_amd.backend import GqaSpec

            s["spec"] = GqaSpec(case["heads"], case["kv_heads"], case["dim"])
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    backend, case, s = _backend(), state["case"], state["own"]
    kind = case["kind"]
    if kind == "layout":
        backend.draft_layout(s["sequences"], s["positions"], s["places"], s["mask"], s["starts"],
                             s["parents"], s["lengths"])
        return Outputs(s, ("sequences", "positions", "places", "mask"))
    if kind == "tree":
        backend.paged_tree_gqa(s["out"], s["query"], s["key_pages"], s["value_pages"], s["table"],
                               s["starts"], s["lengths"], s["mask"], s["spec"])
        return Outputs(s, ("out",))
    if kind == "enter":
        backend.paged_latent_append(s["out"], s["pages"], s["query"], s["latent"], s["key"],
                                    s["weight"], s["rotation"], s["table"], s["rows"],
                                    s["positions"], None, case["heads"], case["interleaved"],
                                    EPSILON)
        return Outputs(s, ("out", "pages"))
    if kind == "latent":
        backend.paged_latent_attention(s["out"], s["latent_query"], s["query"], s["pages"],
                                       s["table"], s["starts"], s["lengths"], s["mask"],
                                       case["heads"], state["scale"])
        return Outputs(s, ("out",))
    backend.settle_drafts(s["emitted"], s["counts"], s["next"], s["pages"], s["tokens"],
                          s["choices"], s["starts"], s["parents"], s["lengths"], s["table"])
    return Outputs(s, ["emitted", "counts", "next"] +
                   ["pages%d" % i for i in range(case["buffers"])])


# ---- the plain forms ----------------------------------------------------------

def _rotate(x, cosine, sine, interleaved):
    """[tokens, heads, rope]."""
    pairs = cosine.shape[-1]
    cosine, sine = cosine[:, None, :], sine[:, None, :]
    if interleaved:
        first, second = x[..., 0::2], x[..., 1::2]
    else:
        first, second = x[..., :pairs], x[..., pairs:]
    first, second = first * cosine - second * sine, second * cosine + first * sine
    return (torch.stack([first, second], dim=-1).flatten(-2) if interleaved
            else torch.cat([first, second], dim=-1))


def _admitted(v, case, keys):
    """[sequences, longest run, keys]: whether a run's token attends a key."""
    most, device = case["run_high"], v["starts"].device
    key, number = torch.arange(keys, device=device), torch.arange(most, device=device)
    at = key[None, :] - v["lengths"][:, None]  # the run's token that a key is
    inside = (at >= 0) & (at < v["runs"][:, None])
    if case["chain"]:
        run = at[:, None, :] <= number[None, :, None]
    else:
        token = (v["starts"][:-1, None] + number).clamp(max=len(v["mask"]) - 1)
        bits = v["mask"][token][:, :, torch.arange(8 * v["mask"].shape[1], device=device) // 8]
        bits = (bits >> (torch.arange(bits.shape[2], device=device) % 8)) & 1
        run = bits.gather(2, at.clamp(0, bits.shape[2] - 1)[:, None, :].expand(-1, most, -1)) > 0
    return (at < 0)[:, None, :] | inside[:, None, :] & run


def _attend(v, case, query, key, value, scale):
    """query [tokens, kv_heads, group, d], key and value [sequences, kv_heads, keys, d]."""
    sequences, kv_heads, keys = key.shape[:3]
    most, group = case["run_high"], query.shape[2]
    token = (v["starts"][:-1, None] + torch.arange(most, device=query.device)).clamp(
        max=len(query) - 1)
    rows = query[token].permute(0, 2, 1, 3, 4).reshape(sequences * kv_heads, most * group, -1)
    scores = torch.bmm(rows, key.reshape(sequences * kv_heads, keys, -1).transpose(1, 2)
                       .contiguous()) * scale
    scores = scores.reshape(sequences, kv_heads, most, group, keys)
    scores = scores.masked_fill(~_admitted(v, case, keys)[:, None, :, None, :], -math.inf)
    weight = torch.exp(scores - scores.amax(dim=4, keepdim=True).clamp(min=-1e30))
    total = weight.sum(dim=4, keepdim=True)
    weight = weight / torch.where(total > 0, total, 1.0)
    out = torch.bmm(weight.reshape(sequences * kv_heads, most * group, keys),
                    value.reshape(sequences * kv_heads, keys, -1))
    out = out.reshape(sequences, kv_heads, most, group, -1).transpose(1, 2)
    return out[v["sequence"], v["number"]].reshape(len(query), -1)


def _gathered(pages, table):
    """[sequences, kv_heads, keys, width] of every table entry."""
    x = pages[table].float().transpose(1, 2)
    return x.reshape(*x.shape[:2], -1, x.shape[-1])


def _run_plain(v):
    case = v["case"]
    kind = case["kind"]
    if kind == "layout":
        bits = _ancestors(v, case["run_high"])
        base = v["lengths"][v["sequence"]]
        return {"sequences": v["sequence"].float(),
                "positions": (base + bits.sum(dim=1) - 1).float(),
                "places": (base + v["number"]).float(), "mask": _packed(bits)}
    if kind == "tree":
        query = v["query"].reshape(len(v["query"]), case["kv_heads"], -1, case["dim"])
        return {"out": _attend(v, case, query, _gathered(v["key_pages"], v["table"]),
                               _gathered(v["value_pages"], v["table"]),
                               1.0 / math.sqrt(case["dim"]))}
    if kind == "latent":
        tokens, heads = len(v["query"]), case["heads"]
        query = torch.cat([v["latent_query"].reshape(tokens, heads, -1),
                           v["query"].reshape(tokens, heads, -1)], dim=2)
        keys = _gathered(v["pages"], v["table"])
        return {"out": _attend(v, case, query[:, None], keys,
                               keys[..., :case["rank"]].contiguous(), v["scale"])}
    if kind == "enter":
        tokens, page = case["tokens"], case["page"]
        cosine, sine = v["rotation"][v["positions"]].chunk(2, dim=1)
        latent = v["latent"] * torch.rsqrt(v["latent"].square().mean(dim=1, keepdim=True) +
                                           EPSILON) * v["weight"]
        key = _rotate(v["key"][:, None], cosine, sine, case["interleaved"])[:, 0]
        at = v["table"][v["rows"], v["positions"] // page]
        v["pages"][at, 0, v["positions"] % page] = torch.cat([latent, key], dim=1).to(
            v["pages"].dtype)
        query = _rotate(v["query"].reshape(tokens, case["heads"], -1), cosine, sine,
                        case["interleaved"])
        return {"out": query.reshape(tokens, -1), "pages": v["pages"]}
    return _settle(v, case)


def _settle(v, case):
    sequences, most, columns = case["sequences"], case["run_high"], case["columns"]
    device, page = v["starts"].device, case["page"]
    number = torch.arange(most, device=device)
    inside = number[None, :] < v["runs"][:, None]
    token = (v["starts"][:-1, None] + number).clamp(max=len(v["tokens"]) - 1)
    parents = (number - 1).expand(sequences, -1) if case["chain"] else v["parents"][token]
    tokens, choices = v["tokens"][token], v["choices"][token]
    at = torch.zeros(sequences, dtype=torch.long, device=device)
    going = torch.ones(sequences, dtype=torch.bool, device=device)
    row = torch.arange(sequences, device=device)
    emitted = torch.full((sequences, columns), -1, device=device)
    counts = torch.zeros(sequences, dtype=torch.long, device=device)
    last = torch.full((sequences,), -1, device=device)
    for step in range(columns):
        # The path's token of this step moves to its place.
        if step:
            source = v["lengths"] + torch.where(going, at, 0)
            target = v["lengths"] + torch.where(going, step, 0)
            from_page = v["table"][row, source // page]
            to_page = v["table"][row, target // page]
            for pages in v["pages"]:
                pages[to_page, :, target % page] = pages[from_page, :, source % page]
        choice = choices[row, at]
        emitted[:, step] = torch.where(going, choice, -1)
        last = torch.where(going, choice, last)
        counts = counts + going
        fits = (inside & (parents == at[:, None]) & (tokens == choice[:, None]) &
                (number[None, :] > at[:, None]))
        first = torch.where(fits, number, most).amin(dim=1)
        going = going & (first < most)
        at = torch.where(going, first, at)
    return {"emitted": emitted.float(), "counts": counts.float(), "next": last.float(),
            **{"pages%d" % i: pages for i, pages in enumerate(v["pages"])}}


# ---- what a pass cannot do without ------------------------------------------

def _pairs(case):
    """(tokens, keys, admitted (token, key) pairs) of a case's runs, the context and the
    runs paired in order, half of a run's earlier tokens admitted."""
    lengths = _even(case["sequences"], case["shortest"], case["longest"])
    runs = _even(case["sequences"], case["run_low"], case["run_high"])
    return (float(sum(runs)), float(sum(lengths) + sum(runs)),
            float(sum(n * (mean + 0.5 * (n + 1)) for n, mean in
                      ((n, sum(lengths) / len(lengths)) for n in runs))))


def work(case):
    kind, cell = case["kind"], 2 if case.get("half") else 4
    if kind == "layout":
        tokens = float(sum(_even(case["sequences"], case["run_low"], case["run_high"])))
        return {"bytes": tokens * (16.0 + -(-case["run_high"] // 8)) + 8.0 * case["sequences"],
                "flops": 4.0 * tokens}
    if kind == "enter":
        rank, rope, heads = case["rank"], case["rope"], case["heads"]
        each = 4.0 * (rank + rope + 2 * heads * rope + rope + 3) + cell * (rank + rope)
        return {"bytes": case["tokens"] * each + 4.0 * rank,
                "flops": case["tokens"] * (4.0 * rank + 3.0 * rope * (heads + 1))}
    if kind == "settle":
        # Three rows of a run on average are moved.
        tokens = float(sum(_even(case["sequences"], case["run_low"], case["run_high"])))
        moved = sum(min(3, n - 1) for n in _even(case["sequences"], case["run_low"],
                                                 case["run_high"]))
        return {"bytes": 12.0 * tokens + 4.0 * case["sequences"] * (case["columns"] + 4) +
                2.0 * moved * case["buffers"] * case["kv_heads"] * case["dim"] * cell,
                "flops": 0.0}
    tokens, keys, pairs = _pairs(case)
    table = 4.0 * keys / case["page"] + 12.0 * case["sequences"]
    mask = 0.0 if case["chain"] else tokens * -(-case["run_high"] // 8)
    if kind == "tree":
        heads, dim = case["heads"], case["dim"]
        return {"bytes": 2.0 * cell * case["kv_heads"] * dim * keys + 8.0 * tokens * heads * dim +
                table + mask, "flops": 4.0 * heads * dim * pairs}
    heads, rank, rope = case["heads"], case["rank"], case["rope"]
    return {"bytes": cell * (rank + rope) * keys + 4.0 * tokens * heads * (2 * rank + rope) +
            table + mask, "flops": 2.0 * heads * (2 * rank + rope) * pairs}


# ---- the same in 64 bits ------------------------------------------------------

def _chain_of(parents, i):
    """A run's token and its ancestors."""
    found = []
    while i >= 0:
        found.append(i)
        i = int(parents[i])
    return found


def _exact_attend(case, v, query, key_of, scale):
    """query(first, last, kv head) and key_of(pages, kv head) -> (keys, values) in 64 bits."""
    kv_heads = case.get("kv_heads", 1)
    starts, outs = v["starts"].tolist(), []
    for s, length in enumerate(v["lengths"].tolist()):
        n = starts[s + 1] - starts[s]
        pages = v["table"][s, :-(-(length + n) // case["page"])]
        seen = torch.ones(n, length + n, dtype=torch.bool, device="cuda")
        if case["chain"]:
            seen[:, length:] = torch.tril(seen[:, length:])
        else:
            parents, tree = v["parents"][starts[s]:starts[s + 1]].tolist(), np.zeros((n, n), bool)
            for i in range(n):
                tree[i, _chain_of(parents, i)] = True
            seen[:, length:] = torch.from_numpy(tree).cuda()
        heads = []
        for h in range(kv_heads):
            key, value = (x[:length + n] for x in key_of(pages, h))
            rows = query(starts[s], starts[s + 1], h)  # [group, n, d]
            score = (rows @ key.T.contiguous()) * scale
            weight = torch.softmax(score.masked_fill(~seen, -math.inf), dim=2)
            heads.append(weight @ value)
        outs.append(torch.cat(heads).transpose(0, 1).reshape(n, -1))
    return {"out": torch.cat(outs).cpu().numpy()}


def exact(case, seed):
    v, kind = _values(case, seed), case["kind"]
    if kind == "tree":
        dim, group = case["dim"], case["heads"] // case["kv_heads"]

        def query(first, last, h):
            x = v["query"][first:last].double().reshape(last - first, case["heads"], dim)
            return x[:, h * group:(h + 1) * group].transpose(0, 1).contiguous()

        def keys(pages, h):
            return tuple(v[name][pages, h].double().reshape(-1, dim)
                         for name in ("key_pages", "value_pages"))

        return _exact_attend(case, v, query, keys, dim ** -0.5)
    if kind == "latent":
        rank, heads = case["rank"], case["heads"]

        def query(first, last, h):
            parts = [v[name][first:last].double().reshape(last - first, heads, -1)
                     for name in ("latent_query", "query")]
            return torch.cat(parts, dim=2).transpose(0, 1).contiguous()

        def keys(pages, h):
            x = v["pages"][pages, 0].double().reshape(-1, rank + case["rope"])
            return x, x[:, :rank].contiguous()

        return _exact_attend(case, v, query, keys, v["scale"])
    host = lambda t: t.cpu().numpy()  # noqa: E731
    if kind == "enter":
        tokens, rank, pairs = case["tokens"], case["rank"], case["rope"] // 2
        turn = torch.complex(*v["rotation"][v["positions"]].double().chunk(2, dim=1))[:, None]

        def turned(x):
            x = x.double().reshape(tokens, -1, 2 * pairs)
            if case["interleaved"]:
                return torch.view_as_real(torch.view_as_complex(
                    x.reshape(tokens, -1, pairs, 2).contiguous()) * turn).reshape(x.shape)
            z = torch.complex(x[..., :pairs].contiguous(), x[..., pairs:].contiguous()) * turn
            return torch.cat([z.real, z.imag], dim=2)

        latent = v["latent"].double()
        latent = v["weight"].double() * latent / torch.sqrt(
            latent.pow(2).sum(1, keepdim=True) / rank + float(np.float32(EPSILON)))
        pages = v["pages"].double()
        where = torch.div(v["positions"], case["page"], rounding_mode="floor")
        page, slot = v["table"][v["rows"], where], v["positions"] - where * case["page"]
        pages[page, 0, slot, :rank] = latent
        pages[page, 0, slot, rank:] = turned(v["key"])[:, 0]
        return {"out": host(turned(v["query"]).reshape(tokens, -1)), "pages": host(pages)}
    starts, lengths = v["starts"].tolist(), v["lengths"].tolist()
    number = v["number"].tolist()
    parents = v["parents"].tolist() if "parents" in v else [i - 1 for i in number]
    if kind == "layout":
        mask = np.zeros((starts[-1], -(-case["run_high"] // 8)), np.uint8)
        outs = np.zeros((3, starts[-1]))
        for s, length in enumerate(lengths):
            mine = parents[starts[s]:starts[s + 1]]
            for i in range(len(mine)):
                path = _chain_of(mine, i)
                for j in path:
                    mask[starts[s] + i, j >> 3] |= 1 << (j & 7)
                outs[:, starts[s] + i] = s, length + len(path) - 1, length + i
        return {"sequences": outs[0], "positions": outs[1], "places": outs[2], "mask": mask}
    tokens, choices = v["tokens"].tolist(), v["choices"].tolist()
    emitted = np.full((len(lengths), case["columns"]), -1.0)
    counts, last = np.zeros(len(lengths)), np.full(len(lengths), -1.0)
    arrays, table, page = [host(p).copy() for p in v["pages"]], host(v["table"]), case["page"]
    for s, length in enumerate(lengths):
        first, path = starts[s], [0]
        while len(path) < case["columns"]:
            fits = [i for i in range(path[-1] + 1, starts[s + 1] - first)
                    if parents[first + i] == path[-1] and tokens[first + i] == choices[first + path[-1]]]
            if not fits:
                break
            path.append(fits[0])
        for k, i in enumerate(path):
            emitted[s, k] = choices[first + i]
            a, b = length + i, length + k
            for array in arrays:
                array[table[s, b // page], :, b % page] = array[table[s, a // page], :, a % page]
        counts[s], last[s] = len(path), emitted[s, len(path) - 1]
    return {"emitted": emitted, "counts": counts, "next": last,
            **{"pages%d" % i: array for i, array in enumerate(arrays)}}
