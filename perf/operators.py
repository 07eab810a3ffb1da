"""The operators of paged decoding and sampling, as measured cases.

Each case is one pass through one operator:

- "rotation": a model's rotation coefficients by position, at load.
- "append":   head norms, rotation and the cache write of new tokens.
- "attend":   attention of one new token per sequence over paged caches.
- "copy":     pages copied in every layer's caches (fork, compaction).
- "sample":   the next tokens' ids from their logits and given uniforms.

A page buffer is [pages, kv_heads, page_size, head_dim]; a sequence's tokens
lie in the pages its table row names, in order.
"""
import math

import numpy as np
import torch

own = False

EPSILON = 1.0e-5
THETA = 1.0e6
VOCAB = 65536
SCALINGS = {
    "none": {},
    "linear": {"factor": 4.0},
    "ntk": {"factor": 8.0},
    "wavelength": {"factor": 8.0, "original_positions": 8192.0, "low": 1.0, "high": 4.0},
    "yarn": {"factor": 16.0, "original_positions": 8192.0, "low": 1.0, "high": 32.0,
             "magnitude": 1.2772588},
}


def listed():
    return [
        # The rotation of a small model, built when it is loaded.
        {"name": "rotation_2048x64", "kind": "rotation", "positions": 2048, "dim": 64,
         "scaling": "none"},
        # The same for a model stretched to long documents.
        {"name": "rotation_131072x128_yarn", "kind": "rotation", "positions": 131072, "dim": 128,
         "scaling": "yarn"},
        # One new token of one conversation enters its cache.
        {"name": "append_1x32x8x64_f32", "kind": "append", "tokens": 1, "prompt": False,
         "heads": 32, "kv_heads": 8, "dim": 64, "rotary": 64, "interleaved": False, "page": 16,
         "half": False, "context": 2048},
        # A ragged prompt enters its cache, half of each head rotated.
        {"name": "append_prompt_4099x32x8x128_f16", "kind": "append", "tokens": 4099,
         "prompt": True, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 64,
         "interleaved": True, "page": 32, "half": True, "context": 8192},
        # One conversation's next token: latency.
        {"name": "attend_1x2047_32x8x64_f32", "kind": "attend", "sequences": 1, "shortest": 2047,
         "longest": 2047, "heads": 32, "kv_heads": 8, "dim": 64, "page": 16, "half": False},
        # A server's decode step of a small model, conversations of all ages.
        {"name": "attend_96x33-2048_16x8x64_f32", "kind": "attend", "sequences": 96,
         "shortest": 33, "longest": 2048, "heads": 16, "kv_heads": 8, "dim": 64, "page": 64,
         "half": False},
        # The same with wide heads, a half-precision cache and a few long documents.
        {"name": "attend_48x17-8191_32x8x128_f16", "kind": "attend", "sequences": 48,
         "shortest": 17, "longest": 8191, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "half": True},
        # One book-length context.
        {"name": "attend_1x131071_32x8x64_f16", "kind": "attend", "sequences": 1,
         "shortest": 131071, "longest": 131071, "heads": 32, "kv_heads": 8, "dim": 64,
         "page": 16, "half": True},
        # A fork: the page that two sequences would both write, in six layers.
        {"name": "copy_1x12_16x8x64_f32", "kind": "copy", "moved": 1, "buffers": 12,
         "kv_heads": 8, "dim": 64, "page": 16, "half": False},
        # A cache's compaction after many sequences ended.
        {"name": "copy_599x12_16x8x64_f16", "kind": "copy", "moved": 599, "buffers": 12,
         "kv_heads": 8, "dim": 64, "page": 16, "half": True},
        # The next token of one conversation.
        {"name": "sample_1x65536", "kind": "sample", "rows": 1, "width": VOCAB, "rounded": False},
        # A full server's next tokens, each row with its user's settings; the
        # logits come from a head that rounds to bfloat16, so values repeat.
        {"name": "sample_192x65536", "kind": "sample", "rows": 192, "width": VOCAB,
         "rounded": True},
    ]


def _spread(rng, low, high):
    """An integer of [low, high], uniform over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["rotation", "append", "append", "attend", "attend", "attend", "copy",
                       "sample", "sample"])
    if kind == "rotation":
        dim = 2 * _spread(rng, 8, 64)
        return {"kind": kind, "positions": _spread(rng, 64, 131072), "dim": dim,
                "scaling": rng.choice(sorted(SCALINGS))}
    if kind == "sample":
        rows = _spread(rng, 1, 192)
        return {"kind": kind, "rows": rows,
                "width": _spread(rng, 1024, min(200000, 192 * VOCAB // rows)),
                "rounded": rng.random() < 0.5}
    kv_heads, dim = rng.choice([1, 2, 4, 5, 8]), rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    page, half = 1 << rng.randint(3, 8), rng.random() < 0.5
    row = kv_heads * dim * (2 if half else 4)  # one token's bytes of K or V
    if kind == "copy":
        buffers = rng.choice([2, 12, 24])
        moved = _spread(rng, 1, max(2, int(100e6) // (row * page * buffers)))
        return {"kind": kind, "moved": moved, "buffers": buffers, "kv_heads": kv_heads,
                "dim": dim, "page": page, "half": half}
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    if kind == "append":
        most = min(4099, int(30e6) // (4 * dim * (heads + kv_heads)))
        prompt = rng.random() < 0.5
        if not prompt:  # a page of its own for each token
            most = min(most, int(60e6) // (row * page))
        tokens = _spread(rng, 1, max(2, most))
        return {"kind": kind, "tokens": tokens, "prompt": prompt, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rotary": dim // rng.choice([1, 1, 2]),
                "interleaved": rng.random() < 0.5, "page": page, "half": half,
                "context": 8192 if tokens > 1500 else _spread(rng, 2048, 8192)}
    sequences = _spread(rng, 1, 128)
    page = min(page, max(16, int(60e6) // (row * sequences)))
    page = 1 << page.bit_length() - 1
    most = int(250e6) // (2 * row * sequences)  # tokens a sequence may have on average
    longest = _spread(rng, 16, max(16, min(131071, most)))
    return {"kind": kind, "sequences": sequences, "shortest": _spread(rng, 1, longest),
            "longest": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "half": half}


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

    def heads(self, rows, heads, dim):
        """Projections with channels of different gains."""
        return (self.normal(rows, heads, dim) * torch.exp(0.5 * self.normal(dim))).reshape(rows, -1)

    def norm_weight(self, width):
        return 1.0 + 0.1 * self.normal(width)

    def pages(self, count, case, gain=1.0):
        values = gain * self.normal(count, case["kv_heads"], case["page"], case["dim"])
        return values.half() if case["half"] else values


def _lengths(case):
    """The sequences' lengths, evenly spread over the logarithm."""
    n, low, high = case["sequences"], case["shortest"], case["longest"]
    if n == 1:
        return [high]
    return [round(low * (high / low) ** (i / (n - 1))) for i in range(n)]


def _tables(s, lengths, page, longest):
    """(page count, table rows): distinct pages in random order; the entries
    behind a sequence's last page name page 0."""
    need = [-(-n // page) for n in lengths]
    order = s.order(sum(need) + 1)
    columns = -(-longest // page)
    counts = torch.tensor(need, device=order.device)
    first = torch.cumsum(counts, 0) - counts
    column = torch.arange(columns, device=order.device)
    inside = column[None, :] < counts[:, None]
    at = torch.where(inside, first[:, None] + column[None, :], 0)
    return sum(need) + 1, torch.where(inside, order[at], 0)


def _values(case, seed):
    """The case's inputs as torch tensors, by name."""
    s, v, kind = _Source(seed), {}, case["kind"]
    if kind == "rotation":
        # A user's own base frequency: the only value that a rotation has.
        v["theta"] = float(np.float32(THETA * (1.0 + 0.5 * float(s.uniform(1)))))
    elif kind == "append":
        tokens, dim, page = case["tokens"], case["dim"], case["page"]
        v["query"] = s.heads(tokens, case["heads"], dim)
        v["key"] = s.heads(tokens, case["kv_heads"], dim)
        v["value"] = s.heads(tokens, case["kv_heads"], dim)
        v["query_weight"], v["key_weight"] = s.norm_weight(dim), s.norm_weight(dim)
        if case["prompt"]:
            # One sequence's next tokens, behind what it holds already; its
            # table has the pages of its whole context.
            sequences = 1
            start = int(s.whole(0, case["context"] - tokens + 1, 1))
            v["positions"] = torch.arange(start, start + tokens, device=s.device)
            v["rows"] = torch.zeros(tokens, dtype=torch.long, device=s.device)
            count, table = _tables(s, [case["context"]], page, case["context"])
        else:
            # One token of each sequence; all pages but the last ones lie
            # elsewhere, so the table names only those.
            sequences = tokens
            v["positions"] = s.whole(0, case["context"], tokens)
            v["rows"] = torch.arange(tokens, device=s.device)
            count = tokens + 1
            columns = -(-case["context"] // page)
            table = torch.zeros(sequences, columns, dtype=torch.long, device=s.device)
            table[v["rows"], v["positions"] // page] = s.order(count)[:tokens]
        v["table"] = table
        angle = (torch.arange(case["context"], device=s.device).double()[:, None] *
                 torch.pow(THETA, -2.0 * torch.arange(case["rotary"] // 2, device=s.device).double()
                           / case["rotary"]))
        v["rotation"] = torch.cat([torch.cos(angle), torch.sin(angle)], dim=1).float()
        v["key_pages"], v["value_pages"] = s.pages(count, case), s.pages(count, case)
    elif kind == "attend":
        lengths = _lengths(case)
        count, table = _tables(s, lengths, case["page"], case["longest"])
        shuffled = s.order(len(lengths))
        v["lengths"] = torch.tensor(lengths, device=s.device)[shuffled]
        v["table"] = table[shuffled]
        v["query"] = 1.5 * s.normal(case["sequences"], case["heads"] * case["dim"])
        v["key_pages"], v["value_pages"] = s.pages(count, case, 1.2), s.pages(count, case)
    elif kind == "copy":
        moved = case["moved"]
        count = 2 * moved + moved // 4 + 2
        order = s.order(count)
        v["from"], v["to"] = order[:moved], order[moved:2 * moved]
        v["pages"] = [s.pages(count, case) for _ in range(case["buffers"])]
    else:
        rows, width = case["rows"], case["width"]
        logits = 2.5 * s.normal(rows, width)
        logits[:, :: max(1, width // 40)] += 6.0  # the few tokens that fit
        v["logits"] = logits.bfloat16().float() if case["rounded"] else logits
        v["uniforms"] = s.uniform(rows)
        if rows == 1:
            params = torch.tensor([[0.8, 50.0, 0.95, 0.0]], device=s.device)
        else:
            choose = lambda *of: torch.tensor(of, device=s.device)[  # noqa: E731
                s.whole(0, len(of), rows)]
            params = torch.stack([choose(0.0, 0.6, 0.7, 0.8, 1.0, 1.0, 1.2, 1.5),
                                  choose(0.0, 0.0, 20.0, 50.0, 64.0, 1000.0),
                                  choose(0.8, 0.9, 0.95, 1.0, 1.0),
                                  choose(0.0, 0.0, 0.02, 0.05, 0.1)], dim=1).float()
        v["params"] = params
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
        self.state = state

    def __getitem__(self, name):
        buffer, backend = super().__getitem__(name), _backend()
        if buffer.dtype == 0:
            return backend.read(buffer)
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


def _prepare_own(v):
    """The same inputs in the backend's buffers, with the outputs' own."""
    backend, case, s = _backend(), v["case"], {}
    kind = case["kind"]
    if kind == "rotation":
        from runtime_amd.backend import RopeScaling

        s["scaling"] = RopeScaling(case["scaling"], **SCALINGS[case["scaling"]])
        s["rotation"] = backend.allocate_f32((case["positions"], case["dim"]))
    elif kind == "copy":
        for i, pages in enumerate(v["pages"]):
            s["pages%d" % i] = _upload(pages)
        s["pages"] = [s["pages%d" % i] for i in range(case["buffers"])]
        s["from"] = v["from"].cpu().numpy().astype(np.uint32)
        s["to"] = v["to"].cpu().numpy().astype(np.uint32)
    else:
        names = {"append": ("query", "key", "value", "query_weight", "key_weight", "positions",
                            "rows", "table", "rotation", "key_pages", "value_pages"),
                 "attend": ("query", "lengths", "table", "key_pages", "value_pages"),
                 "sample": ("logits", "uniforms", "params")}[kind]
        for name in names:
            s[name] = _upload(v[name])
        if kind == "sample":
            s["tokens"] = backend.allocate_f32((case["rows"],))
        else:
            s["out"] = backend.allocate_f32(s["query"].shape)
            from runtime_amd.backend import GqaSpec, PagedRopeSpec

            shape = (case["heads"], case["kv_heads"], case["dim"])
            s["spec"] = (PagedRopeSpec(*shape, interleaved=case["interleaved"])
                         if kind == "append" else GqaSpec(*shape))
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    backend, case, s = _backend(), state["case"], state["own"]
    kind = case["kind"]
    if kind == "rotation":
        backend.rotation_table(s["rotation"], state["theta"], s["scaling"])
        return Outputs(s, ("rotation",))
    if kind == "append":
        backend.paged_qk_norm_rope(s["out"], s["key_pages"], s["value_pages"], s["query"],
                                   s["key"], s["value"], s["query_weight"], s["key_weight"],
                                   s["rotation"], s["table"], s["rows"], s["positions"],
                                   s["spec"], EPSILON)
        return Outputs(s, ("out", "key_pages", "value_pages"))
    if kind == "attend":
        backend.paged_gqa(s["out"], s["query"], s["key_pages"], s["value_pages"], s["table"],
                          s["lengths"], s["spec"])
        return Outputs(s, ("out",))
    if kind == "copy":
        backend.copy_pages(s["pages"], s["pages"], s["from"], s["to"])
        return Outputs(s, ["pages%d" % i for i in range(case["buffers"])])
    backend.sample_rows(s["tokens"], s["logits"], s["uniforms"], s["params"])
    return Outputs(s, ("tokens",))


# ---- the plain forms ----------------------------------------------------------

def _frequencies(case, theta, device):
    """The rotation's angle per position of each pair, in 64 bits."""
    dim, rule = case["dim"], SCALINGS[case["scaling"]]
    pair = torch.arange(dim // 2, device=device).double()
    factor = rule.get("factor", 1.0)
    if case["scaling"] == "ntk":
        theta = theta * factor ** (dim / (dim - 2))
    plain = torch.exp(-2.0 * pair / dim * math.log(theta))
    if case["scaling"] == "linear":
        return plain / factor
    if case["scaling"] == "wavelength":
        # Waves shorter than the context's `high`-th part stay, those longer
        # than its `low`-th part stretch, a linear blend between.
        turns = rule["original_positions"] * plain / (2.0 * math.pi)
        keep = ((turns - rule["low"]) / (rule["high"] - rule["low"])).clamp(0.0, 1.0)
        return plain * (keep + (1.0 - keep) / factor)
    if case["scaling"] == "yarn":
        # Pairs that turn over `high` times in the context stay, those under
        # `low` times stretch, a ramp over the pair number between.
        at = lambda turns: dim * math.log(  # noqa: E731
            rule["original_positions"] / (2.0 * math.pi * turns)) / (2.0 * math.log(theta))
        first, last = max(math.floor(at(rule["high"])), 0), min(math.ceil(at(rule["low"])), dim - 1)
        ramp = ((pair - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        return plain * (1.0 - ramp + ramp / factor)
    return plain


def _norm_rotate(x, weight, cosine, sine, interleaved):
    """[tokens, heads, dim] normed per head, its first 2 * pairs dims rotated."""
    x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPSILON) * weight
    pairs = cosine.shape[-1]
    cosine, sine = cosine[:, None, :], sine[:, None, :]
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if interleaved:
        first, second = turned[..., 0::2], turned[..., 1::2]
    else:
        first, second = turned[..., :pairs], turned[..., pairs:]
    first, second = first * cosine - second * sine, second * cosine + first * sine
    turned = (torch.stack([first, second], dim=-1).flatten(-2) if interleaved
              else torch.cat([first, second], dim=-1))
    return torch.cat([turned, rest], dim=-1)


def _run_plain(v):
    case = v["case"]
    kind = case["kind"]
    if kind == "rotation":
        device = torch.device("cuda")
        angle = (torch.arange(case["positions"], device=device).double()[:, None] *
                 _frequencies(case, v["theta"], device))
        magnitude = float(np.float32(SCALINGS[case["scaling"]].get("magnitude", 1.0)))
        return {"rotation": (magnitude * torch.cat([torch.cos(angle), torch.sin(angle)],
                                                   dim=1)).float()}
    if kind == "append":
        tokens, dim, page = case["tokens"], case["dim"], case["page"]
        cosine, sine = v["rotation"][v["positions"]].chunk(2, dim=1)
        split = lambda x: x.reshape(tokens, -1, dim)  # noqa: E731
        turn = lambda x, w: _norm_rotate(split(x), w, cosine, sine,  # noqa: E731
                                         case["interleaved"])
        at = v["table"][v["rows"], v["positions"] // page]
        slot = v["positions"] % page
        v["key_pages"][at, :, slot] = turn(v["key"], v["key_weight"]).to(v["key_pages"].dtype)
        v["value_pages"][at, :, slot] = split(v["value"]).to(v["value_pages"].dtype)
        return {"out": turn(v["query"], v["query_weight"]).reshape(tokens, -1),
                "key_pages": v["key_pages"], "value_pages": v["value_pages"]}
    if kind == "attend":
        n, kv_heads, dim = case["sequences"], case["kv_heads"], case["dim"]
        # [sequences, kv_heads, tokens, dim] of every table entry.
        gather = lambda pages: pages[v["table"]].float().transpose(  # noqa: E731
            1, 2).reshape(n * kv_heads, -1, dim)
        query = v["query"].reshape(n * kv_heads, -1, dim)
        scores = torch.bmm(query, gather(v["key_pages"]).transpose(1, 2).contiguous())
        scores = scores.reshape(n, case["heads"], -1) / math.sqrt(dim)
        hidden = torch.arange(scores.shape[2], device=scores.device) >= v["lengths"][:, None]
        scores = scores.masked_fill(hidden[:, None, :], -math.inf)
        weight = torch.exp(scores - scores.amax(dim=2, keepdim=True))
        weight = weight / weight.sum(dim=2, keepdim=True)
        out = torch.bmm(weight.reshape(n * kv_heads, query.shape[1], -1), gather(v["value_pages"]))
        return {"out": out.reshape(n, -1)}
    if kind == "copy":
        for pages in v["pages"]:
            pages[v["to"]] = pages[v["from"]]
        return {"pages%d" % i: pages for i, pages in enumerate(v["pages"])}
    return {"tokens": _sample(v["logits"], v["uniforms"], v["params"])}


def _sample(logits, uniforms, params):
    """The chosen ids, as 32-bit floats.  Sums are in 64 bits: a choice next
    to a border would fall to either side in 32."""
    rows, width = logits.shape
    temperature, top_k, top_p, min_p = params.double().expand(rows, 4).unsqueeze(2).unbind(1)
    value, index = torch.sort(logits, dim=1, descending=True, stable=True)
    value = value.double()
    greedy = temperature == 0.0
    weight = torch.exp((value - value[:, :1]) / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(width, device=logits.device)
    weight = weight.masked_fill((top_k > 0) & (rank >= top_k) | greedy & (rank >= 1), 0.0)
    before = torch.cumsum(weight, 1) - weight
    keep = (before < top_p * weight.sum(dim=1, keepdim=True)) & (weight >= min_p) | (rank == 0)
    # Back in the vocabulary's order.
    weight = torch.zeros_like(weight).scatter_(1, index, weight * keep)
    total = torch.cumsum(weight, 1)
    past = total > uniforms.double()[:, None] * total[:, -1:]
    return torch.where(past, rank, width).amin(dim=1).float()


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "rotation":
        count = float(case["positions"] * case["dim"])
        return {"bytes": 4.0 * count, "flops": 2.0 * count}
    if kind == "sample":
        count = float(case["rows"] * case["width"])
        return {"bytes": 4.0 * count + 24.0 * case["rows"], "flops": 4.0 * count}
    kv_heads, dim, cell = case["kv_heads"], case["dim"], 2 if case["half"] else 4
    if kind == "copy":
        page = kv_heads * dim * cell * case["page"]
        return {"bytes": 2.0 * page * case["moved"] * case["buffers"], "flops": 0.0}
    heads = case["heads"]
    if kind == "append":
        each = (4.0 * dim * (2 * heads + 2 * kv_heads) + 2 * cell * kv_heads * dim +
                4.0 * case["rotary"] + 12.0)
        return {"bytes": case["tokens"] * each + 8.0 * dim,
                "flops": case["tokens"] * 8.0 * dim * (heads + kv_heads)}
    tokens = float(sum(_lengths(case)))
    table = 4.0 * (sum(-(-n // case["page"]) for n in _lengths(case)) + case["sequences"])
    return {"bytes": 2 * cell * kv_heads * dim * tokens + 8.0 * case["sequences"] * heads * dim +
            table, "flops": 4.0 * heads * dim * tokens}


# ---- the same in 64 bits ------------------------------------------------------

def exact(case, seed):
    v, kind = _values(case, seed), case["kind"]
    if kind == "rotation":
        return {"rotation": _exact_rotation(case, v["theta"])}
    if kind == "append":
        return _exact_append(case, v)
    if kind == "attend":
        out = torch.empty(case["sequences"], case["heads"], case["dim"], dtype=torch.float64,
                          device="cuda")
        group = case["heads"] // case["kv_heads"]
        for i, length in enumerate(v["lengths"].tolist()):
            pages = v["table"][i, :-(-length // case["page"])]
            for h in range(case["kv_heads"]):
                key = v["key_pages"][pages, h].double().reshape(-1, case["dim"])[:length]
                value = v["value_pages"][pages, h].double().reshape(-1, case["dim"])[:length]
                mine = slice(h * group, (h + 1) * group)
                query = v["query"][i].double().view(case["heads"], -1)[mine]
                scores = (key @ query.T.contiguous()) * case["dim"] ** -0.5
                out[i, mine] = torch.softmax(scores, dim=0).T.contiguous() @ value
        return {"out": out.reshape(case["sequences"], -1).cpu().numpy()}
    if kind == "copy":
        source, target = v["from"].cpu().numpy(), v["to"].cpu().numpy()
        outs = {}
        for i, pages in enumerate(v["pages"]):
            array = pages.cpu().numpy()
            moved = array[source]
            array[target] = moved
            outs["pages%d" % i] = array
        return outs
    logits, uniforms = v["logits"].cpu().numpy(), v["uniforms"].cpu().numpy().astype(np.float64)
    params = np.broadcast_to(v["params"].cpu().numpy().astype(np.float64), (len(logits), 4))
    return {"tokens": np.array([_exact_token(row.astype(np.float64), u, *p)
                                for row, u, p in zip(logits, uniforms, params)])}


def _exact_rotation(case, theta):
    """Pair by pair, from the rules' own statements."""
    dim, rule = case["dim"], SCALINGS[case["scaling"]]
    factor, context = rule.get("factor", 1.0), rule.get("original_positions")
    table = np.empty((case["positions"], dim))
    position = np.arange(case["positions"], dtype=np.float64)
    for c in range(dim // 2):
        base = theta * factor ** (dim / (dim - 2)) if case["scaling"] == "ntk" else theta
        f = base ** (-2.0 * c / dim)
        if case["scaling"] == "linear":
            f /= factor
        elif case["scaling"] == "wavelength":
            wave = 2.0 * math.pi / f
            if wave > context / rule["low"]:
                f /= factor
            elif wave >= context / rule["high"]:
                blend = (context / wave - rule["low"]) / (rule["high"] - rule["low"])
                f = (1.0 - blend) * f / factor + blend * f
        elif case["scaling"] == "yarn":
            pair_of = lambda n: (dim * math.log(context / (n * 2.0 * math.pi))  # noqa: E731
                                 / (2.0 * math.log(theta)))
            first = max(math.floor(pair_of(rule["high"])), 0)
            last = min(math.ceil(pair_of(rule["low"])), dim - 1)
            stretch = min(max((c - first) / (last - first if last > first else 0.001), 0.0), 1.0)
            f = f / factor * stretch + f * (1.0 - stretch)
        table[:, c], table[:, c + dim // 2] = np.cos(position * f), np.sin(position * f)
    return table * float(np.float32(rule.get("magnitude", 1.0)))


def _exact_append(case, v):
    tokens, dim, pairs = case["tokens"], case["dim"], case["rotary"] // 2
    turn = torch.complex(*v["rotation"][v["positions"]].double().chunk(2, dim=1))[:, None]
    epsilon = float(np.float32(EPSILON))

    def head(x, weight):
        x = x.double().view(tokens, -1, dim)
        x = weight.double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / dim + epsilon)
        if case["interleaved"]:
            z = torch.complex(x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) * turn
            x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2] = z.real, z.imag
        else:
            z = torch.complex(x[..., :pairs], x[..., pairs:2 * pairs]) * turn
            x[..., :pairs], x[..., pairs:2 * pairs] = z.real, z.imag
        return x

    keys, values = v["key_pages"].double(), v["value_pages"].double()
    new_keys, new_values = head(v["key"], v["key_weight"]), v["value"].double().view(tokens, -1, dim)
    where = torch.div(v["positions"], case["page"], rounding_mode="floor")
    page, slot = v["table"][v["rows"], where], v["positions"] - where * case["page"]
    for h in range(case["kv_heads"]):
        keys[page, h, slot], values[page, h, slot] = new_keys[:, h], new_values[:, h]
    host = lambda t: t.cpu().numpy()  # noqa: E731
    return {"out": host(head(v["query"], v["query_weight"]).reshape(tokens, -1)),
            "key_pages": host(keys), "value_pages": host(values)}


def _exact_token(logits, u, temperature, top_k, top_p, min_p):
    if temperature == 0.0:
        return float(np.argmax(logits))
    order = np.argsort(-logits, kind="stable")
    weight = np.exp((logits - logits.max()) / temperature)
    if top_k > 0:
        order = order[:int(top_k)]
    reached = np.cumsum(weight[order])
    order = order[:1 + int(np.searchsorted(reached[:-1], top_p * reached[-1], side="left"))]
    order = np.sort(order[weight[order] >= min_p])
    reached = np.cumsum(weight[order])
    return float(order[np.searchsorted(reached, u * reached[-1], side="right")])
