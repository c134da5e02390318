"""Timed cases of the operators of a key/value cache in 4 bits whose tables are built on the GPU: the tables and slots of a step from
the requests' lengths (`tables`), keys and values into the cache and out of it again (`cache`), attention of sequences that bring one
token (`decode`) and of portions of prompts (`prompt`) over it.

The cache. A token's key (and value) of one kv head is `head_dim` numbers, padded with zeros to whole 64s, in groups of 32. Of a group,
with lo = min(0, its least) and hi = max(0, its largest):

    s = (hi - lo) / 15 in 32 bits, at least 2^-100, rounded up to three significant bits (4, 5, 6 or 7 times a power of two)
    z = round(-lo / s),   code = clamp(round(x / s) + z, 0, 15)      (ties to even),   what it stands for: s (code - z)

so that every value it stands for is a bfloat16 number. A token's codes of a head lie in padded / 2 bytes, dimension d in byte d // 2,
the even one in the low bits; a group's 16-bit word holds s as a bfloat16 number (whose low five bits are zero) and z in its low four
bits. Where a key or value of a token and head has a number that is not finite, or one of magnitude 2^120 or more, all its key words
are NaN (0x7fc0), its value words and all its codes zero.
Planes: codes uint8 [pages, kv_heads, page_size, padded / 2], words int16 [pages, kv_heads, page_size, padded / 32].
"""
import math

import torch

own = False

PAGE = 16
CODES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    def tables(name, seqs, rows, context, columns):
        return {"name": name, "kind": "tables", "seqs": seqs, "rows": rows, "context": context, "columns": columns, "page": PAGE}

    def cache(name, rows, kv_heads, head_dim, dtype="bfloat16", page=PAGE):
        return {"name": name, "kind": "cache", "rows": rows, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page}

    def attend(name, kind, seqs, queries, context, heads, kv_heads, head_dim, ragged=False, dtype="bfloat16", page=PAGE, window=0):
        return {"name": name, "kind": kind, "seqs": seqs, "queries": queries, "context": context, "ragged": ragged, "heads": heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page, "window": window}
    return [
        # A decode step of 64 requests: one slot each, and their block tables.
        tables("tables_decode_64", 64, 64, 4096, 256),
        # A step of a large server: 512 requests, of which some bring portions of prompts.
        tables("tables_mixed_512", 512, 16384, 8192, 1024),
        # The newest token of eight requests, the smallest call.
        cache("cache_8", 8, 8, 128),
        # A step of long prompts.
        cache("cache_8192", 8192, 8, 128),
        # The 32-bit path, a head size that fills no whole 64, an odd page size and an odd number of rows.
        cache("cache_f32_2049", 2049, 5, 96, dtype="float32", page=12),
        # One user waiting for the next token at the benchmark's context.
        attend("decode_1", "decode", 1, 1, 4096, 32, 8, 128),
        # Eight requests at the benchmark's longest context.
        attend("decode_8_32k", "decode", 8, 1, 32768, 32, 8, 128),
        # A busy server, contexts of every length.
        attend("decode_64", "decode", 64, 1, 4096, 32, 8, 128, ragged=True),
        # The 32-bit path: a small model, pages of eight, a window.
        attend("decode_f32", "decode", 5, 1, 1531, 12, 4, 64, ragged=True, dtype="float32", page=8, window=1000),
        # A prompt in one step.
        attend("prompt_2048", "prompt", 1, 2048, 2048, 32, 8, 128),
        # Portions of four prompts behind long contexts.
        attend("prompt_4_portions", "prompt", 4, 512, 8192, 16, 4, 64, ragged=True),
        # The 32-bit path: three short prompts of odd lengths.
        attend("prompt_f32", "prompt", 3, 131, 517, 8, 2, 96, ragged=True, dtype="float32", page=12),
    ]


def draw(rng):
    """One more case of the same ranges: sizes even over their logarithm, no case larger than the largest listed of its kind."""
    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(["tables", "cache", "decode", "prompt"])
    if kind == "tables":
        seqs, page = size(1, 512), rng.choice([8, 16, 32, 48])
        context = size(64, 8192)
        return {"kind": kind, "seqs": seqs, "rows": seqs + size(1, 16384 - seqs), "context": context,
                "columns": -(-context // page) + rng.randrange(0, 9), "page": page}
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    page = rng.choice([8, 12, 16, 16, 32, 64])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8])
    if kind == "cache":
        return {"kind": kind, "rows": size(1, 8192 * 1024 // (kv_heads * head_dim * (2 if dtype == "float32" else 1))), "kv_heads": kv_heads,
                "head_dim": head_dim, "dtype": dtype, "page": page}
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    window = rng.choice([0, 0, 0, 512, 777])
    if kind == "decode":
        seqs = size(1, 64)
        context = size(1, min(32768, 8 * 32768 * 1024 // (seqs * kv_heads * head_dim)))
        queries = 1
    else:
        seqs = size(1, 8)
        most = 2048 * 32 * 128 // (seqs * heads * head_dim)     # queries at contexts of 2,048
        queries = size(2, max(2, min(2048, most)))
        context = queries + size(1, max(2, min(8192, 2048 * most // queries // (4 if dtype == "float32" else 1))))
    return {"kind": kind, "seqs": seqs, "queries": queries, "context": context, "ragged": rng.random() < 0.5, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page, "window": window}


# ---- inputs

def _padded(head_dim):
    return -(-head_dim // 64) * 64


def _quantise(k, v):
    """Keys and values [..., head_dim] to (codes, words) of each, as the cache holds them."""
    pad = _padded(k.shape[-1]) - k.shape[-1]
    bad = ~((k.float().abs() < 2.0 ** 120).all(-1) & (v.float().abs() < 2.0 ** 120).all(-1))
    out = []
    for x, word in ((k, 0x7fc0), (v, 0)):
        x = torch.nn.functional.pad(torch.where(bad[..., None], torch.zeros((), device=x.device), x.float()), (0, pad))
        g = x.unflatten(-1, (-1, 32))
        lo, hi = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
        # (divided by a tensor: by a plain number torch multiplies with its reciprocal)
        least = ((hi - lo) / torch.full((), 15.0, device=x.device)).clamp(min=2.0 ** -100)
        bits = (least.view(torch.int32) + 0x1fffff) & ~0x1fffff
        s = bits.view(torch.float32)
        z = torch.round(-lo / s)
        c = (torch.round(g / s[..., None]) + z[..., None]).clamp(0, 15).to(torch.uint8)
        c = torch.where(bad[..., None, None], torch.zeros((), dtype=torch.uint8, device=c.device), c).flatten(-2)
        w = torch.where(bad[..., None], torch.full((), word, dtype=torch.int32, device=c.device), (bits >> 16) | z.int())
        out.append((c[..., 0::2] | (c[..., 1::2] << 4), w.to(torch.int16)))
    return out


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _lens(gen, case):
    """Contexts: the longest first, the others down to an eighth of it where the batch is ragged."""
    n, longest = case["seqs"], case["context"]
    if not case.get("ragged", True) or n == 1:
        return torch.full((n,), longest, device="cuda")
    low = max(case.get("queries", 1), longest // 8, 1)
    lens = torch.randint(min(low, longest), longest + 1, (n,), generator=gen, device="cuda")
    lens[0] = longest
    return lens


def _queries(case):
    """How many tokens each sequence brings: all alike, or from the most down to two."""
    n, most = case["seqs"], case["queries"]
    if not case["ragged"] or n == 1 or most == 1:
        return [most] * n
    return [max(2, most - i * (most - 2) // (n - 1)) for i in range(n)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    page = case["page"]
    if case["kind"] == "tables":
        n, columns = case["seqs"], case["columns"]
        lens = _lens(gen, case)
        # every request brings a token, and the rest of the rows go to those that bring portions
        extra = case["rows"] - n
        share = torch.rand(n, generator=gen, device="cuda") ** 4
        counts = 1 + torch.floor(share / share.sum() * extra).long()
        counts = torch.minimum(counts, lens)
        held = lens - counts
        pages = -(-held // page)
        requests = torch.randperm(n + 7, generator=gen, device="cuda")[:n]
        taken = int(pages.sum())
        total = taken + int((-(-lens // page) - pages).sum()) + 5
        ids = torch.randperm(total, generator=gen, device="cuda").int()
        table = torch.zeros(n + 7, columns, dtype=torch.int32, device="cuda")
        place = torch.arange(columns, device="cuda")[None, :]
        first = torch.cumsum(pages, 0) - pages
        table[requests] = torch.where(place < pages[:, None], ids[(first[:, None] + place).clamp(max=total - 1)], 0)
        all_held = torch.zeros(n + 7, dtype=torch.int32, device="cuda")
        all_held[requests] = held.int()
        free = torch.zeros(total, dtype=torch.int32, device="cuda")
        free[:total - taken] = ids[taken:]

        def empty(*shape):
            return torch.empty(*shape, dtype=torch.int32, device="cuda")
        rows = case["rows"]
        return {"case": case, "requests": requests.int(), "counts": counts.int(), "lens": all_held, "tables": table, "free_pages": free,
                "free_count": torch.tensor([total - taken], dtype=torch.int32, device="cuda"),
                "out": {"query_start": empty(n + 1), "context_lens": empty(n), "positions": empty(rows), "seq_of_row": empty(rows),
                        "slots": empty(rows), "block_tables": empty(n, columns), "free_left": empty(1), "status": empty(1)}}

    kv_heads, head_dim = case["kv_heads"], case["head_dim"]
    padded = _padded(head_dim)
    dtype = CODES[case["dtype"]]
    # channels of different size and a few far outliers, as keys behind a rotation have them
    loud = torch.exp(0.5 * _normal(gen, 2, kv_heads, head_dim))
    loud[0, :, :: 29] *= 4.0

    def planes(pages):
        shape = (pages, kv_heads, page)
        return {"codes": torch.zeros(*shape, padded // 2, dtype=torch.uint8, device="cuda"),
                "words": torch.zeros(*shape, padded // 32, dtype=torch.int16, device="cuda")}

    if case["kind"] == "cache":
        rows = case["rows"]
        x = _normal(gen, rows, 3, kv_heads, head_dim)
        x[:, 1:] *= loud.transpose(0, 1).reshape(kv_heads, 2, head_dim).transpose(0, 1)
        qkv = x.flatten(1).to(dtype)                    # rows of a step's q/k/v product: keys and values are slices of it
        width = kv_heads * head_dim
        pages = -(-rows // page) + 3
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:rows].int()
        return {"case": case, "k": qkv[:, width:2 * width], "v": qkv[:, 2 * width:], "slots": slots, "key": planes(pages), "value": planes(pages),
                "k_out": torch.empty(rows, width, dtype=dtype, device="cuda"), "v_out": torch.empty(rows, width, dtype=dtype, device="cuda")}

    n, heads = case["seqs"], case["heads"]
    lens = _lens(gen, case)
    if case["kind"] == "decode":
        counts = torch.ones(n, dtype=torch.int64, device="cuda")
    else:
        counts = torch.tensor(_queries(case), device="cuda")
    pages = -(-lens // page)
    total, columns = int(pages.sum()), int(pages.max())
    ids = torch.randperm(total, generator=gen, device="cuda").int()
    place = torch.arange(columns, device="cuda")[None, :]
    first = torch.cumsum(pages, 0) - pages
    block_tables = torch.where(place < pages[:, None], ids[(first[:, None] + place).clamp(max=total - 1)], 0).int()
    key, value = planes(total), planes(total)
    at = max(1, (1 << 26) // (kv_heads * page * head_dim))
    for p in range(0, total, at):
        m = min(at, total - p)
        k, v = (_normal(gen, m, kv_heads, page, head_dim) * loud[i][:, None, :] for i in (0, 1))
        for plane, (codes, words) in zip((key, value), _quantise(k, v)):
            plane["codes"][p:p + m], plane["words"][p:p + m] = codes, words
    rows = int(counts.sum())
    # queries that look harder at some keys than at others (scores of a standard deviation of about one and a half)
    q = 1.5 * _normal(gen, rows, heads, head_dim) / loud[0].repeat_interleave(heads // kv_heads, 0).square().mean(-1, keepdim=True).sqrt()
    query_start = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    query_start[1:] = torch.cumsum(counts, 0)
    return {"case": case, "q": q.flatten(1).to(dtype), "key": key, "value": value, "query_start": query_start, "context_lens": lens.int(),
            "block_tables": block_tables, "seq_list": torch.arange(n, dtype=torch.int32, device="cuda"),
            "out": torch.empty(rows, heads * head_dim, dtype=dtype, device="cuda"), "max_queries": int(counts.max())}


# ---- one pass

def run(state):
    case = state["case"]
    if own:
        return _own(state)
    return {"tables": _plain_tables, "cache": _plain_cache, "decode": _plain_attention, "prompt": _plain_attention}[case["kind"]](state)


def _own(state):
    from tiny_inference_engine_b200 import ops
    case = state["case"]
    if case["kind"] == "tables":
        arrays = ops.StepArrays(**state["out"])
        ops.step_tables(state["requests"], state["counts"], state["lens"], state["tables"], state["free_pages"], state["free_count"],
                        case["page"], arrays, commit=False)
        return {**state["out"], "tables": state["tables"]}
    cache = ops.Kv4Cache(state["key"]["codes"], state["key"]["words"], state["value"]["codes"], state["value"]["words"], case["head_dim"])
    if case["kind"] == "cache":
        ops.kv4_append(state["k"], state["v"], state["slots"], cache)
        ops.kv4_read(cache, state["slots"], state["k_out"], state["v_out"])
        return [state["k_out"], state["v_out"]]
    if "workspace" not in state:
        state["workspace"] = ops.kv4_workspace(case["heads"], case["kv_heads"], case["head_dim"], state["q"].device)
    scale = case["head_dim"] ** -0.5
    if case["kind"] == "decode":
        ops.attention_kv4_decode(state["q"], cache, state["out"], state["query_start"], state["context_lens"], state["block_tables"],
                                 case["heads"], scale, state["seq_list"], case["seqs"], case["context"], state["workspace"], window=case["window"])
    else:
        ops.attention_kv4_prompt(state["q"], cache, state["out"], state["query_start"], state["context_lens"], state["block_tables"],
                                 case["seqs"], state["max_queries"], case["heads"], scale, case["context"], state["workspace"],
                                 window=case["window"])
    return state["out"]


def _plain_tables(state):
    case, out = state["case"], state["out"]
    page, columns = case["page"], case["columns"]
    requests, counts = state["requests"].long(), state["counts"]
    n, rows = len(requests), len(out["slots"])
    held = state["lens"][requests]
    lens = held + counts
    query_start = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    query_start[1:] = torch.cumsum(counts, 0)
    old, new = (held + page - 1) // page, (lens + page - 1) // page
    taken = torch.cumsum(new - old, 0)
    # every request's pages, in their order, from the end of the list of free ones
    place = torch.arange(columns, device="cuda")[None, :]
    fresh = (taken - (new - old))[:, None] + place - old[:, None]
    got = state["free_pages"][(state["free_count"] - 1 - fresh).clamp(min=0, max=len(state["free_pages"]) - 1).long()]
    block_tables = torch.where(place < old[:, None], state["tables"][requests], torch.where(place < new[:, None], got, 0)).int()
    tables = state["tables"].clone()
    tables[requests] = torch.where((place >= old[:, None]) & (place < new[:, None]), got, state["tables"][requests])
    row = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(query_start[1:], row, right=True).clamp(max=n - 1)
    live = row < query_start[n]
    position = held[seq] + row - query_start[seq]
    slots = block_tables[seq, (position // page).clamp(min=0, max=columns - 1).long()] * page + position % page
    return {"query_start": query_start, "context_lens": lens.int(), "positions": torch.where(live, position, 0).int(),
            "seq_of_row": torch.where(live, seq, -1).int(), "slots": torch.where(live, slots, -1).int(), "block_tables": block_tables,
            "free_left": (state["free_count"] - taken[-1]).int(), "status": torch.zeros(1, dtype=torch.int32, device="cuda"), "tables": tables}


def _values(codes, words, head_dim):
    """What codes [..., padded / 2] and words [..., padded / 32] stand for: [..., head_dim] in 32 bits."""
    w = words.int()
    s = ((w & 0xffe0) << 16).view(torch.float32)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, 32))
    return (s[..., None] * (c - (w & 15).to(torch.float32)[..., None])).flatten(-2)[..., :head_dim]


def _plain_cache(state):
    case = state["case"]
    kv_heads, head_dim, page = case["kv_heads"], case["head_dim"], case["page"]
    slots = state["slots"].long()
    k, v = (state[name].unflatten(-1, (kv_heads, head_dim)) for name in ("k", "v"))
    out = []
    for plane, (codes, words) in zip((state["key"], state["value"]), _quantise(k, v)):
        plane["codes"][slots // page, :, slots % page] = codes
        plane["words"][slots // page, :, slots % page] = words
        out.append(_values(plane["codes"][slots // page, :, slots % page], plane["words"][slots // page, :, slots % page], head_dim).flatten(1).to(state["k"].dtype))
    return out


def _plain_attention(state):
    case = state["case"]
    heads, kv_heads, head_dim, page, window = (case[x] for x in ("heads", "kv_heads", "head_dim", "page", "window"))
    group, most = heads // kv_heads, state["max_queries"]
    lens, start = state["context_lens"].long(), state["query_start"].long()
    counts = start[1:] - start[:-1]
    n, columns = state["block_tables"].shape
    tables = state["block_tables"].long()

    def whole(plane):        # [sequences, kv heads, keys, head size] in 32 bits
        codes, words = (plane[x][tables].transpose(1, 2).flatten(2, 3) for x in ("codes", "words"))
        return _values(codes, words, head_dim)
    place = torch.arange(most, device="cuda")[None, :]
    row = (start[:-1, None] + place).clamp(max=len(state["q"]) - 1)
    q = state["q"].float()[row].view(n, most, kv_heads, group, head_dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, group * most, head_dim)
    scores = (q @ whole(state["key"]).transpose(-1, -2)) * head_dim ** -0.5
    scores = scores.view(n, kv_heads, group, most, columns * page)
    position = (lens - counts)[:, None] + place
    at = torch.arange(columns * page, device="cuda")
    seen = at <= position[..., None]
    if window:
        seen = seen & (at > position[..., None] - window)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    o = weights.view(n, kv_heads, group * most, columns * page) @ whole(state["value"])
    o = o.view(n, kv_heads, group, most, head_dim).permute(0, 3, 1, 2, 4).reshape(n, most, heads * head_dim)
    return o[place < counts[:, None]].to(state["q"].dtype)


# ---- the bytes and operations that a pass cannot do without, and the definition in 64 bits

def _token_bytes(head_dim):
    return head_dim / 2 + 2 * math.ceil(head_dim / 32)


def _counts(case):
    """(context, queries) of the sequences, contexts as `_lens` spreads them on average."""
    longest = case["context"]
    low = min(max(case["queries"], longest // 8, 1), longest)
    return [(longest if i == 0 or not case["ragged"] else (low + longest) / 2, queries) for i, queries in enumerate(_queries(case))]


def work(case):
    if case["kind"] == "tables":
        n, rows, columns = case["seqs"], case["rows"], case["columns"]
        return {"bytes": 4 * (3 * n + 3 * rows + 2 * n * columns + 2 * n), "flops": 0}
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "cache":     # rows in, codes and words written, values out
        head = 4 * size * case["head_dim"] + 2 * _token_bytes(case["head_dim"])
        return {"bytes": case["rows"] * (case["kv_heads"] * head + 4), "flops": 12 * case["rows"] * case["kv_heads"] * case["head_dim"]}
    total_bytes, flops = 0.0, 0.0
    for context, queries in _counts(case):
        seen = min(context, case["window"] + queries - 1) if case["window"] else context
        total_bytes += seen * case["kv_heads"] * 2 * _token_bytes(case["head_dim"]) + 2 * queries * case["heads"] * case["head_dim"] * size
        # query i of the portion sees context - queries + 1 + i keys, the window's at most
        if case["window"]:
            keys = sum(min(case["window"], context - queries + 1 + i) for i in range(queries))
        else:
            keys = queries * (context - (queries - 1) / 2)
        flops += 4 * case["heads"] * case["head_dim"] * keys
    return {"bytes": total_bytes, "flops": flops}


def exact(case, seed):
    if case["kind"] == "tables":
        return None
    state = prepare(case, seed)
    head_dim, kv_heads = case["head_dim"], case["kv_heads"]
    if case["kind"] == "cache":
        return [_exact_values(state[x].double().view(-1, kv_heads, head_dim)).reshape(case["rows"], -1) for x in ("k", "v")]
    heads = case["heads"]
    group = heads // kv_heads
    lens, start = state["context_lens"].tolist(), state["query_start"].tolist()
    if sum(lens) * case["queries"] * heads > 2 ** 32:
        return None
    answer = torch.empty(start[-1], heads * head_dim, dtype=torch.float64, device="cuda")
    for i, context in enumerate(lens):
        pages = state["block_tables"][i, :-(-context // case["page"])].long()
        first, last = start[i], start[i + 1]
        position = torch.arange(context - (last - first), context, device="cuda")
        key = torch.arange(context, device="cuda")
        hidden = key[None, :] > position[:, None]
        if case["window"]:
            hidden |= key[None, :] <= position[:, None] - case["window"]
        for h in range(kv_heads):
            k, v = (_exact_dequantise(state[x]["codes"][pages, h], state[x]["words"][pages, h]).flatten(0, 1)[:context, :head_dim] for x in ("key", "value"))
            for j in range(h * group, (h + 1) * group):
                q = state["q"][first:last, j * head_dim:(j + 1) * head_dim].double()
                score = torch.where(hidden, -math.inf, q @ k.T / math.sqrt(head_dim))
                answer[first:last, j * head_dim:(j + 1) * head_dim] = torch.softmax(score, -1) @ v
    return answer


def _exact_dequantise(codes, words):
    """codes [..., padded / 2], words [..., padded / 32] to 64-bit values: sign, exponent and two bits of mantissa taken apart."""
    w = words.long() & 0xffff
    step = torch.ldexp(1 + ((w >> 5) & 3).double() / 4, ((w >> 7) & 0xff) - 127)
    zero = (w & 15).double()
    both = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    both[..., 0::2], both[..., 1::2] = (codes % 16).double(), (codes // 16).double()
    each = torch.arange(both.shape[-1], device=codes.device) // 32
    return (both - zero[..., each]) * step[..., each]


def _exact_values(x):
    """x [rows, heads, head_dim] in 64 bits, all finite: the values that the cache holds for it."""
    answer = torch.empty_like(x)
    for d in range(0, x.shape[-1], 32):
        g = x[..., d:d + 32]
        low, high = (-g).amax(-1).clamp(min=0), g.amax(-1).clamp(min=0)         # how far the group goes below and above zero
        least = ((low + high).float().double() / 15).float().double().clamp(min=2.0 ** -100)     # (a sum and a quotient of 32 bits)
        e = torch.floor(torch.log2(least))
        e = e - (torch.exp2(e) > least).double() + (torch.exp2(e + 1) <= least).double()
        step = torch.ceil(least / torch.exp2(e - 2)) * torch.exp2(e - 2)
        zero = torch.round(low / step)
        code = torch.round(g / step[..., None]) + zero[..., None]
        answer[..., d:d + 32] = (code.clamp(0, 15) - zero[..., None]) * step[..., None]
    return answer
