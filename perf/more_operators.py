"""Operators of a paged key/value cache and of the attention that reads it, as measured cases.

Four operators over a cache of fp16 pages that the sequences of a packed batch
reach through tables of page numbers; activations fp32 or fp16 (the library's
two types):

``attention``  attention of a batch's new tokens (one per conversation, a few
               drafted ones, chunks of prompts) over the cache, causal, with
               grouped heads and, as the model has them, capped scores, a
               window, a bias that falls with distance;
``write``      keys and values of the new tokens into their places;
``assign``     slots take over the states of their parents (forks, beams in a
               new order, freed slots) and get pages for their next tokens;
``compact``    pages move to the front of the pool, the tables follow.

Sizes are those of the decoder that the library serves (16 query and 4 key
heads of 256, 8 attention layers, pages of 128 tokens, contexts up to 65536,
batches of 8, at most 5 drafted tokens, ragged prompts of 821 rows) and generic
ones.
"""
import math

import torch

own = False

TEXT = 65536  # the longest context


def listed():
    return [
        # One conversation's next token: what counts is latency.
        {"name": "attn_m1_f16", "kind": "attention", "queries": 1, "rows": 1, "heads": 16, "kv_heads": 4, "dim": 256, "page": 128,
         "context": 777, "softcap": 0.0, "window": 0, "slopes": False, "dtype": "f16"},
        # Eight conversations of different lengths, one token each.
        {"name": "attn_m8_f16", "kind": "attention", "queries": 8, "rows": 8, "heads": 16, "kv_heads": 4, "dim": 256, "page": 128,
         "context": TEXT, "softcap": 0.0, "window": 0, "slopes": False, "dtype": "f16"},
        # Five drafted tokens of each of eight conversations to verify, capped scores, small pages.
        {"name": "attn_m40_cap_f32", "kind": "attention", "queries": 8, "rows": 40, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "context": 16384, "softcap": 50.0, "window": 0, "slopes": False, "dtype": "f32"},
        # Ragged prompts behind ragged contexts, a window and a bias that falls with distance.
        {"name": "attn_m821_slopes_f32", "kind": "attention", "queries": 8, "rows": 821, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "context": 4096, "softcap": 0.0, "window": 1024, "slopes": True, "dtype": "f32"},
        # Chunks of eight long prompts.
        {"name": "attn_m2048_f16", "kind": "attention", "queries": 8, "rows": 2048, "heads": 16, "kv_heads": 4, "dim": 256, "page": 128,
         "context": 8192, "softcap": 0.0, "window": 0, "slopes": False, "dtype": "f16"},
        # One long prompt from its first token on.
        {"name": "attn_m8192_f16", "kind": "attention", "queries": 1, "rows": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "page": 128,
         "context": 8192, "softcap": 0.0, "window": 0, "slopes": False, "dtype": "f16"},
        # One token of each of eight conversations.
        {"name": "write_m8_f16", "kind": "write", "queries": 8, "rows": 8, "kv_heads": 4, "dim": 256, "page": 128, "context": 4096, "dtype": "f16"},
        # Chunks of eight prompts, keys and values in the rows of the joined projection.
        {"name": "write_m8192_f32", "kind": "write", "queries": 8, "rows": 8192, "kv_heads": 8, "dim": 128, "page": 64, "context": 4096,
         "dtype": "f32"},
        # Two questions, four beams each, after a step: some beams go on twice, some end.
        {"name": "assign_8", "kind": "assign", "groups": 2, "beams": 4, "tokens": 500, "layers": 1, "kv_heads": 4, "dim": 256, "page": 128},
        # Eight questions, eight beams each, all attention layers.
        {"name": "assign_64", "kind": "assign", "groups": 8, "beams": 8, "tokens": 200, "layers": 8, "kv_heads": 4, "dim": 256, "page": 32},
        # A small pool after some conversations have ended.
        {"name": "compact_8", "kind": "compact", "slots": 8, "tokens": 300, "layers": 1, "kv_heads": 4, "dim": 256, "page": 64},
        # All attention layers, half the pool free.
        {"name": "compact_64", "kind": "compact", "slots": 64, "tokens": 500, "layers": 8, "kv_heads": 4, "dim": 256, "page": 16},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "write", "assign", "compact"])
    dtype = rng.choice(["f32", "f16"])
    kv, dim, page = rng.randint(1, 8), rng.choice([64, 80, 96, 128, 128, 192, 256]), rng.choice([16, 32, 64, 128])
    if kind in ("attention", "write"):
        case = {"kind": kind, "queries": rng.randint(1, 8), "kv_heads": kv, "dim": dim, "page": page, "dtype": dtype}
        if kind == "write":
            case["rows"] = _log(rng, case["queries"], 8192)
            case["context"] = max(_log(rng, 1, 8192), max(_counts(case["rows"], case["queries"])))
            return case
        case["heads"] = heads = kv * rng.randint(1, 8)
        case["softcap"], case["window"] = rng.choice([0.0, 0.0, 30.0, 50.0]), rng.choice([0, 0, 1, 100, 1024, 4096])
        case["slopes"] = rng.random() < 0.3
        if rng.random() < 0.5:
            case["rows"] = case["queries"] * rng.randint(1, 5)
            case["context"] = max(5, _log(rng, 1, TEXT))
        else:
            case["rows"] = _log(rng, 6 * case["queries"], 4096)
            most = 8192 * 8192 * 32 * 128 // 4 // (case["rows"] * heads * dim)
            case["context"] = max(max(_counts(case["rows"], case["queries"])), min(_log(rng, 16, TEXT), most))
        return case
    layers = rng.choice([1, 2, 8])
    case = {"kind": kind, "layers": layers, "kv_heads": min(kv, 4), "dim": dim, "page": page}
    most = 250 * 32 // page  # pages of a pool of the largest listed case
    if kind == "assign":
        case["groups"], case["beams"] = rng.randint(1, 8), rng.randint(1, 8)
        case["tokens"] = _log(rng, 1, max(2, page * min(most // (2 * case["groups"]) - 1, 20)))
    else:
        case["slots"] = rng.randint(1, 64)
        case["tokens"] = _log(rng, 1, max(2, page * min(most // case["slots"], 40)))
    return case


# ---- inputs -----------------------------------------------------------------

def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.float16


def _size(case):
    return 4 if case["dtype"] == "f32" else 2


def _gen(seed, part):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * int(seed) + part)
    return g


def _randn(seed, part, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=_gen(seed, part), device="cuda", dtype=dtype)


def _counts(rows, queries):
    """Rows of each sequence: alike for a decode batch, ragged for prompts."""
    if rows <= 5 * queries:
        return [rows // queries + (1 if i < rows % queries else 0) for i in range(queries)]
    total = queries * (queries + 1) // 2
    counts = [max(1, rows * (i + 1) // total) for i in range(queries)]
    counts[-1] += rows - sum(counts)
    return counts


def _contexts(case):
    """Tokens of each sequence after the pass: a quarter to all of the context."""
    n = case["queries"]
    return [max(c, case["context"] * (1 + 3 * (i + 1) // n) // 4) for i, c in enumerate(_counts(case["rows"], n))]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _ints(seed, part, n, hi):
    """n whole numbers below hi (a list)."""
    g = torch.Generator()
    g.manual_seed(1_000_003 * int(seed) + part)
    return torch.randint(0, hi, (n,), generator=g).tolist()


def _paged(case, seed):
    """A layer's cache and the sequences' tables: pages in no order, a few more than the sequences need."""
    page, contexts = case["page"], _contexts(case)
    need = [-(-c // page) for c in contexts]
    pages, width = sum(need) + 3, max(need) + 1
    order = torch.randperm(pages, generator=_gen(seed, 20), device="cuda").to(torch.int32)
    tables = torch.full((case["queries"], width), -1, device="cuda", dtype=torch.int32)
    at = 0
    for q, n in enumerate(need):
        tables[q, :n] = order[at:at + n]
        at += n
    cache = _randn(seed, 21, pages, 2, case["kv_heads"], page, case["dim"], dtype=torch.float16)
    counts = _counts(case["rows"], case["queries"])
    return {"k_cache": cache[:, 0], "v_cache": cache[:, 1], "tables": tables, "counts": counts,
            "positions": _i32([t - c for t, c in zip(contexts, counts)]), "longest": max(contexts)}


def _groups(case, seed):
    """Tables of beams: the full pages of a question's prompt are shared, each beam has pages of its own behind them.  As the pool
    knows them: (tables, lengths, parents, tokens to come, pages)."""
    page, beams, slots = case["page"], case["beams"], case["groups"] * case["beams"]
    lengths, rows, used = [], [], 0
    for n in _ints(seed, 30, case["groups"], case["tokens"]):
        tokens = case["tokens"] // 2 + n // 2 + 1
        shared = tokens * 2 // 3 // page
        front, used = list(range(used, used + shared)), used + shared
        for _ in range(beams):
            more = -(-tokens // page) - shared
            rows.append(front + list(range(used, used + more)))
            lengths.append(tokens)
            used += more
    most = -(-case["tokens"] // page)  # pages of the longest
    width, pages = most + 2, case["groups"] * (most + beams * (most // 3 + 2)) + slots
    g = torch.Generator()
    g.manual_seed(1_000_003 * int(seed) + 31)
    order = torch.randperm(pages, generator=g).tolist()
    tables = [[order[p] for p in r] + [-1] * (width - len(r)) for r in rows]
    parents = [s // beams * beams + p for s, p in enumerate(_ints(seed, 32, slots, beams))]
    parents = [-1 if r == 0 else p for p, r in zip(parents, _ints(seed, 33, slots, 9))]
    return tables, lengths, parents, [1] * slots, pages


def _ended(case, seed):
    """Tables of conversations of which some have ended: (tables, lengths, pages)."""
    page, slots = case["page"], case["slots"]
    lengths = [t + 1 for t in _ints(seed, 40, slots, case["tokens"])]
    alive = [r < 2 for r in _ints(seed, 41, slots, 3)]
    need = [-(-t // page) for t in lengths]
    width = -(-case["tokens"] // page)
    pages = slots * width + 2
    g = torch.Generator()
    g.manual_seed(1_000_003 * int(seed) + 42)
    order, tables, at = torch.randperm(pages, generator=g).tolist(), [], 0
    for n, a in zip(need, alive):
        tables.append((order[at:at + n] if a else []) + [-1] * (width - (n if a else 0)))
        at += n
    return tables, [t if a else 0 for t, a in zip(lengths, alive)], pages


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case}
    if kind in ("attention", "write"):
        s.update(_paged(case, seed))
        rows, kv, dim, dt = case["rows"], case["kv_heads"], case["dim"], _dtype(case)
        if kind == "attention":
            heads = case["heads"]
            s["q"] = (1.5 * _randn(seed, 1, rows, heads, dim)).to(dt)
            s["slopes"] = None
            if case["slopes"]:
                s["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda", dtype=torch.float32) / heads)
            s["out"] = torch.empty_like(s["q"])
        else:
            joined = _randn(seed, 1, rows, 4 * kv * dim).to(dt)  # queries (twice the key heads), keys, values
            s["k"] = joined[:, 2 * kv * dim:3 * kv * dim].view(rows, kv, dim)
            s["v"] = joined[:, 3 * kv * dim:].view(rows, kv, dim)
        return s
    shape = (case["layers"], 2, case["kv_heads"], case["page"], case["dim"])
    if kind == "assign":
        tables, lengths, parents, counts, pages = _groups(case, seed)
        s["parents"], s["counts"] = _i32(parents), _i32(counts)
        s["new_lengths"], s["missing"] = torch.empty(len(lengths), device="cuda", dtype=torch.int32), _i32([0])
    else:
        tables, lengths, pages = _ended(case, seed)
        s["used"] = _i32([0])
    s["tables"], s["lengths"] = _i32(tables), _i32(lengths)
    s["new_tables"] = torch.empty_like(s["tables"])
    s["pool"] = _randn(seed, 2, pages, *shape, dtype=torch.float16)
    return s


# ---- one pass -----------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["kind"] == "attention":
        return _attention(s, c)
    if c["kind"] == "write":
        return _write(s, c)
    return _assign(s, c) if c["kind"] == "assign" else _compact(s, c)


def _run_own(s, c):
    import mtlqwen_amd as q4k
    if c["kind"] == "attention":
        return q4k.attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["positions"], s["out"], query_counts=s["counts"],
                             softcap=c["softcap"], window=c["window"], slopes=s["slopes"])
    if c["kind"] == "write":
        return q4k.cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["positions"], query_counts=s["counts"])
    if c["kind"] == "assign":
        q4k.cache_assign(s["pool"], s["tables"], s["lengths"], s["parents"], s["new_tables"], s["new_lengths"], counts=s["counts"],
                         missing=s["missing"])
        return s["new_tables"], s["new_lengths"], s["missing"], s["pool"]
    q4k.cache_compact(s["pool"], s["tables"], s["lengths"], s["new_tables"], used=s["used"])
    return s["new_tables"], s["used"], s["pool"]


def _rows_of(s, rows):
    """The sequence and the number within it of every row of the packed batch."""
    counts = torch.tensor(s["counts"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(s["counts"]), device="cuda"), counts, output_size=rows)
    return seq, torch.arange(rows, device="cuda") - (torch.cumsum(counts, 0) - counts)[seq]


def _attention(s, c):
    rows, heads, kv, dim, page = c["rows"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    n, most, longest, group = c["queries"], max(s["counts"]), s["longest"], heads // kv
    seq, nth = _rows_of(s, rows)
    # Every sequence's queries, keys and values side by side, as long as the longest's.
    q = torch.zeros((n, most, heads, dim), device="cuda")
    q[seq, nth] = s["q"].float()
    q = q.view(n, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n * kv, group * most, dim)
    pages = s["tables"][:, :-(-longest // page)].clamp(min=0).long()
    k = s["k_cache"][pages].permute(0, 2, 1, 3, 4).reshape(n * kv, -1, dim)[:, :longest].float()
    v = s["v_cache"][pages].permute(0, 2, 1, 3, 4).reshape(n * kv, -1, dim)[:, :longest].float()
    scores = (q @ k.transpose(1, 2).contiguous()).view(n, heads, most, longest) / math.sqrt(dim)
    if c["softcap"]:
        scores = c["softcap"] * torch.tanh(scores / c["softcap"])
    far = torch.arange(longest, device="cuda") - (s["positions"].long().unsqueeze(1) + torch.arange(most, device="cuda")).unsqueeze(2)
    if s["slopes"] is not None:
        scores = scores + s["slopes"].view(1, heads, 1, 1) * far.unsqueeze(1).float()
    hidden = far > 0
    if c["window"]:
        hidden = hidden | (far <= -c["window"])
    scores = scores.masked_fill(hidden.unsqueeze(1), float("-inf"))
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    o = (p.view(n * kv, group * most, longest) @ v).view(n, heads, most, dim)
    return o.transpose(1, 2)[seq, nth].to(s["q"].dtype)


def _write(s, c):
    seq, nth = _rows_of(s, c["rows"])
    at = s["positions"].long()[seq] + nth
    page = s["tables"].long()[seq, at // c["page"]]
    s["k_cache"][page, :, at % c["page"]] = s["k"].to(torch.float16)
    s["v_cache"][page, :, at % c["page"]] = s["v"].to(torch.float16)
    return s["k_cache"], s["v_cache"]


def _assign(s, c):
    page, pages, (slots, width) = c["page"], s["pool"].shape[0], s["tables"].shape
    slot, entry = torch.arange(slots, device="cuda"), torch.arange(width, device="cuda")
    live, parent = s["parents"] >= 0, s["parents"].clamp(min=0).long()
    length = torch.where(live, s["lengths"][parent], 0)
    table = torch.where(live.unsqueeze(1), s["tables"][parent], -1).long()
    full, part = length.long() // page, length.long() % page
    # Full pages are shared.  A page that is written on goes to the lowest slot that holds it, the others copy it.
    held = entry < full.unsqueeze(1)
    used = torch.zeros(pages + 1, device="cuda", dtype=torch.bool)
    used[torch.where(held & (table >= 0), table, pages)] = True
    last = torch.where(part > 0, table.gather(1, full.clamp(max=width - 1).unsqueeze(1)).squeeze(1), -1)
    before = (last.unsqueeze(1) == last) & (slot < slot.unsqueeze(1))
    keep = (last >= 0) & ~before.any(dim=1) & ~used[last.clamp(min=0)]
    copy = (last >= 0) & ~keep
    used[torch.where(keep, last, pages)] = True
    # The rest gets free pages, the lowest first, in the order of the slots.
    need = (length.long() + s["counts"] + page - 1) // page
    wants = (entry >= (full + keep).unsqueeze(1)) & (entry < need.unsqueeze(1))
    rank = torch.cumsum(wants.flatten().long(), 0).view(slots, width) - 1
    free = torch.argsort(used[:pages].to(torch.uint8), stable=True)
    there = (~used[:pages]).sum()
    given = torch.where(wants & (rank < there), free[rank.clamp(0, pages - 1)], -1)
    mine = keep.unsqueeze(1) & (entry == full.unsqueeze(1))
    new = torch.where(held | mine, table, given)
    source = last[copy]
    target = new.gather(1, full.clamp(max=width - 1).unsqueeze(1)).squeeze(1)[copy]
    valid = (torch.arange(page, device="cuda") < part[copy].unsqueeze(1)).view(-1, 1, 1, 1, page, 1)
    s["pool"][target] = torch.where(valid, s["pool"][source], s["pool"][target])
    s["new_tables"].copy_(new)
    s["new_lengths"].copy_(length)
    s["missing"].copy_((rank.flatten()[-1:] + 1 - there).clamp(min=0))
    return s["new_tables"], s["new_lengths"], s["missing"], s["pool"]


def _compact(s, c):
    page, pages, (slots, width) = c["page"], s["pool"].shape[0], s["tables"].shape
    table = s["tables"].long()
    held = (torch.arange(width, device="cuda") < ((s["lengths"].long() + page - 1) // page).unsqueeze(1)) & (table >= 0)
    used = torch.zeros(pages + 1, device="cuda", dtype=torch.bool)
    used[torch.where(held, table, pages)] = True
    used = used[:pages]
    n, number = used.sum(), torch.arange(pages, device="cuda")
    hole, high = ~used & (number < n), used & (number >= n)
    source, target = number[high], number[hole]
    to = number.clone()
    to[source] = target
    s["pool"][target] = s["pool"][source]
    s["new_tables"].copy_(torch.where(held, to[table.clamp(min=0)], -1))
    s["used"].copy_(n)
    return s["new_tables"], s["used"], s["pool"]


# ---- what a pass cannot do without ------------------------------------------------

def _seen(case):
    """(keys that the queries see, summed over the rows, and keys of each sequence that any of its rows sees, summed)."""
    pairs = keys = 0
    window = case["window"] or 1 << 30
    for t, n in zip(_contexts(case), _counts(case["rows"], case["queries"])):
        first = t - n  # the keys before the first row
        whole = min(n, max(0, window - first))  # rows whose window reaches the first key
        pairs += whole * first + whole * (whole + 1) // 2 + (n - whole) * window
        keys += min(t, n + window - 1)
    return pairs, keys


def work(case):
    """Each input read once, each output written once."""
    kind = case["kind"]
    if kind == "attention":
        pairs, keys = _seen(case)
        rows, heads, dim = case["rows"], case["heads"], case["dim"]
        return {"bytes": 2 * keys * case["kv_heads"] * dim * 2 + 2 * rows * heads * dim * _size(case) + 4 * (keys // case["page"] + case["queries"]),
                "flops": 4 * pairs * heads * dim}
    if kind == "write":
        values = 2 * case["rows"] * case["kv_heads"] * case["dim"]
        return {"bytes": values * (_size(case) + 2) + 8 * case["rows"] // case["page"] + 4 * case["queries"], "flops": values}
    token = case["layers"] * 2 * case["kv_heads"] * case["dim"] * 2
    if kind == "assign":  # on average over the seeds: how many beams share a parent, and how full their last pages are
        slots, beams = case["groups"] * case["beams"], case["beams"]
        alone = case["groups"] * beams * (1 - (1 - 8 / (9 * beams)) ** beams)
        copies = max(0.0, slots * 8 / 9 - alone)
        tables = 8 * slots * (case["tokens"] // case["page"] + 2)
        return {"bytes": int(copies * min(case["tokens"], case["page"]) / 2 * 2 * token + tables), "flops": int(tables)}
    pool = case["slots"] * -(-case["tokens"] // case["page"]) + 2
    held = case["slots"] * 2 / 3 * (case["tokens"] / 2 / case["page"] + 0.5)  # on average over the seeds
    return {"bytes": int(held * max(0.0, 1 - held / pool) * 2 * case["page"] * token + 8 * held), "flops": int(8 * held)}


# ---- the same in 64 bits -----------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind, page = case["kind"], case["page"]
    if kind == "attention":
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        out = torch.empty(case["rows"], heads, dim, device="cuda", dtype=torch.float64)
        start = 0
        for i, n in enumerate(s["counts"]):
            first = int(s["positions"][i])
            length = first + n
            mine = s["tables"][i, :-(-length // page)].long()
            at = first + torch.arange(n, device="cuda").unsqueeze(1)
            key = torch.arange(length, device="cuda")
            seen = (key <= at) & (key > at - (case["window"] or 1 << 40))
            for j in range(kv):
                k = s["k_cache"][mine, j].flatten(0, 1)[:length].double()
                v = s["v_cache"][mine, j].flatten(0, 1)[:length].double()
                for h in range(j * heads // kv, (j + 1) * heads // kv):
                    x = (s["q"][start:start + n, h].double() @ k.t().contiguous()) * dim ** -0.5
                    if case["softcap"]:
                        x = (x / case["softcap"]).tanh() * case["softcap"]
                    if s["slopes"] is not None:
                        x = x - s["slopes"][h].double() * (at - key)
                    x[~seen] = -math.inf
                    out[start:start + n, h] = torch.softmax(x, dim=1) @ v
            start += n
        return out
    if kind == "write":
        k, v, start = s["k_cache"].clone(), s["v_cache"].clone(), 0
        for i, n in enumerate(s["counts"]):
            at = torch.arange(int(s["positions"][i]), int(s["positions"][i]) + n, device="cuda")
            where = s["tables"][i].long()[torch.div(at, page, rounding_mode="floor")]
            k[where, :, at % page] = s["k"][start:start + n].half()
            v[where, :, at % page] = s["v"][start:start + n].half()
            start += n
        return k, v
    pool, tables, lengths = s["pool"].clone(), s["tables"].tolist(), s["lengths"].tolist()
    if kind == "compact":
        held = [t[:-(-n // page)] + [-1] * (len(t) + (-n // page)) for t, n in zip(tables, lengths)]
        used = sorted({p for t in held for p in t if p >= 0})
        n = len(used)
        holes = sorted(set(range(n)) - set(used))
        to = dict(zip([p for p in used if p >= n], holes))
        for a, b in to.items():
            pool[b] = s["pool"][a]
        return _i32([[to.get(p, p) for p in t] for t in held]), _i32([n]), pool
    parents, counts = s["parents"].tolist(), s["counts"].tolist()
    length = [lengths[p] if p >= 0 else 0 for p in parents]
    new = [tables[p][:n // page] if p >= 0 else [] for p, n in zip(parents, length)]
    taken, jobs = {p for t in new for p in t}, []
    for i, (p, n) in enumerate(zip(parents, length)):
        if n % page:
            tail = tables[p][n // page]
            if tail in taken:
                jobs.append((i, tail, n % page))
            else:
                taken.add(tail)
                new[i].append(tail)
    free = [p for p in range(pool.shape[0]) if p not in taken]
    lacking = 0
    for i, n in enumerate(length):
        for e in range(len(new[i]), -(-(n + counts[i]) // page)):
            lacking += not free
            new[i].append(free.pop(0) if free else -1)
    for i, tail, n in jobs:
        if new[i][length[i] // page] >= 0:
            pool[new[i][length[i] // page], :, :, :, :n] = s["pool"][tail, :, :, :, :n]
    return _i32([t + [-1] * (len(tables[0]) - len(t)) for t in new]), _i32(length), _i32([lacking]), pool
