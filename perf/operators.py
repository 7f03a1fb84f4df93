"""Operators of a decoder pass around the library's projections, as measured cases.

Four operators over a packed batch of up to 8 sequences, fp32 or fp16
activations (the library's two types):

``rope``      rotary positions of ``heads`` heads a row;
``qk_norm``   RMS norm of every query and key head and their rotation, read
              in place in the output row of the joined projection;
``lora``      low-rank adapters, one per sequence, added beside a projection;
``logits``    penalties, biases and grammar masks on vocabulary rows.

Sizes are those of the decoder that the library serves (hidden size 4096,
projections of 1024 to 12288 outputs, a vocabulary of 248,320, batches of 8,
ragged prompts of 821 rows, prefills of 2048) and, for heads, ranks,
vocabularies and histories, generic ones.
"""
import math

import torch

own = False

HIDDEN, FFN, VOCAB = 4096, 12288, 248320
EPS = 1e-6
PROJECTIONS = [(4096, 1024), (4096, 4096), (4096, 6144), (4096, 8192), (4096, 12288), (12288, 4096)]  # (k, n)


def listed():
    return [
        # One token of each of eight conversations: the query heads of one layer.
        {"name": "rope_m8_f16", "kind": "rope", "rows": 8, "heads": 32, "dim": 128, "rot": 128, "interleaved": False, "factor": 1.0,
         "context": 65536, "dtype": "f16"},
        # Ragged prompts in a stretched context, a quarter of the head rotated, adjacent pairs.
        {"name": "rope_m821_part_f32", "kind": "rope", "rows": 821, "heads": 16, "dim": 256, "rot": 64, "interleaved": True, "factor": 8.0,
         "context": 524288, "dtype": "f32"},
        # The longest prefill: every head of eight long prompts.
        {"name": "rope_m8192_f32", "kind": "rope", "rows": 8192, "heads": 40, "dim": 128, "rot": 128, "interleaved": False, "factor": 4.0,
         "context": 131072, "dtype": "f32"},
        # One token of each of eight conversations: 32 query and 8 key heads in a joined row of 6144.
        {"name": "qk_norm_m8_f32", "kind": "qk_norm", "rows": 8, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "gated": False,
         "interleaved": False, "context": 65536, "dtype": "f32"},
        # Ragged prompts: queries with their output gates between them (8192 outputs), 4 key heads, a quarter rotated.
        {"name": "qk_norm_m821_gated_f16", "kind": "qk_norm", "rows": 821, "heads": 16, "kv_heads": 4, "dim": 256, "rot": 64, "gated": True,
         "interleaved": False, "context": 65536, "dtype": "f16"},
        # The longest prefill.
        {"name": "qk_norm_m8192_f16", "kind": "qk_norm", "rows": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "gated": False,
         "interleaved": False, "context": 65536, "dtype": "f16"},
        # Eight conversations, one token and one adapter each, beside an MLP projection.
        {"name": "lora_m8_r16_f16", "kind": "lora", "m": 8, "queries": 8, "k": 4096, "n": 12288, "rank": 16, "mixed": False, "aux": True,
         "dtype": "f16"},
        # Ragged prompts and single tokens, adapters of several ranks, sequences without one, beside the joined projection.
        {"name": "lora_m333_mixed_f16", "kind": "lora", "m": 333, "queries": 8, "k": 4096, "n": 6144, "rank": 64, "mixed": True, "aux": False,
         "dtype": "f16"},
        # The longest prefill: eight prompts with adapters of rank 64 beside an MLP projection.
        {"name": "lora_m2048_r64_f32", "kind": "lora", "m": 2048, "queries": 8, "k": 4096, "n": 12288, "rank": 64, "mixed": False, "aux": True,
         "dtype": "f32"},
        # One conversation's next token: penalties for what it has said.
        {"name": "logits_m1_f32", "kind": "logits", "rows": 1, "vocab": 248320, "history": 900, "bias": 0, "mask": False, "dtype": "f32"},
        # Five drafted tokens to verify under a grammar, biases, a vocabulary of odd size.
        {"name": "logits_m5_odd_f16", "kind": "logits", "rows": 5, "vocab": 50257, "history": 4001, "bias": 100, "mask": True, "dtype": "f16"},
        # As many rows as a pass samples, histories of the longest context.
        {"name": "logits_m64_f32", "kind": "logits", "rows": 64, "vocab": 248320, "history": 65536, "bias": 300, "mask": True, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "qk_norm", "lora", "logits"])
    dtype = rng.choice(["f32", "f16"])
    if kind in ("rope", "qk_norm"):
        dim = rng.choice([64, 80, 96, 112, 128, 128, 192, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        rot -= rot % 2
        case = {"kind": kind, "heads": _log(rng, 1, 64), "dim": dim, "rot": rot, "interleaved": rng.random() < 0.4, "dtype": dtype,
                "context": _log(rng, 512, 1 << 20)}
        if kind == "rope":
            case["factor"] = rng.choice([1.0, 1.0, 2.0, 8.0, 32.0])
        else:
            case["kv_heads"] = rng.randint(1, min(8, case["heads"]))
            case["gated"] = rng.random() < 0.3
        total = case["heads"] + case.get("kv_heads", 0)
        case["rows"] = min(_log(rng, 1, 8192), 8192 * 40 * 128 // (total * dim))
        return case
    if kind == "lora":
        m = _log(rng, 1, 2048)
        k, n = rng.choice(PROJECTIONS)
        return {"kind": kind, "m": m, "queries": rng.randint(1, min(8, m)), "k": k, "n": n, "rank": _log(rng, 4, 64), "mixed": rng.random() < 0.5,
                "aux": rng.random() < 0.5, "dtype": dtype}
    return {"kind": kind, "rows": _log(rng, 1, 64), "vocab": _log(rng, 1000, VOCAB), "history": _log(rng, 1, 65536),
            "bias": rng.choice([0, 0, 1, 17, 100, 300]), "mask": rng.random() < 0.5, "dtype": dtype}


# ---- inputs -----------------------------------------------------------------

def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.float16


def _size(case):
    return 4 if case["dtype"] == "f32" else 2


def _gen(seed, part):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * int(seed) + part)
    return g


def _randn(seed, part, *shape):
    return torch.randn(shape, generator=_gen(seed, part), device="cuda")


def _ints(seed, part, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=_gen(seed, part), device="cuda", dtype=torch.int32)


def _counts(m, queries):
    """Rows of each sequence: alike for a decode batch, ragged for prompts."""
    if m <= 5 * queries:
        return [m // queries + (1 if i < m % queries else 0) for i in range(queries)]
    total = queries * (queries + 1) // 2
    counts = [max(1, m * (i + 1) // total) for i in range(queries)]
    counts[-1] += m - sum(counts)
    return counts


def _frequencies(rot, factor, context):
    """Angle per position of each pair in 64 bits: base 10000, and the ramp
    between interpolated and kept frequencies for a context ``factor`` times
    the original one; the scale of the rotated values that goes with it."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if factor == 1.0:
        return inv.cuda(), 1.0
    turns = (context / factor) * inv / (2 * math.pi)
    kept = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return ((1.0 - kept) * inv / factor + kept * inv).cuda(), 0.1 * math.log(factor) + 1.0


def _positions(seed, rows, context):
    """Up to 8 rows: the next position of as many conversations; more: one
    run of positions that starts anywhere in the context."""
    if rows <= 8:
        return _ints(seed, 2, 0, context, rows)
    return _ints(seed, 2, 0, max(1, context - rows), 1) + torch.arange(rows, device="cuda", dtype=torch.int32)


def _adapter_ranks(case):
    """Ranks of the eight adapters: all the largest, or a quarter to all of it."""
    r = case["rank"]
    return [max(1, r * (i % 4 + 1) // 4) if case["mixed"] else r for i in range(8)]


def _adapter_ids(case):
    """The adapter of each sequence; with mixed ranks every third has none."""
    return [-1 if case["mixed"] and i % 3 == 2 else (5 * i + 3) % 8 for i in range(case["queries"])]


def prepare(case, seed):
    kind, dt = case["kind"], _dtype(case)
    s = {"case": case}
    if kind in ("rope", "qk_norm"):
        rows, heads, dim = case["rows"], case["heads"], case["dim"]
        s["inv_freq"], s["scale"] = _frequencies(case["rot"], case.get("factor", 1.0), case["context"])
        s["positions"] = _positions(seed, rows, case["context"])
        if kind == "rope":
            s["x"] = _randn(seed, 1, rows, heads, dim).to(dt)
            s["y"] = torch.empty_like(s["x"])
        else:
            kv, step = case["kv_heads"], 2 if case["gated"] else 1
            joined = _randn(seed, 1, rows, (heads * step + 2 * kv) * dim).to(dt)  # queries (and gates), keys, values
            s["q"] = joined[:, :heads * step * dim].view(rows, heads, step * dim)[:, :, :dim]
            s["k"] = joined[:, heads * step * dim:(heads * step + kv) * dim].view(rows, kv, dim)
            s["q_weight"] = 0.5 + torch.rand((dim,), generator=_gen(seed, 3), device="cuda")
            s["k_weight"] = 0.5 + torch.rand((dim,), generator=_gen(seed, 4), device="cuda")
            s["q_out"] = torch.empty((rows, heads, dim), device="cuda", dtype=dt)
            s["k_out"] = torch.empty((rows, kv, dim), device="cuda", dtype=dt)
    elif kind == "lora":
        m, k, n, r = case["m"], case["k"], case["n"], case["rank"]
        s["x"] = _randn(seed, 1, m, k).to(dt)
        s["a"] = (_randn(seed, 2, 8, r, k) / math.sqrt(k)).to(torch.float16)
        s["b"] = (0.3 * _randn(seed, 3, 8, n, r) / math.sqrt(r)).to(torch.float16)
        s["ranks"] = torch.tensor(_adapter_ranks(case), device="cuda", dtype=torch.int32)
        s["scales"] = 0.5 + 1.5 * torch.rand((8,), generator=_gen(seed, 4), device="cuda")
        s["counts"] = _counts(m, case["queries"])
        s["ids"] = torch.tensor(_adapter_ids(case), device="cuda", dtype=torch.int32)
        s["aux"] = _randn(seed, 5, m, n).to(dt) if case["aux"] else None
        s["y"] = torch.empty((m, n), device="cuda", dtype=dt)
    else:
        rows, vocab, history = case["rows"], case["vocab"], case["history"]
        s["logits"] = (4.0 * _randn(seed, 1, rows, vocab)).to(dt)
        # Texts repeat: token ids fall off towards the rare ones.
        u = torch.rand((rows, history), generator=_gen(seed, 2), device="cuda")
        s["tokens"] = (vocab * u ** 4).to(torch.int32).clamp_(max=vocab - 1)
        s["slots"] = torch.randperm(rows, generator=_gen(seed, 3), device="cuda").to(torch.int32)
        s["lengths"] = _ints(seed, 4, history // 2, history + 1, rows)
        s["prompts"] = s["lengths"] // 2
        s["repetition"] = 1.0 + 0.3 * torch.rand((rows,), generator=_gen(seed, 5), device="cuda")
        s["frequency"] = 0.5 * torch.rand((rows,), generator=_gen(seed, 6), device="cuda")
        s["presence"] = torch.rand((rows,), generator=_gen(seed, 7), device="cuda")
        if case["bias"]:
            b = case["bias"]
            s["bias_offsets"] = torch.arange(0, (rows + 1) * b, b, device="cuda", dtype=torch.int32)
            s["bias_tokens"] = torch.rand((rows, vocab), generator=_gen(seed, 8), device="cuda").topk(b, dim=1).indices.to(torch.int32).view(-1)
            s["bias_values"] = 5.0 * _randn(seed, 9, rows * b)
        if case["mask"]:
            # A grammar at one of four states: each allows a part of the vocabulary.
            words, g = (vocab + 31) // 32, _gen(seed, 10)
            s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (4, words), generator=g, device="cuda").to(torch.int32)
            s["mask"] &= torch.randint(-2 ** 31, 2 ** 31, (4, words), generator=g, device="cuda").to(torch.int32)
            s["mask_rows"] = _ints(seed, 11, -1, 4, rows)
        s["out"] = torch.empty_like(s["logits"])
    return s


# ---- one pass -----------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["kind"] == "rope":
        cos, sin = _cos_sin(s["positions"], s["inv_freq"], s["scale"])
        return _rotated(s["x"].float(), cos, sin, c["interleaved"]).to(s["x"].dtype)
    if c["kind"] == "qk_norm":
        cos, sin = _cos_sin(s["positions"], s["inv_freq"], 1.0)
        q = _rotated(_normed(s["q"].float(), s["q_weight"]), cos, sin, c["interleaved"])
        k = _rotated(_normed(s["k"].float(), s["k_weight"]), cos, sin, c["interleaved"])
        return q.to(s["q"].dtype), k.to(s["k"].dtype)
    if c["kind"] == "lora":
        return _adapted(s, c)
    return _logits(s, c)


def _run_own(s, c):
    import mtlqwen_amd as q4k
    if c["kind"] == "rope":
        return q4k.rope(s["x"], s["inv_freq"], s["positions"], s["y"], interleaved=c["interleaved"], scale=s["scale"])
    if c["kind"] == "qk_norm":
        return q4k.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["inv_freq"], s["positions"], s["q_out"], s["k_out"],
                                interleaved=c["interleaved"], eps=EPS)
    if c["kind"] == "lora":
        return q4k.lora(s["x"], s["a"], s["b"], s["ids"], c["m"], s["y"], auxiliary=s["aux"], query_counts=s["counts"], ranks=s["ranks"],
                        scales=s["scales"])
    return q4k.process_logits(s["logits"], s["out"], tokens=s["tokens"], slots=s["slots"], lengths=s["lengths"], prompts=s["prompts"],
                              repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                              bias_offsets=s.get("bias_offsets"), bias_tokens=s.get("bias_tokens"), bias_values=s.get("bias_values"),
                              mask=s.get("mask"), mask_rows=s.get("mask_rows"))


def _cos_sin(positions, inv_freq, scale):
    """Angles in 64 bits: at far positions 32 lose them."""
    angle = positions.double().unsqueeze(1) * inv_freq
    return (scale * torch.cos(angle)).float().unsqueeze(1), (scale * torch.sin(angle)).float().unsqueeze(1)


def _rotated(x, cos, sin, interleaved):
    h = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., 2 * h:]], dim=-1)


def _normed(x, weight):
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight


def _adapted(s, c):
    m, k, n, r = c["m"], c["k"], c["n"], c["rank"]
    counts = torch.tensor(s["counts"], device="cuda")
    row_adapter = torch.repeat_interleave(s["ids"], counts, output_size=m)
    # Every adapter's columns side by side; a row keeps those of its own adapter, up to its rank.
    mine = row_adapter.unsqueeze(1) == torch.arange(8, device="cuda")
    used = torch.arange(r, device="cuda") < s["ranks"].unsqueeze(1)
    factor = (mine.unsqueeze(2) & used) * s["scales"].view(8, 1)
    u = (s["x"].float() @ s["a"].float().view(8 * r, k).t()) * factor.view(m, 8 * r)
    y = u @ s["b"].float().transpose(1, 2).reshape(8 * r, n)
    if s["aux"] is not None:
        y = s["aux"].float() + y
    return y.to(s["x"].dtype)


def _logits(s, c):
    rows, vocab = c["rows"], c["vocab"]
    at = torch.arange(c["history"], device="cuda")
    text = s["tokens"][s["slots"].long()].long()
    present = (at < s["lengths"].unsqueeze(1)).float()
    written = present * (at >= s["prompts"].unsqueeze(1))
    seen = torch.zeros((rows, vocab), device="cuda").scatter_add_(1, text, present) > 0
    count = torch.zeros((rows, vocab), device="cuda").scatter_add_(1, text, written)
    p = s["repetition"].unsqueeze(1)
    v = s["logits"].float()
    v = torch.where(seen, torch.where(v > 0, v / p, v * p), v)
    v = v - s["frequency"].unsqueeze(1) * count - s["presence"].unsqueeze(1) * (count > 0)
    if c["bias"]:
        v = v.scatter_add(1, s["bias_tokens"].view(rows, -1).long(), s["bias_values"].view(rows, -1))
    if c["mask"]:
        words = s["mask"][s["mask_rows"].clamp(min=0).long()]
        bits = (words.unsqueeze(2) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        allowed = (bits.view(rows, -1)[:, :vocab] == 1) | (s["mask_rows"] < 0).unsqueeze(1)
        v = v.masked_fill(~allowed, float("-inf"))
    return v.to(s["logits"].dtype)


# ---- what a pass cannot do without ------------------------------------------------

def work(case):
    """Each input read once, each output written once."""
    kind, e = case["kind"], _size(case)
    if kind in ("rope", "qk_norm"):
        heads = case["heads"] + case.get("kv_heads", 0)
        values = case["rows"] * heads * case["dim"]
        flops = 3 * case["rows"] * heads * case["rot"] + (4 * values if kind == "qk_norm" else 0)
        return {"bytes": 2 * values * e + 4 * case["rows"] + 4 * case["rot"] + (8 * case["dim"] if kind == "qk_norm" else 0), "flops": flops}
    if kind == "lora":
        m, k, n = case["m"], case["k"], case["n"]
        ranks, ids, counts = _adapter_ranks(case), _adapter_ids(case), _counts(case["m"], case["queries"])
        read = sum(2 * ranks[a] * (k + n) for a in set(ids) if a >= 0)
        adapted = sum(c for a, c in zip(ids, counts) if a >= 0)
        flops = sum(2 * c * ranks[a] * (k + n) for a, c in zip(ids, counts) if a >= 0)
        return {"bytes": read + adapted * k * e + m * n * e * (2 if case["aux"] else 1), "flops": max(flops, m * n)}
    rows, vocab = case["rows"], case["vocab"]
    read = 4 * rows * (case["history"] * 3 // 4 + 6) + 8 * rows * case["bias"] + (vocab // 8 * min(4, rows) if case["mask"] else 0)
    return {"bytes": 2 * rows * vocab * e + read, "flops": rows * vocab}


# ---- the same in 64 bits -----------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("rope", "qk_norm"):
        # Pairs as complex numbers, turned by exp(i position frequency).
        angle = torch.outer(s["positions"].double(), s["inv_freq"])
        turn = torch.polar(torch.full_like(angle, s["scale"]), angle).unsqueeze(1)

        def rotate(x):
            h, y = case["rot"] // 2, x.clone()
            first, second = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if case["interleaved"] else (slice(0, h), slice(h, 2 * h))
            z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
            y[..., first], y[..., second] = z.real, z.imag
            return y

        def norm(x, weight):
            return x / ((x ** 2).sum(dim=-1, keepdim=True) / case["dim"] + EPS).sqrt() * weight.double()

        if kind == "rope":
            return rotate(s["x"].double())
        return rotate(norm(s["q"].double(), s["q_weight"])), rotate(norm(s["k"].double(), s["k_weight"]))
    if kind == "lora":
        y = torch.zeros(case["m"], case["n"], device="cuda", dtype=torch.float64) if s["aux"] is None else s["aux"].double()
        start = 0
        for a, rows in zip(_adapter_ids(case), s["counts"]):
            if a >= 0:
                r, here = _adapter_ranks(case)[a], slice(start, start + rows)
                u = s["x"][here].double() @ s["a"][a, :r].double().t().contiguous()
                y[here] += s["scales"][a].double() * (u @ s["b"][a, :, :r].double().t().contiguous())
            start += rows
        return y
    rows, vocab = case["rows"], case["vocab"]
    v = s["logits"].double()
    for r in range(rows):
        text = s["tokens"][int(s["slots"][r]), :int(s["lengths"][r])].long()
        every = torch.bincount(text, minlength=vocab)
        written = torch.bincount(text[int(s["prompts"][r]):], minlength=vocab).double()
        p = s["repetition"][r].double()
        x = v[r]
        x = torch.where(every == 0, x, torch.maximum(x, torch.zeros_like(x)) / p + torch.minimum(x, torch.zeros_like(x)) * p)
        x = x - (written * s["frequency"][r].double() + (written != 0).double() * s["presence"][r].double())
        if case["bias"]:
            mine = slice(r * case["bias"], (r + 1) * case["bias"])
            x[s["bias_tokens"][mine].long()] += s["bias_values"][mine].double()
        if case["mask"] and int(s["mask_rows"][r]) >= 0:
            token = torch.arange(vocab, device="cuda")
            word = s["mask"][int(s["mask_rows"][r])].long()[token // 32]
            x[(word >> (token % 32)) % 2 == 0] = -math.inf
        v[r] = x
    return v
