"""Operators of a server that decodes a batch of sequences over a paged cache, with drafted tokens.

* ``append``  rotates the new rows' queries and keys by their positions and puts keys and values on the sequences' pages.
* ``attend``  attention of the new rows over the pages of their sequence and over a prefix that all sequences share.
* ``verify``  which drafted tokens stand against the target's probabilities, and the token that follows them.

A batch is packed: ``row_start`` [seqs + 1] says which rows belong to a sequence, ``length`` [seqs] how many tokens it has in its
own pages, those of this call included.  Row i of n of a sequence is its token ``length - n + i``, at the position ``prefix`` behind
that.  Head counts and sizes are those of the repository's decoders, the vocabulary its benchmark's.
"""
import ctypes as C
import math
import random

import torch

own = False

HEADS = {2048: (16, 4), 4096: (32, 8), 5120: (40, 8)}  # width of the decoder -> query heads, key heads
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
THETA = 1e6
NEVER = -math.inf


# ── what is measured ────────────────────────────────────────────────────────
def listed():
    return [
        # one token of one chat: the smallest call there is
        {"name": "append_token", "op": "append", "type": "f16", "width": 4096, "dim": 128, "seqs": 1, "rows": 1, "ragged": False, "length": 600, "page": 16, "order": "heads",
         "layout": "halves", "part": 1.0, "scaling": "none", "fused": False},
        # a server's step: sequences with zero to four drafts each, half of every head rotated, projections side by side in one row
        {"name": "append_drafts", "op": "append", "type": "bf16", "width": 4096, "dim": 128, "seqs": 48, "rows": 5, "ragged": True, "length": 3000, "page": 64, "order": "tokens",
         "layout": "adjacent", "part": 0.5, "scaling": "linear", "fused": True},
        # chunks of three long prompts, far behind the positions the frequencies were made for
        {"name": "append_prompts", "op": "append", "type": "f16", "width": 5120, "dim": 128, "seqs": 3, "rows": 2048, "ragged": True, "length": 90000, "page": 32, "order": "heads",
         "layout": "halves", "part": 1.0, "scaling": "ramp", "fused": True},
        # one token of one chat again
        {"name": "attend_token", "op": "attend", "type": "f16", "width": 4096, "dim": 128, "seqs": 1, "rows": 1, "ragged": False, "length": 600, "page": 16, "order": "heads", "prefix": 0,
         "window": 0},
        # a server's batch: sequences from a few tokens to thousands
        {"name": "attend_batch", "op": "attend", "type": "bf16", "width": 4096, "dim": 128, "seqs": 32, "rows": 1, "ragged": True, "length": 9000, "page": 16, "order": "tokens", "prefix": 0,
         "window": 0},
        # two long documents
        {"name": "attend_long", "op": "attend", "type": "f16", "width": 4096, "dim": 128, "seqs": 2, "rows": 1, "ragged": False, "length": 100001, "page": 128, "order": "heads", "prefix": 0,
         "window": 0},
        # the target's pass over drafted tokens, heads of 64
        {"name": "attend_drafts", "op": "attend", "type": "f16", "width": 5120, "dim": 64, "seqs": 16, "rows": 6, "ragged": True, "length": 4000, "page": 32, "order": "heads", "prefix": 0,
         "window": 0},
        # the last chunks of two prompts
        {"name": "attend_prompts", "op": "attend", "type": "bf16", "width": 5120, "dim": 128, "seqs": 2, "rows": 1500, "ragged": True, "length": 4100, "page": 32, "order": "heads", "prefix": 0,
         "window": 0},
        # many short chats behind one long system prompt
        {"name": "attend_shared", "op": "attend", "type": "bf16", "width": 4096, "dim": 128, "seqs": 64, "rows": 1, "ragged": True, "length": 500, "page": 16, "order": "heads", "prefix": 8192,
         "window": 0},
        # a few samples of one prompt, with drafts
        {"name": "attend_samples", "op": "attend", "type": "f16", "width": 2048, "dim": 128, "seqs": 5, "rows": 4, "ragged": True, "length": 200, "page": 16, "order": "heads", "prefix": 1900,
         "window": 0},
        # one chat whose drafts come from a look-up, so that they have no probabilities
        {"name": "verify_lookup", "op": "verify", "type": "f16", "vocab": 32768, "seqs": 1, "rows": 5, "ragged": False, "draft": False, "greedy": 0.0, "masked": 0.0},
        # a server's batch: up to five drafts a sequence, some sequences without sampling, the table's padding masked
        {"name": "verify_batch", "op": "verify", "type": "f16", "vocab": 151936, "seqs": 48, "rows": 6, "ragged": True, "draft": True, "greedy": 0.2, "masked": 0.002},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "verify"])
    if op == "verify":
        vocab = rng.choice([32768, 151936, _log_int(rng, 1000, 152000)])
        seqs, rows = _log_int(rng, 1, 48), rng.randint(1, 8)
        while seqs * rows > 48 * 6:
            seqs //= 2
        kind = rng.choice(["f16", "bf16", "f32"])
        if kind == "f32":
            seqs = max(1, seqs // 2)
        return {"op": op, "type": kind, "vocab": vocab, "seqs": seqs, "rows": rows, "ragged": rng.random() < 0.7, "draft": rng.random() < 0.7, "greedy": rng.choice([0.0, 0.3, 1.0]),
                "masked": rng.choice([0.0, 0.01, 0.6])}
    width, dim = rng.choice([2048, 4096, 5120]), rng.choice([64, 128, 128, 256])
    case = {"op": op, "type": rng.choice(["f16", "bf16"]), "width": width, "dim": dim, "seqs": _log_int(rng, 1, 96)}
    case["rows"] = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, 2000)])
    while case["seqs"] * case["rows"] > 4000:
        case["seqs"] = max(1, case["seqs"] // 2)
    case["ragged"] = rng.random() < 0.7
    case["length"] = max(case["rows"], _log_int(rng, 1, 100000))
    heads, kv = HEADS[width]
    most = 180_000 * 128 // dim  # tokens on the pages
    while case["seqs"] * case["length"] > most or 4 * case["seqs"] * case["rows"] * heads * dim * case["length"] > 2.2e11:
        if case["length"] > 2 * case["rows"] and case["length"] > 600:
            case["length"] //= 2
        elif case["seqs"] > 1:
            case["seqs"] //= 2
        else:
            case["rows"] = case["length"] = max(1, case["length"] // 2)
    case["page"] = rng.choice([16, 32, 64, 128, rng.randint(1, 100)])
    case["order"] = rng.choice(["heads", "tokens"])
    if op == "append":
        return {**case, "layout": rng.choice(["halves", "adjacent"]), "part": rng.choice([1.0, 1.0, 0.5, 0.25]), "scaling": rng.choice(["none", "linear", "base", "ramp"]),
                "fused": rng.random() < 0.5}
    case["prefix"] = rng.choice([0, 0, _log_int(rng, 1, 16000)])
    if 4 * case["seqs"] * case["rows"] * heads * dim * case["prefix"] > 1e11:
        case["prefix"] = 0
    return {**case, "window": rng.choice([0, 0, _log_int(rng, 1, 8000)])}


def _rows_and_lengths(case):
    """Rows and tokens of each sequence, the same for every seed: a few sequences near the most, most of them well below."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    rows = [r.randint(1, case["rows"]) if case["ragged"] else case["rows"] for _ in range(case["seqs"])]
    rows[0] = case["rows"]
    if "length" not in case:
        return rows, None
    lengths = [_log_int(r, max(1, case["length"] // 32), case["length"]) if case["ragged"] else case["length"] for _ in range(case["seqs"])]
    lengths[0] = case["length"]
    return rows, [max(n, m) for n, m in zip(rows, lengths)]


# ── inputs ──────────────────────────────────────────────────────────────────
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed((int(seed) & 0xFFFFFFFF) * 1009 + 7)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(rows):
    at = [0]
    for n in rows:
        at.append(at[-1] + n)
    return _ints(at)


def _pages(case, lengths, g):
    """Page tables over a pool whose pages were handed out in no order, and the pool's size."""
    size, prefix = case["page"], case.get("prefix", 0)
    need, wide = [-(-n // size) for n in lengths], -(-prefix // size)
    pages = sum(need) + wide + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return pages, table, order[at:at + wide].contiguous() if wide else torch.zeros(1, dtype=torch.int32, device="cuda")


def _pool(case, pages, kv, g):
    """[pages, key heads, page, dim] as seen, in memory with the heads or the tokens of a page outermost."""
    size, dim = case["page"], case["dim"]
    shape = (pages, kv, size, dim) if case["order"] == "heads" else (pages, size, kv, dim)
    pool = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(DTYPES[case["type"]])
    return pool if case["order"] == "heads" else pool.transpose(1, 2)


def _frequencies(case):
    """Radians a position of each pair, as float64, and the factor of sine and cosine; scaled so that a model made for 8192
    positions reads 131072."""
    n, kind, s, known = max(2, int(case["dim"] * case["part"])), case["scaling"], 16.0, 8192.0
    at = torch.arange(0, n, 2, dtype=torch.float64, device="cuda") / n
    base = THETA * s ** (n / max(1, n - 2)) if kind == "base" else THETA
    freq, factor = base ** -at, 1.0
    if kind == "linear":
        freq = freq / s
    if kind == "ramp":  # pairs that turn over 32 times in the known length stay, those that do not turn once are stretched
        turns = known * freq / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        freq, factor = freq * keep + freq / s * (1 - keep), 0.1 * math.log(s) + 1
    return freq, float(torch.tensor(factor, dtype=torch.float32))


def _cache_prepare(case, seed):
    g, (heads, kv), dtype, dim = _generator(seed), HEADS[case["width"]], DTYPES[case["type"]], case["dim"]
    rows, lengths = _rows_and_lengths(case)
    total = sum(rows)
    pages, table, prefix_table = _pages(case, lengths, g)
    s = {"case": case, "heads": heads, "kv": kv, "row_start": _starts(rows), "length": _ints(lengths), "table": table, "prefix_table": prefix_table, "total": total, "pages": pages,
         "k_pool": _pool(case, pages, kv, g), "v_pool": _pool(case, pages, kv, g)}
    if case["op"] == "attend":
        s["q"] = (torch.randn(total, heads, dim, generator=g, device="cuda") * 1.5).to(dtype)
        s["out"] = torch.zeros_like(s["q"])
        return s
    new = torch.randn(total, heads + 2 * kv, dim, generator=g, device="cuda").to(dtype)
    parts = (new[:, :heads], new[:, heads:heads + kv], new[:, heads + kv:])
    s["q"], s["k"], s["v"] = parts if case["fused"] else tuple(p.contiguous() for p in parts)
    s["q_out"] = torch.zeros(total, heads, dim, dtype=dtype, device="cuda")
    s["freq"], s["factor"] = _frequencies(case)
    return s


def _verify_prepare(case, seed):
    g, (rows, _), V, B = _generator(seed), _rows_and_lengths(case), case["vocab"], case["seqs"]
    dtype, steps, total = DTYPES[case["type"]], max(1, case["rows"] - 1), sum(rows)
    masked = int(V * case["masked"])

    def logits(n):  # a few likely tokens over a long tail
        a = torch.randn(n, V, generator=g, device="cuda") * 2.0
        a.scatter_add_(1, torch.randint(0, V, (n, 6), generator=g, device="cuda"), torch.rand(n, 6, generator=g, device="cuda") * 8 + 4)
        a[:, V - masked:] = NEVER
        return a

    target = logits(total)
    start = _starts(rows)
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), _ints(rows))
    step = torch.arange(total, device="cuda") - start[:-1][seq]
    s = {"case": case, "row_start": start, "total": total, "steps": steps, "draft": None}
    drafts = step < _ints(rows)[seq] - 1  # rows that are followed by a drafted token
    model = torch.zeros(steps, B, V, device="cuda")
    model[step[drafts], seq[drafts]] = target[drafts] + 0.7 * torch.randn(int(drafts.sum()), V, generator=g, device="cuda")
    chance = torch.rand(total, V, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
    given = torch.full((total, V), NEVER, device="cuda")
    given[drafts] = model[step[drafts], seq[drafts]]
    tokens = torch.randint(0, V - masked, (total,), generator=g, device="cuda")
    drawn = (given - (-chance.log()).log()).argmax(1)
    follow = torch.nonzero(drafts)[:, 0]
    tokens[follow + 1] = drawn[follow]
    if case["draft"]:
        s["draft"] = model.to(dtype)
    temperature = torch.rand(B, generator=g, device="cuda") * 0.8 + 0.5
    temperature[torch.arange(B, device="cuda") < round(B * case["greedy"])] = 0
    s |= {"target": target.to(dtype), "tokens": tokens.to(torch.int32), "temperature": temperature, "random": torch.rand(total, generator=g, device="cuda"),
          "out": torch.zeros(total, dtype=torch.int32, device="cuda"), "accepted": torch.zeros(B, dtype=torch.int32, device="cuda")}
    return s


def prepare(case, seed):
    return _verify_prepare(case, seed) if case["op"] == "verify" else _cache_prepare(case, seed)


# ── plain forms ─────────────────────────────────────────────────────────────
def _row_places(s):
    """Sequence and token (in its own pages) of every row."""
    start, length = s["row_start"].long(), s["length"].long()
    rows = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(start[1:], rows, right=True)
    return seq, length[seq] - start[seq + 1] + rows


def _rotate(x, cos, sin, layout):
    n = 2 * cos.shape[-1]
    a, rest = x[..., :n].float(), x[..., n:].float()
    first, second = (a[..., :n // 2], a[..., n // 2:]) if layout == "halves" else (a[..., 0::2], a[..., 1::2])
    one, two = first * cos - second * sin, second * cos + first * sin
    turned = torch.cat([one, two], -1) if layout == "halves" else torch.stack([one, two], -1).flatten(-2)
    return torch.cat([turned, rest], -1).to(x.dtype)


def _append_plain(s):
    case = s["case"]
    seq, token = _row_places(s)
    angle = token.double()[:, None, None] * s["freq"]
    cos, sin = (torch.cos(angle) * s["factor"]).float(), (torch.sin(angle) * s["factor"]).float()
    page, slot = s["table"].long()[seq, token // case["page"]], token % case["page"]
    s["q_out"].copy_(_rotate(s["q"], cos, sin, case["layout"]))
    s["k_pool"][page, :, slot] = _rotate(s["k"], cos, sin, case["layout"])
    s["v_pool"][page, :, slot] = s["v"]
    return [s["q_out"], s["k_pool"], s["v_pool"]]


def _attend_plain(s):
    case, size = s["case"], s["case"]["page"]
    start, length = s["row_start"].long(), s["length"].long()
    B, G, group, prefix = case["seqs"], s["kv"], s["heads"] // s["kv"], case["prefix"]
    n = start[1:] - start[:-1]
    i = torch.arange(case["rows"], device="cuda")
    row, live = (start[:-1, None] + i).clamp(max=s["total"] - 1), i < n[:, None]
    q = s["q"][row].float().view(B, case["rows"], G, group, case["dim"]) * case["dim"] ** -0.5
    at = torch.arange(s["table"].shape[1] * size, device="cuda")
    page = s["table"].long()[:, at // size].clamp(min=0)
    k, v = s["k_pool"][page, :, at % size].float(), s["v_pool"][page, :, at % size].float()  # [B, L, G, dim]
    place = (length - n)[:, None] + i  # [B, rows]: the row's token
    seen = at <= place[..., None]
    score = torch.einsum("brgjd,blgd->bgjrl", q, k)
    if prefix:
        ahead = torch.arange(prefix, device="cuda")
        page = s["prefix_table"].long()[ahead // size]
        pk, pv = s["k_pool"][page, :, ahead % size].float(), s["v_pool"][page, :, ahead % size].float()  # [P, G, dim]
        score = torch.cat([torch.einsum("brgjd,lgd->bgjrl", q, pk), score], -1)
        seen = torch.cat([torch.ones(B, case["rows"], prefix, dtype=torch.bool, device="cuda"), seen], -1)
    if case["window"]:
        seen = seen & (torch.arange(prefix + at.numel(), device="cuda") > place[..., None] + prefix - case["window"])
    score = score.masked_fill(~seen[:, None, None], NEVER)
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    weight = weight / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.einsum("bgjrl,blgd->brgjd", weight[..., prefix:], v)
    if prefix:
        out = out + torch.einsum("bgjrl,lgd->brgjd", weight[..., :prefix], pv)
    s["out"][row[live]] = out.reshape(B, case["rows"], s["heads"], case["dim"])[live].to(s["out"].dtype)
    return s["out"]


def _chances(logits, temperature):
    """Probabilities in 64 bits; temperature 0: all on the lowest index of the largest logit."""
    a = logits.double()
    top = a.amax(-1, keepdim=True)
    cold = temperature == 0
    e = torch.exp((a - top) / torch.where(cold, 1.0, temperature.double())[..., None])
    index = torch.arange(a.shape[-1], device="cuda")
    first = torch.where(a == top, index, a.shape[-1]).amin(-1, keepdim=True)
    return torch.where(cold[..., None], (index == first).double(), e / e.sum(-1, keepdim=True))


def _verify_plain(s):
    case, start = s["case"], s["row_start"].long()
    B, R = case["seqs"], case["rows"]
    n = (start[1:] - start[:-1])[:, None]
    i = torch.arange(R, device="cuda")
    row = (start[:-1, None] + i).clamp(max=s["total"] - 1)  # [B, R]
    p = _chances(s["target"], s["temperature"][torch.searchsorted(start[1:], torch.arange(s["total"], device="cuda"), right=True)])
    drafted = s["tokens"].long()[(row[:, :-1] + 1).clamp(max=s["total"] - 1)]  # [B, R - 1]
    px = p[row[:, :-1], drafted]
    qx = torch.ones_like(px)
    q = None
    if s["draft"] is not None:
        q = _chances(s["draft"].transpose(0, 1), s["temperature"][:, None].expand(B, s["steps"]))
        qx = q[torch.arange(B, device="cuda")[:, None], i[:-1], drafted]
    stands = (s["random"].double()[row[:, :-1]] * qx < px) & (i[:-1] < n - 1)
    kept = stands.long().cumprod(1).sum(1)  # [B]: drafts before the first that falls
    at = row.gather(1, kept[:, None])[:, 0]
    weight = p[at]
    falls = kept < n[:, 0] - 1
    step = kept.clamp(max=s["steps"] - 1)
    if q is not None:
        less = q[torch.arange(B, device="cuda"), step]
    else:
        token = torch.cat([drafted, drafted.new_zeros(B, 1)], 1).gather(1, kept[:, None])
        less = (torch.arange(case["vocab"], device="cuda") == token).double()
    rest = torch.where(falls[:, None], (weight - less).clamp(min=0), weight)
    weight = torch.where(rest.sum(-1, keepdim=True) > 0, rest, weight)
    run = weight.cumsum(-1)
    last = torch.arange(start[:-1].numel(), device="cuda")
    chance = s["random"].double()[start[1:] - 1] * run[:, -1]
    index = torch.arange(case["vocab"], device="cuda")
    best = torch.where(weight > 0, index, -1).amax(-1)
    token = torch.minimum((run <= chance[:, None]).sum(-1), best)
    said = torch.cat([drafted, drafted.new_zeros(B, 1)], 1)
    said = torch.where(i < kept[:, None], said, torch.where(i == kept[:, None], token[last][:, None], -1))
    live = i < n
    s["out"][row[live]] = said[live].to(torch.int32)
    s["accepted"].copy_(kept)
    return [s["out"], s["accepted"]]


# ── the framework's operators ───────────────────────────────────────────────
_CONTEXT = []


def _context():
    if not _CONTEXT:
        from smelt_b200 import capi

        _CONTEXT.append(capi.Context(0))
    return _CONTEXT[0]


def _cache_and_batch(s):
    from smelt_b200 import capi

    case, k = s["case"], s["k_pool"]
    cache = capi.PagedCache(precision=capi.PAGED_F16 if case["type"] == "f16" else capi.PAGED_BF16, n_q=s["heads"], n_kv=s["kv"], head_dim=case["dim"], page_size=case["page"],
                            n_pages=s["pages"], page_stride=k.stride(0), head_stride=k.stride(1), token_stride=k.stride(2), k=k.data_ptr(), v=s["v_pool"].data_ptr())
    batch = capi.PagedBatch(n_seqs=case["seqs"], rows=s["total"], max_rows=case["rows"], table_stride=s["table"].shape[1], prefix_length=case.get("prefix", 0),
                            row_start=s["row_start"].data_ptr(), length=s["length"].data_ptr(), table=s["table"].data_ptr(), prefix_table=s["prefix_table"].data_ptr())
    return cache, batch


def _append_own(s):
    from smelt_b200 import capi

    if "call" not in s:
        case, (cache, batch) = s["case"], _cache_and_batch(s)
        rope = capi.RopeDesc(rope_dim=2 * s["freq"].numel(), layout=capi.ROPE_HALVES if case["layout"] == "halves" else capi.ROPE_ADJACENT, factor=s["factor"], freq=s["freq"].data_ptr())
        s["call"] = (C.byref(cache), C.byref(batch), C.byref(rope), s["q"].data_ptr(), s["q"].stride(0), s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0),
                     s["q_out"].data_ptr(), s["q_out"].stride(0))
    _context().call("paged_append", *s["call"])
    return [s["q_out"], s["k_pool"], s["v_pool"]]


def _attend_own(s):
    if "call" not in s:
        case, (cache, batch), size = s["case"], _cache_and_batch(s), C.c_size_t()
        _context().call("paged_attention_workspace", C.byref(cache), C.byref(batch), C.byref(size))
        s["workspace"] = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        s["call"] = (C.byref(cache), C.byref(batch), s["q"].data_ptr(), s["q"].stride(0), s["out"].data_ptr(), s["out"].stride(0), case["dim"] ** -0.5, case["window"],
                     s["workspace"].data_ptr(), size.value)
    _context().call("paged_attention", *s["call"])
    return s["out"]


def _verify_own(s):
    from smelt_b200 import capi

    if "call" not in s:
        case, draft, size = s["case"], s["draft"], C.c_size_t()
        args = capi.VerifyArgs(precision={"f16": capi.LOGITS_F16, "bf16": capi.LOGITS_BF16, "f32": capi.LOGITS_F32}[case["type"]], n_seqs=case["seqs"], rows=s["total"],
                               vocab=case["vocab"], target_stride=s["target"].stride(0), row_start=s["row_start"].data_ptr(), target=s["target"].data_ptr(), tokens=s["tokens"].data_ptr(),
                               temperature=s["temperature"].data_ptr(), random=s["random"].data_ptr(), out_tokens=s["out"].data_ptr(), accepted=s["accepted"].data_ptr())
        if draft is not None:
            args.draft, args.draft_step_stride, args.draft_seq_stride = draft.data_ptr(), draft.stride(0), draft.stride(1)
        _context().call("verify_drafts_workspace", C.byref(args), C.byref(size))
        s["workspace"] = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        args.workspace, args.workspace_bytes = s["workspace"].data_ptr(), size.value
        s["call"] = (C.byref(args),)
    _context().call("verify_drafts", *s["call"])
    return [s["out"], s["accepted"]]


_PLAIN = {"append": _append_plain, "attend": _attend_plain, "verify": _verify_plain}
_OWN = {"append": _append_own, "attend": _attend_own, "verify": _verify_own}


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state)


# ── the definitions again, in 64 bits, a sequence at a time ─────────────────
def _keys(pool, table, count, size):
    """The first `count` tokens of a table of pages: [key heads, count, dim]."""
    pages = pool[table[:-(-count // size)].long()].double()
    return pages.permute(1, 0, 2, 3).flatten(1, 2)[:, :count]


def _append_exact(case, s):
    outs = [s["q_out"].double(), s["k_pool"].double(), s["v_pool"].double()]
    start, length, n = s["row_start"].tolist(), s["length"].tolist(), 2 * s["freq"].numel()
    first = torch.arange(n // 2, device="cuda") if case["layout"] == "halves" else torch.arange(0, n, 2, device="cuda")
    second = first + (n // 2 if case["layout"] == "halves" else 1)

    def turn(x, c, sn):
        y = x.double().clone()
        y[..., first] = x[..., first].double() * c - x[..., second].double() * sn
        y[..., second] = x[..., first].double() * sn + x[..., second].double() * c
        return y

    for b, (r0, r1) in enumerate(zip(start, start[1:])):
        token = torch.arange(length[b] - (r1 - r0), length[b], device="cuda")
        phase = (token.double()[:, None] * s["freq"]).unsqueeze(1)
        c, sn = torch.cos(phase) * s["factor"], torch.sin(phase) * s["factor"]
        where = s["table"][b].long()[token // case["page"]]
        outs[0][r0:r1] = turn(s["q"][r0:r1], c, sn)
        outs[1][where, :, token % case["page"]] = turn(s["k"][r0:r1], c, sn)
        outs[2][where, :, token % case["page"]] = s["v"][r0:r1].double()
    return outs


def _attend_exact(case, s):
    start, length, P, G = s["row_start"].tolist(), s["length"].tolist(), case["prefix"], s["kv"]
    if sum((r1 - r0) * (P + n) for r0, r1, n in zip(start, start[1:], length)) * s["heads"] * case["dim"] > 1e11:
        return None
    out = torch.zeros(s["total"], s["heads"], case["dim"], dtype=torch.float64, device="cuda")
    ahead = [_keys(s[name], s["prefix_table"], P, case["page"]) for name in ("k_pool", "v_pool")]
    for b, (r0, r1) in enumerate(zip(start, start[1:])):
        k, v = (torch.cat([ahead[i], _keys(s[name], s["table"][b], length[b], case["page"])], 1) for i, name in enumerate(("k_pool", "v_pool")))
        q = s["q"][r0:r1].double().transpose(0, 1).reshape(G, -1, case["dim"])  # heads of a group, rows
        score = q @ k.transpose(1, 2) / math.sqrt(case["dim"])
        mine = (torch.arange(P + length[b] - (r1 - r0), P + length[b], device="cuda")).repeat(s["heads"] // G)[:, None]
        key = torch.arange(P + length[b], device="cuda")
        hidden = key > mine
        if case["window"]:
            hidden = hidden | (mine - key >= case["window"])
        score.masked_fill_(hidden, NEVER)
        out[r0:r1] = (torch.softmax(score, -1) @ v).reshape(s["heads"], r1 - r0, case["dim"]).transpose(0, 1)
    return out


def _verify_exact(case, s):
    start, said, kept = s["row_start"].tolist(), [], []
    chance, tokens = s["random"].double(), s["tokens"].tolist()

    def law(a, t):
        a = a.double()
        if t == 0:
            one = torch.zeros_like(a)
            one[int(torch.nonzero(a == a.max())[0, 0])] = 1
            return one
        return torch.softmax(a / t, -1)

    for b, (r0, r1) in enumerate(zip(start, start[1:])):
        t, line = float(s["temperature"][b]), []
        for j in range(r1 - r0):
            p = law(s["target"][r0 + j], t)
            if j == r1 - r0 - 1:
                break
            x = tokens[r0 + j + 1]
            if s["draft"] is None:
                q = torch.zeros_like(p)
                q[x] = 1
            else:
                q = law(s["draft"][j, b], t)
            if not bool(chance[r0 + j] * q[x] < p[x]):
                rest = torch.relu(p - q)
                p = rest if float(rest.sum()) > 0 else p
                break
            line.append(x)
        run = p.cumsum(0)
        past = torch.nonzero(run > chance[r1 - 1] * run[-1])
        kept.append(len(line))
        line.append(int(past[0, 0]) if past.numel() else int(torch.nonzero(p)[-1, 0]))
        said += line + [-1] * (r1 - r0 - len(line))
    return [_ints(said), _ints(kept)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append_exact, "attend": _attend_exact, "verify": _verify_exact}[case["op"]](case, s)


# ── what a pass cannot do without ───────────────────────────────────────────
def work(case):
    size = DTYPES[case["type"]].itemsize
    rows, lengths = _rows_and_lengths(case)
    total = sum(rows)
    if case["op"] == "verify":
        read = total + (total - case["seqs"] if case["draft"] else 0)
        return {"bytes": read * case["vocab"] * size + total * 12 + case["seqs"] * 12, "flops": 3 * read * case["vocab"]}
    heads, kv = HEADS[case["width"]]
    dim = case["dim"]
    if case["op"] == "append":
        return {"bytes": 2 * total * (heads + 2 * kv) * dim * size, "flops": 3 * total * (heads + kv) * dim * case["part"]}
    P, W = case["prefix"], case["window"] or 1 << 40
    pairs = sum(min(W, P + m - n + i + 1) for n, m in zip(rows, lengths) for i in range(n))
    keys = sum(min(m, W + n - 1) for n, m in zip(rows, lengths)) + min(P, max(min(P, max(0, W + n - 1 - m)) for n, m in zip(rows, lengths)))
    return {"bytes": (2 * keys * kv + 2 * total * heads) * dim * size, "flops": 4 * pairs * heads * dim}
