"""Attention over a long stream of tokens, as cases that can be timed and compared: windows with sinks in training and prefill,
and the paged cache that serves single new tokens (append, attention, eviction by accumulated weight).

`own` false: the operators in plain form, elementary torch operations in 32 bits.  `own` true: this package's entry points.

A case is a dict of plain values.  op "window": batch, heads, kv_heads, len (of keys), q_len, window, sinks, causal, ragged (sequences
of several lengths, padded), layout ("bhsd", or "bshd" as a projection leaves it), step (forward and backward), dtype.
op "attend", "append", "evict": batch, heads, kv_heads, len, page, ragged, dtype and what the operator takes.
"""
import math

import torch

own = False

DIM = 128
SCALE = 1 / math.sqrt(DIM)
GOLDEN = 0.6180339887498949


def _window(name, heads, kv_heads, length, window, sinks, *, batch=1, q_len=0, causal=True, ragged=False, layout="bhsd", step=False, dtype="bfloat16"):
    case = {"op": "window", "batch": batch, "heads": heads, "kv_heads": kv_heads, "len": length, "q_len": q_len or length, "window": window, "sinks": sinks,
            "causal": causal, "ragged": ragged, "layout": layout, "step": step, "dtype": dtype}
    return dict(case, name=name) if name else case


def _attend(name, batch, heads, kv_heads, length, page, *, ragged=False, window=0, sinks=0, accumulate=False, dtype="bfloat16"):
    case = {"op": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "len": length, "page": page, "ragged": ragged, "window": window, "sinks": sinks,
            "accumulate": accumulate, "dtype": dtype}
    return dict(case, name=name) if name else case


def _append(name, batch, kv_heads, length, new, page, *, ragged=False, dtype="bfloat16"):
    case = {"op": "append", "batch": batch, "kv_heads": kv_heads, "len": length, "new": new, "page": page, "ragged": ragged, "dtype": dtype}
    return dict(case, name=name) if name else case


def _evict(name, batch, kv_heads, length, budget, recent, sinks, page, *, ragged=False, dtype="bfloat16"):
    case = {"op": "evict", "batch": batch, "kv_heads": kv_heads, "len": length, "budget": budget, "recent": recent, "sinks": sinks, "page": page, "ragged": ragged, "dtype": dtype}
    return dict(case, name=name) if name else case


def listed():
    return [
        # A short clip through one head, without gradients: launches and host work are all of it.
        _window("window_small", 1, 1, 768, 128, 4),
        # A training batch of sequences of several lengths, padded to an odd one, grouped heads, in the layout of a projection.
        _window("window_ragged_step", 8, 2, 3136, 384, 16, batch=2, ragged=True, layout="bshd", step=True, dtype="float16"),
        # Training of a video layer: every token sees its neighbours on both sides and the tokens of the first tile.
        _window("window_video_step", 24, 24, 30720, 1152, 384, causal=False, step=True),
        # Prefill of a long stream with grouped heads: a causal window and a short prompt that stays visible.
        _window("window_prefill", 24, 6, 69120, 1536, 128),
        # One user's next token over a short cache: latency.
        _attend("attend_small", 1, 8, 8, 768, 16),
        # A serving batch in the middle of its answers: lengths between nothing and the longest.
        _attend("attend_ragged", 32, 24, 6, 16384, 64, ragged=True, dtype="float16"),
        # Long streams through a window with sinks: little of a large cache is visible.
        _attend("attend_window", 8, 16, 4, 115200, 128, window=8192, sinks=128),
        # The next tokens of a batch whose caches are kept to a budget: every slot's weight is added up.
        _attend("attend_weights", 16, 24, 6, 10240, 32, accumulate=True),
        # The new tokens of a serving batch.
        _append("append_token", 64, 8, 4096, 1, 16, ragged=True),
        # Two long prompts.
        _append("append_prompt", 2, 6, 0, 30720, 64),
        # A serving batch's step over its budget: one token of every head goes.
        _evict("evict_one", 32, 6, 4097, 4096, 256, 4, 16),
        # Prompts brought down to a budget.
        _evict("evict_prompt", 4, 6, 30720, 8192, 512, 128, 64, ragged=True),
    ]


def _log_uniform(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def _draw_heads(rng, most):
    group = rng.choice([1, 1, 2, 3, 4, 8])
    kv_heads = max(1, round(_log_uniform(rng, 1, max(1.01, most / group))))
    return kv_heads * group, kv_heads


def _draw_any(rng):
    op = rng.choice(["window", "window", "window", "attend", "attend", "append", "evict"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    ragged = rng.random() < 0.4
    batch = rng.choice([1, 1, 2, 3]) if op == "window" else max(1, round(_log_uniform(rng, 1, 64)))
    heads, kv_heads = _draw_heads(rng, 24)
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "window":
        length = round(_log_uniform(rng, 256, 40000))
        cross = rng.random() < 0.2 and not ragged  # a chunk of new queries against what came before
        return _window("", heads, kv_heads, length, round(_log_uniform(rng, 16, min(length, 4096))), rng.choice([0, 1, 4, 16, 64, 100, 128, 384]), batch=batch,
                       q_len=max(1, round(length * rng.uniform(0.05, 0.9))) if cross else length, causal=rng.random() < 0.7, ragged=ragged,
                       layout=rng.choice(["bhsd", "bhsd", "bshd"]), step=rng.random() < 0.6, dtype=dtype)
    length = round(_log_uniform(rng, 256, 100000))
    if op == "attend":
        accumulate = rng.random() < 0.4
        windowed = not accumulate and rng.random() < 0.3
        return _attend("", batch, heads, kv_heads, length, page, ragged=ragged, window=round(_log_uniform(rng, 16, length)) if windowed else 0,
                       sinks=rng.choice([0, 4, 64, 100]) if windowed else 0, accumulate=accumulate, dtype=dtype)
    if op == "append":
        new = rng.choice([1, 1, round(_log_uniform(rng, 2, 30000))])
        return _append("", batch, kv_heads, rng.choice([0, min(length, 20000)]), new, page, ragged=ragged, dtype=dtype)
    budget = max(64, round(length * rng.uniform(0.1, 0.99)))
    return _evict("", batch, kv_heads, max(length, budget + 1), budget, min(budget // 2, rng.choice([0, 32, 512])), min(budget // 4, rng.choice([0, 4, 64])), page, ragged=ragged, dtype=dtype)


def draw(rng):
    most_bytes, most_flops = 4e9, max(work(c)["flops"] for c in listed())
    while True:
        case = _draw_any(rng)
        w = work(case)
        small = w["bytes"] <= most_bytes and w["flops"] <= most_flops
        if case["op"] == "window":  # the plain form's products, which are larger than the visible ones
            small &= case["batch"] * case["heads"] * case["q_len"] * (2.5 * case["window"] + case["sinks"] + 64) <= 24 * 30720 * 3300 * (1 if case["step"] else 2)
        else:  # the pool, three times on the card, and what the plain form gathers of it
            small &= case["batch"] * case["kv_heads"] * (case["len"] + case.get("new", 0)) <= 8 * 4 * 115200
        if small:
            return case


# ---------------------------------------------------------------------------------------------------------------------
# what a case is made of
# ---------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Lengths of the batch's sequences: of a ragged one the longest, and others down to one token (a cache: to none) between."""
    n, most = case["batch"], case["len"]
    if not case["ragged"]:
        return [most] * n
    least = 1 if case["op"] == "window" else 0
    return [most] + [least + int((most - least) * ((i * GOLDEN + 0.3) % 1)) for i in range(1, n)]


def _counts(case):
    """New tokens of every sequence."""
    if not case["ragged"] or case["new"] == 1:
        return [case["new"]] * case["batch"]
    return [case["new"]] + [int(case["new"] * ((i * GOLDEN + 0.7) % 1)) for i in range(1, case["batch"])]


def _pairs(case, length):
    """Visible (row, key) pairs of a head of a sequence."""
    rows = case["q_len"] if not case["ragged"] else length
    first = length - rows  # position of the first row
    total = 0
    at = torch.arange(first, length, dtype=torch.int64)
    at = at[at >= 0]
    low = (at - case["window"] + 1).clamp_min(0)
    if case["causal"]:
        total = (at + 1 - low) + torch.minimum(torch.full_like(low, case["sinks"]), low)
    else:
        high = (at + case["window"]).clamp_max(length)
        total = (high - low) + torch.minimum(torch.full_like(low, case["sinks"]), low) + (min(case["sinks"], length) - high).clamp_min(0)
    return int(total.sum())


def work(case):
    lengths = _lengths(case)
    if case["op"] == "window":
        h, hk = case["heads"], case["kv_heads"]
        pairs = sum(_pairs(case, n) for n in lengths) * h
        rows = sum(lengths) if case["ragged"] else case["batch"] * case["q_len"]
        q_bytes, kv_bytes = rows * h * 2 * DIM, sum(lengths) * hk * 2 * DIM
        moved = 2 * q_bytes + 2 * kv_bytes + 4 * rows * h
        flops = 4 * DIM * pairs
        if case["step"]:
            moved += 4 * q_bytes + 4 * kv_bytes
            flops += 10 * DIM * pairs
        return {"bytes": moved, "flops": flops}
    if case["op"] == "attend":
        seen = lengths if not case["window"] else [min(n, case["window"]) + min(case["sinks"], max(0, n - case["window"])) for n in lengths]
        moved = sum(seen) * case["kv_heads"] * (4 * DIM + (8 if case["accumulate"] else 0)) + 4 * DIM * case["batch"] * case["heads"]
        return {"bytes": moved, "flops": 4 * DIM * sum(seen) * case["heads"]}
    if case["op"] == "append":
        rows = sum(_counts(case)) * case["kv_heads"]
        return {"bytes": rows * (8 * DIM + 8), "flops": 0}
    gone = [max(0, n - case["budget"]) for n in lengths]
    moved = 0.0  # rows that change their place, about: as many as are evicted below the budget
    for n, g in zip(lengths, gone):
        moved += g * case["budget"] / n if n else 0
    return {"bytes": case["kv_heads"] * (8 * sum(n for n, g in zip(lengths, gone) if g) + moved * (8 * DIM + 8)), "flops": 0}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape, size=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * size).to(dtype)

    lengths = _lengths(case)
    state = dict(case=case, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    if case["op"] == "window":
        def tensor(heads, n, size=1.0):
            return normal(case["batch"], n, heads, DIM, size=size) if case["layout"] == "bshd" else normal(case["batch"], heads, n, DIM, size=size)

        # scores with a spread of two: a few keys have most of a row's weight, as in trained layers
        q, k, v = tensor(case["heads"], case["q_len"], 2.0), tensor(case["kv_heads"], case["len"]), tensor(case["kv_heads"], case["len"])
        for t in (q, k, v):
            t.requires_grad_(case["step"])
        return dict(state, q=q, k=k, v=v, do=tensor(case["heads"], case["q_len"]))
    page, kv_heads, batch = case["page"], case["kv_heads"], case["batch"]
    new = case.get("new", 0)
    per = -(-(max(lengths) + new) // page)  # pages of a sequence
    pages = batch * per + 3
    pool = (pages, kv_heads, page)
    state["table"] = torch.randperm(pages, generator=g, device="cuda")[: batch * per].to(torch.int32).reshape(batch, per)
    state["k"], state["v"] = normal(*pool, DIM), normal(*pool, DIM)
    if case["op"] == "attend":
        if case["accumulate"]:
            state["weights"] = torch.rand(pool, generator=g, device="cuda") * 4
        return dict(state, q=normal(batch, case["heads"], 1, DIM, size=2.0))
    # weights of a few heavy tokens, many light ones, and some that are new and have none
    heavy = torch.exp(2 * torch.randn(pool, generator=g, device="cuda"))
    state["weights"] = torch.where(torch.rand(pool, generator=g, device="cuda") < 0.1, torch.zeros_like(heavy), heavy)
    if case["op"] == "append":
        state["positions"] = torch.randint(0, 1 << 20, pool, generator=g, device="cuda", dtype=torch.int32)
        state["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")
        return dict(state, new_k=normal(batch, kv_heads, new, DIM), new_v=normal(batch, kv_heads, new, DIM))
    # a cache that has been evicted from before: slots are in no order of positions, and every head has its own
    order = torch.rand((batch, kv_heads, per * page), generator=g, device="cuda").argsort(-1)
    flat = torch.empty(pool, dtype=torch.int32, device="cuda").fill_(-1)
    flat[state["table"].long()] = order.to(torch.int32).reshape(batch, kv_heads, per, page).permute(0, 2, 1, 3)
    # what is put back before every pass: eviction moves both along with the rows
    return dict(state, positions=flat, weights_before=state["weights"].clone(), positions_before=flat.clone())


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    return {"window": _run_window, "attend": _run_attend, "append": _run_append, "evict": _run_evict}[state["case"]["op"]](state)


def _run_window(s):
    case = s["case"]
    q, k, v, do = s["q"], s["k"], s["v"], s["do"]
    lengths = s["lengths"] if case["ragged"] else None
    with torch.set_grad_enabled(case["step"]):
        args = (q, k, v)
        if case["layout"] == "bshd":
            args = tuple(t.transpose(1, 2) for t in args)
        if own:
            import flex_block_attn_amd as fba

            o = fba.window_attn_func(*args, case["window"], sinks=case["sinks"], causal=case["causal"], lengths=lengths)
        else:
            o = _plain_window(*args, case["window"], case["sinks"], case["causal"], lengths)
    if not case["step"]:
        return o
    return (o.detach(), *torch.autograd.grad(o, (q, k, v), do.transpose(1, 2) if case["layout"] == "bshd" else do))


def _plain_window(q, k, v, window, sinks, causal, lengths):
    """Rows in chunks; a chunk's keys are those of the band around it and, apart from them, the sinks."""
    B, H, Sq, _ = q.shape
    Hk, Skv = k.shape[1], k.shape[2]
    G = H // Hk
    window, sinks = min(window, max(Sq, Skv)), min(sinks, Skv)
    C = min(Sq, max(64, window // 2))
    n = -(-Sq // C)
    ahead = 0 if causal else window - 1
    span = C + window - 1 + ahead
    first = Skv - Sq - (window - 1)  # position of the first chunk's first key
    qf = torch.nn.functional.pad(q.float(), (0, 0, 0, n * C - Sq)).reshape(B, Hk, G, n, C, DIM).transpose(2, 3).reshape(B, Hk, n, G * C, DIM)

    def bands(x):  # (B, Hk, n, DIM, span): keys from first + i * C on
        x = x.float()[:, :, max(0, first):]
        return torch.nn.functional.pad(x, (0, 0, max(0, -first), max(0, first + (n - 1) * C + span - Skv))).unfold(2, span, C)[:, :, :n]

    dev = q.device
    row = torch.arange(n * C, device=dev).reshape(n, C, 1)
    at = row + (Skv - Sq)
    key = (first + C * torch.arange(n, device=dev)).reshape(n, 1, 1) + torch.arange(span, device=dev)
    sink = torch.arange(sinks, device=dev)
    band_of = (at - key < window) & (key - at < ahead + 1) & (key > -1) & (key < Skv)
    sink_of = ((at - sink > window - 1) | (sink - at > ahead)) & ((sink < at + 1) if causal else (sink > -1))
    seen = torch.cat([band_of, sink_of], -1)[None, None]
    if lengths is not None:
        ends = lengths.long().reshape(B, 1, 1, 1, 1)
        keys = torch.cat([key.expand(n, C, span), sink.expand(n, C, sinks)], -1)
        seen = seen & (keys < ends) & (row < ends)
    seen = seen.expand(-1, -1, n, C, span + sinks)[:, :, :, None].expand(-1, -1, -1, G, -1, -1).reshape(seen.shape[0], 1, n, G * C, span + sinks)
    kf, vf = k.float()[:, :, None, :sinks], v.float()[:, :, None, :sinks]
    s = torch.cat([qf @ bands(k).contiguous(), (qf.reshape(B, Hk, 1, n * G * C, DIM) @ kf.transpose(-1, -2).contiguous()).reshape(B, Hk, n, G * C, sinks)], -1) * SCALE
    s = s.masked_fill(~seen, -math.inf)
    m = s.detach().amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    o = p[..., :span] @ bands(v).transpose(-1, -2).contiguous() + (p[..., span:].reshape(B, Hk, 1, n * G * C, sinks) @ vf).reshape(B, Hk, n, G * C, DIM)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return o.reshape(B, Hk, n, G, C, DIM).transpose(2, 3).reshape(B, H, n * C, DIM)[:, :, :Sq].to(q.dtype)


def _run_attend(s):
    case = s["case"]
    window = case["window"] or None
    if own:
        import flex_block_attn_amd as fba

        cache = fba.PagedCache(s["k"], s["v"], weights=s.get("weights"))
        o = fba.cache_attn_func(s["q"], cache, s["table"], s["lengths"], window=window, sinks=case["sinks"], accumulate=case["accumulate"])
    else:
        o = _plain_attend(s["q"], s["k"], s["v"], s["table"], s["lengths"], case["len"], window, case["sinks"], s.get("weights"))
    return (o, s["weights"]) if case["accumulate"] else o


def _plain_attend(q, k, v, table, lengths, most, window, sinks, weights):
    B, H = q.shape[:2]
    page, Hk = k.shape[2], k.shape[1]
    n = lengths.long()[:, None]
    if window is None or window + sinks >= most:
        window = most if window is None else window
        slot = torch.arange(most, device=q.device)[None].expand(B, -1)
        seen = (slot < n) & ((slot >= n - window) | (slot < sinks))
    else:
        tail = n - window + torch.arange(window, device=q.device)
        head = torch.arange(sinks, device=q.device)[None].expand(B, -1)
        slot = torch.cat([head, tail], 1)
        seen = torch.cat([(head < n) & (head < n - window), (tail >= 0) & (tail < n)], 1)
        slot = torch.where(seen, slot, torch.zeros_like(slot))
    pages = table.long().gather(1, slot // page)
    at = slot % page
    kf, vf = k[pages, :, at].float().transpose(1, 2), v[pages, :, at].float().transpose(1, 2)  # (B, Hk, slots, DIM)
    sc = (q.float().reshape(B, Hk, H // Hk, DIM) @ kf.transpose(-1, -2).contiguous()) * SCALE
    sc = sc.masked_fill(~seen[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    if weights is not None:  # slots that are not seen add nothing
        flat = (pages[:, None] * Hk + torch.arange(Hk, device=q.device)[None, :, None]) * page + at[:, None]
        weights.view(-1).index_add_(0, flat.reshape(-1), p.sum(2).reshape(-1))
    return (p @ vf.contiguous()).reshape(B, H, 1, DIM).to(q.dtype)


def _run_append(s):
    if own:
        import flex_block_attn_amd as fba

        cache = fba.PagedCache(s["k"], s["v"], positions=s["positions"], weights=s["weights"])
        lengths = fba.cache_append(cache, s["table"], s["lengths"], s["new_k"], s["new_v"], counts=s["counts"])
    else:
        lengths = _plain_append(s["k"], s["v"], s["positions"], s["weights"], s["table"], s["lengths"], s["new_k"], s["new_v"], s["counts"])
    return s["k"], s["v"], s["positions"], s["weights"], lengths


def _plain_append(k, v, positions, weights, table, lengths, new_k, new_v, counts):
    """A token behind its sequence's count leaves what is at its place."""
    B, Hk, T, _ = new_k.shape
    page, dev = k.shape[2], k.device
    slot = lengths.long()[:, None] + torch.arange(T, device=dev)
    flat = (table.long().gather(1, slot // page)[:, None] * Hk + torch.arange(Hk, device=dev)[None, :, None]) * page + (slot % page)[:, None]
    written = (torch.arange(T, device=dev) < counts[:, None])[:, None].expand(B, Hk, T)
    for pool, new in ((k.view(-1, DIM), new_k), (v.view(-1, DIM), new_v), (positions.view(-1), slot[:, None].expand(B, Hk, T).to(torch.int32)),
                      (weights.view(-1), torch.zeros((B, Hk, T), device=dev))):
        pool[flat] = torch.where(written[..., None] if pool.dim() == 2 else written, new, pool[flat])
    return lengths + counts


def _run_evict(s):
    case = s["case"]
    # eviction brings weights and positions along with the rows it moves: both as they were, so that every pass is the same
    torch._foreach_copy_([s["weights"], s["positions"]], [s["weights_before"], s["positions_before"]])
    if own:
        import flex_block_attn_amd as fba

        cache = fba.PagedCache(s["k"], s["v"], positions=s["positions"], weights=s["weights"])
        lengths = fba.cache_evict(cache, s["table"], s["lengths"], case["budget"], recent=case["recent"], sinks=case["sinks"])
    else:
        lengths = _plain_evict(s["k"], s["v"], s["positions"], s["weights"], s["table"], s["lengths"], case["budget"], case["recent"], case["sinks"])
    return s["k"], s["v"], s["positions"], s["weights"], lengths


def _plain_evict(k, v, positions, weights, table, lengths, budget, recent, sinks):
    B, Hk, page, dev = table.shape[0], k.shape[1], k.shape[2], k.device
    slot = torch.arange(table.shape[1] * page, device=dev)
    flat = (table.long()[:, slot // page][:, None] * Hk + torch.arange(Hk, device=dev)[None, :, None]) * page + slot % page  # (B, Hk, slots)
    there = slot < lengths.long()[:, None, None]
    w, at = weights.view(-1)[flat], positions.view(-1)[flat].long()
    newest = torch.where(there, at, torch.full_like(at, -1)).amax(-1, keepdim=True)
    held = (at < sinks) | (at > newest - recent)
    rank = torch.where(there, torch.where(held, torch.full_like(w, math.inf), w), torch.full_like(w, -math.inf))
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(there.expand_as(flat)).scatter_(-1, order[..., :budget], True) & there
    full = (lengths > budget)[:, None, None]
    free = full & there & ~kept & (slot < budget)
    late = full & kept & (slot >= budget)
    most = min(budget, slot.numel() - budget)
    if most > 0:
        to = (~free).to(torch.int8).sort(dim=-1, stable=True).indices[..., :most]  # freed slots first, in order
        source = (~late).to(torch.int8).sort(dim=-1, stable=True).indices[..., :most]
        moved = torch.arange(most, device=dev) < free.sum(-1, keepdim=True)
        to = flat.gather(-1, to)
        source = torch.where(moved, flat.gather(-1, source), to)  # behind the last one a slot keeps what it has
        for pool in (k.view(-1, DIM), v.view(-1, DIM), positions.view(-1), weights.view(-1)):
            pool[to] = pool[source]
    return lengths.clamp_max(budget)


# ---------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"window": _exact_window, "attend": _exact_attend, "append": _exact_append, "evict": _exact_evict}[case["op"]](s)


def _exact_window(s):
    """Sequence by sequence and head by head, some rows at a time against the stretch of keys that they can see and the sinks."""
    case = s["case"]
    turn = case["layout"] == "bshd"
    q, k, v, do = ((t.detach().transpose(1, 2) if turn else t.detach()) for t in (s["q"], s["k"], s["v"], s["do"]))
    G = case["heads"] // case["kv_heads"]
    W, n_sinks, causal = case["window"], case["sinks"], case["causal"]
    o, dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, q, k, v))
    for b, end in enumerate(_lengths(case)):
        rows = end if case["ragged"] else case["q_len"]
        shift = end - rows
        step = max(256, 2048 * 2048 // (W + 1024))
        for r0 in range(0, rows, step):
            r1 = min(rows, r0 + step)
            low = max(0, r0 + shift - W + 1)
            high = min(end, r1 + shift if causal else r1 + shift + W - 1)
            if high <= 0:
                continue
            j = torch.cat([torch.arange(min(n_sinks, low, end)), torch.arange(low, high), torch.arange(high, max(high, 0 if causal else min(n_sinks, end)))]).cuda()
            p = torch.arange(r0, r1, device="cuda")[:, None] + shift
            near = (p - j < W) if causal else ((p - j).abs() < W)
            hidden = ~(near | (j < n_sinks)) | ((j > p) if causal else torch.zeros_like(near))
            none = hidden.all(-1, keepdim=True)
            for h in range(case["kv_heads"]):
                kd, vd = k[b, h, j].double(), v[b, h, j].double()
                for g in range(h * G, (h + 1) * G):
                    qd = q[b, g, r0:r1].double()
                    logits = (qd @ kd.T * SCALE).masked_fill_(hidden, -math.inf)
                    weight = torch.softmax(logits, -1).masked_fill_(none, 0.0)
                    o[b, g, r0:r1] = weight @ vd
                    if case["step"]:
                        od = do[b, g, r0:r1].double()
                        dv[b, h].index_add_(0, j, weight.T @ od)
                        back = od @ vd.T
                        back = weight * (back - (weight * back).sum(-1, keepdim=True)) * SCALE
                        dq[b, g, r0:r1] = back @ kd
                        dk[b, h].index_add_(0, j, back.T @ qd)
    if not case["step"]:
        return o
    return (o, *(t.transpose(1, 2) if turn else t for t in (dq, dk, dv)))


def _exact_attend(s):
    case = s["case"]
    q, page = s["q"].double(), case["page"]
    G = case["heads"] // case["kv_heads"]
    o = torch.zeros_like(q)
    weights = s["weights"].double() if case["accumulate"] else None
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        slots = [i for i in range(n) if not case["window"] or i >= n - case["window"] or i < case["sinks"]]
        slots = torch.tensor(slots, device="cuda")
        pages, at = s["table"][b].long()[slots // page], slots % page
        for h in range(case["kv_heads"]):
            kd, vd = s["k"][pages, h, at].double(), s["v"][pages, h, at].double()
            weight = torch.softmax(q[b, h * G:(h + 1) * G, 0] @ kd.T * SCALE, -1)
            o[b, h * G:(h + 1) * G, 0] = weight @ vd
            if weights is not None:
                weights[pages, h, at] += weight.sum(0)
    return o if weights is None else (o, weights)


def _exact_append(s):
    """Row copies: what comes out has to be the same, and nothing is computed but whole numbers."""
    return None


def _exact_evict(s):
    """Row copies, as above."""
    return None
