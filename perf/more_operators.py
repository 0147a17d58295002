"""Positions by rotation and a paged cache in 4 bits, as cases that can be timed and compared: rotary positions with several axes for video and text, appending to
a paged cache with the rotation on the way, a cache that holds a row of 128 in 64 bytes and 4 scales, its rows read back, and the attention of single tokens over it.

`own` false: the operators in plain form, elementary torch operations in 32 bits, in 64 for angles and next to the borders of 4 bits.  `own` true: this package's entry
points.

A case is a dict of plain values.  op "rotary": batch, heads, kv_heads, len, layout ("bhsd", or "bshd" as a projection leaves it), step (forward and backward), dtype and
the rotation: dims (columns of every axis, as a text), theta, interleaved.  op "append" (16 bits) and "held" (4 bits, then read back): batch, heads of q (0: none),
kv_heads, len, new, page, ragged, dtype, the rotation (dims "": none).  op "read": a 16-bit cache read back.  op "attend": batch, heads, kv_heads, len, page, ragged, window,
sinks, accumulate, dtype, over 4 bits.

The 4 bits: a row is four groups of 32, each with an exponent e, held as the byte e + 127 (255: something in it is no number); a value is 0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign,
times 2^e, to the nearest, ties to the even code; e is the largest value's exponent less 2, and one more from 1.75 of its binade on.  Byte j of a row has values 2j (low) and 2j + 1.
"""
import math

import torch

own = False

DIM = 128
SCALE = 1 / math.sqrt(DIM)
GOLDEN = 0.6180339887498949
STEPS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LIMIT = {"bfloat16": 125, "float16": 13}  # of the exponent, so that every value is a normal number of the type


def _rotary(name, heads, kv_heads, length, dims, *, batch=1, layout="bhsd", step=False, theta=10000.0, interleaved=True, dtype="bfloat16"):
    case = {"op": "rotary", "batch": batch, "heads": heads, "kv_heads": kv_heads, "len": length, "dims": dims, "theta": theta, "interleaved": interleaved, "layout": layout,
            "step": step, "dtype": dtype}
    return dict(case, name=name) if name else case


def _append(name, batch, heads, kv_heads, length, new, page, dims, *, held=False, ragged=False, theta=10000.0, interleaved=False, dtype="bfloat16"):
    case = {"op": "held" if held else "append", "batch": batch, "heads": heads, "kv_heads": kv_heads, "len": length, "new": new, "page": page, "dims": dims, "theta": theta,
            "interleaved": interleaved, "ragged": ragged, "dtype": dtype}
    return dict(case, name=name) if name else case


def _read(name, batch, kv_heads, length, page, *, ragged=False, dtype="bfloat16"):
    case = {"op": "read", "batch": batch, "kv_heads": kv_heads, "len": length, "page": page, "ragged": ragged, "dtype": dtype}
    return dict(case, name=name) if name else case


def _attend(name, batch, heads, kv_heads, length, page, *, ragged=False, window=0, sinks=0, accumulate=False, dtype="bfloat16"):
    case = {"op": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "len": length, "page": page, "ragged": ragged, "window": window, "sinks": sinks,
            "accumulate": accumulate, "dtype": dtype}
    return dict(case, name=name) if name else case


def listed():
    return [
        # A short clip through one head, without gradients: the launch is all of it.
        _rotary("rotary_small", 1, 1, 768, "16,56,56", dtype="float16"),
        # Training on text of an odd length, grouped heads, in the layout of a projection.
        _rotary("rotary_text_step", 8, 2, 3136, "128", batch=2, layout="bshd", step=True, interleaved=False, dtype="float16"),
        # Training of a video layer: time, height and width of every token of a latent grid.
        _rotary("rotary_video_step", 24, 24, 30720, "16,56,56", step=True),
        # The longest clip, forward.
        _rotary("rotary_video_long", 24, 24, 115200, "16,56,56"),
        # The new tokens of a serving batch: q and k rotated, k and v into the cache.
        _append("append_token", 64, 32, 8, 4096, 1, 16, "128", ragged=True),
        # Two long prompts of video tokens.
        _append("append_prompt", 2, 24, 6, 0, 30720, 64, "16,56,56", interleaved=True),
        # The next chunk of several short prompts goes into 4 bits, and all of them are read back for its attention.
        _append("held_chunk", 8, 0, 4, 1000, 200, 32, "64", held=True, ragged=True, dtype="float16"),
        # Two long prompts into 4 bits.
        _append("held_prompt", 2, 0, 6, 0, 30720, 64, "128", held=True),
        # Prefixes of prompts of several lengths read back from 16 bits.
        _read("read_prefix", 4, 8, 16384, 64, ragged=True, dtype="float16"),
        # One user's next token over a short cache: latency.
        _attend("attend_small", 1, 8, 8, 768, 16),
        # A serving batch in the middle of its answers: lengths between nothing and the longest; every slot's weight is added up.
        _attend("attend_weights", 32, 24, 6, 16384, 64, ragged=True, accumulate=True, dtype="float16"),
        # Long streams, all of them visible.
        _attend("attend_long", 8, 16, 4, 115200, 128),
    ]


def _log_uniform(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def _draw_heads(rng, most):
    group = rng.choice([1, 1, 2, 3, 4, 8])
    kv_heads = max(1, round(_log_uniform(rng, 1, max(1.01, most / group))))
    return kv_heads * group, kv_heads


def _draw_any(rng):
    op = rng.choice(["rotary", "rotary", "append", "append", "held", "read", "attend", "attend", "attend"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    ragged = rng.random() < 0.5
    heads, kv_heads = _draw_heads(rng, 24)
    page = rng.choice([16, 32, 64, 128, 256])
    turn = dict(theta=rng.choice([100.0, 10000.0, 1e6]), interleaved=rng.random() < 0.5)
    dims = rng.choice(["128", "64", "32", "16,56,56", "44,42,42", "64,64", "32,16,16", "96"])
    if op == "rotary":
        return _rotary("", heads, kv_heads, round(_log_uniform(rng, 100, 120000)), dims, batch=rng.choice([1, 1, 2, 3]), layout=rng.choice(["bhsd", "bshd"]),
                       step=rng.random() < 0.5, dtype=dtype, **turn)
    batch = max(1, round(_log_uniform(rng, 1, 64)))
    length = round(_log_uniform(rng, 256, 100000))
    if op == "read":
        return _read("", batch, kv_heads, length, page, ragged=ragged, dtype=dtype)
    if op == "attend":
        accumulate = rng.random() < 0.4
        windowed = not accumulate and rng.random() < 0.4
        return _attend("", batch, heads, kv_heads, length, page, ragged=ragged, window=round(_log_uniform(rng, 16, length)) if windowed else 0,
                       sinks=rng.choice([0, 4, 64, 100]) if windowed else 0, accumulate=accumulate, dtype=dtype)
    new = round(_log_uniform(rng, 2, 30000)) if op == "held" else rng.choice([1, 1, round(_log_uniform(rng, 2, 30000))])
    return _append("", batch, rng.choice([0, heads]) if op == "append" else 0, kv_heads, rng.choice([0, min(length, 20000)]), new, page,
                   rng.choice([dims, dims, ""]) if op == "held" else dims, held=op == "held", ragged=ragged, dtype=dtype, **turn)


def draw(rng):
    most = {op: max(work(c)["bytes"] for c in listed() if c["op"] == op) for op in ("rotary", "append", "held", "read", "attend")}
    while True:
        case = _draw_any(rng)
        if work(case)["bytes"] <= most[case["op"]] and case["batch"] * case.get("kv_heads", 1) * (case["len"] + case.get("new", 0)) <= 8 * 4 * 115200:
            return case


# ---------------------------------------------------------------------------------------------------------------------
# what a case is made of
# ---------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Lengths of the batch's sequences: of a ragged one the longest, and others down to nothing between."""
    n, most = case["batch"], case["len"]
    if not case["ragged"]:
        return [most] * n
    return [most] + [int(most * ((i * GOLDEN + 0.3) % 1)) for i in range(1, n)]


def _counts(case):
    """New tokens of every sequence."""
    if not case["ragged"] or case["new"] == 1:
        return [case["new"]] * case["batch"]
    return [case["new"]] + [int(case["new"] * ((i * GOLDEN + 0.7) % 1)) for i in range(1, case["batch"])]


def _dims(case):
    return [int(d) for d in case["dims"].split(",")] if case["dims"] else []


def work(case):
    h, hk = case.get("heads", 0), case["kv_heads"]
    if case["op"] == "rotary":
        rows = case["batch"] * case["len"] * (h + hk) * (2 if case["step"] else 1)
        return {"bytes": rows * 4 * DIM + 4 * len(_dims(case)) * case["batch"] * case["len"], "flops": 3 * rows * sum(_dims(case))}
    if case["op"] in ("append", "held"):
        new = sum(_counts(case))
        turned = 3 * sum(_dims(case)) * new
        if case["op"] == "append":
            return {"bytes": new * (hk * 8 * DIM + h * 4 * DIM), "flops": turned * (h + hk)}
        rows = (sum(_lengths(case)) + new) * hk
        return {"bytes": new * hk * (4 * DIM + 136) + rows * (136 + 4 * DIM), "flops": turned * hk}
    if case["op"] == "read":
        return {"bytes": sum(_lengths(case)) * hk * 4 * DIM + case["batch"] * case["len"] * hk * 4 * DIM, "flops": 0}
    seen = sum(n if not case["window"] else min(n, case["window"]) + min(case["sinks"], max(0, n - case["window"])) for n in _lengths(case))
    return {"bytes": seen * hk * (136 + (8 if case["accumulate"] else 0)) + 4 * DIM * case["batch"] * h, "flops": 4 * DIM * seen * h}


def _frequencies(dims, theta):
    """Radians a step of every pair, axis by axis, and the axes."""
    return [theta ** (-2 * j / d) for d in dims for j in range(d // 2)], [x for x, d in enumerate(dims) for _ in range(d // 2)]


def _coordinates(shape, axes, first):
    """Where tokens stand: on one axis behind `first`; on several in a grid, the last axis fastest, that starts there in time."""
    token = torch.arange(shape[-1], device="cuda").expand(shape)
    if axes == 1:
        return (token + first)[..., None].to(torch.int32)
    width = max(1, int((shape[-1] / 30) ** (1 / (axes - 1)))) if axes > 2 else max(1, int(shape[-1] ** 0.5))
    at = [token // width**i % width for i in range(axes - 1)]
    return torch.stack([token // width ** (axes - 1) + first, *reversed(at)], -1).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    batch, kv_heads = case["batch"], case["kv_heads"]

    def normal(*shape, size=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * size).to(dtype)

    state = dict(case=case)
    if case.get("dims"):  # the rotation as a program keeps it: turns a step times 2^64, and axes
        frequency, axis = _frequencies(_dims(case), case["theta"])
        turns = [(int(f / (2 * math.pi) * 2**64) + 2**63) % 2**64 - 2**63 for f in frequency]
        state.update(frequency=torch.tensor(frequency, dtype=torch.float64, device="cuda"), axis=torch.tensor(axis, dtype=torch.int32, device="cuda"),
                     turns=torch.tensor(turns, dtype=torch.int64, device="cuda"))
    if case["op"] == "rotary":
        def tensor(heads):
            return normal(batch, case["len"], heads, DIM) if case["layout"] == "bshd" else normal(batch, heads, case["len"], DIM)

        q, k = tensor(case["heads"]), tensor(kv_heads)
        for t in (q, k):
            t.requires_grad_(case["step"])
        # a batch's clips and texts start anywhere in their streams
        first = torch.randint(0, 100000, (batch, 1), generator=g, device="cuda")
        return dict(state, q=q, k=k, dq=tensor(case["heads"]), dk=tensor(kv_heads), coordinates=_coordinates((batch, case["len"]), len(_dims(case)), first))
    page = case["page"]
    lengths, new = _lengths(case), case.get("new", 0)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    per = -(-(max(lengths) + new) // page)  # pages of a sequence
    pages = batch * per + 3
    pool = (pages, kv_heads, page)
    state["table"] = torch.randperm(pages, generator=g, device="cuda")[: batch * per].to(torch.int32).reshape(batch, per)
    if case["op"] in ("append", "read"):
        state["k"], state["v"] = normal(*pool, DIM), normal(*pool, DIM)
    else:
        for name in ("k", "v"):
            # keys with some channels that are larger than others, as trained layers have them
            size = 1.0 + 3.0 * (torch.rand(DIM, generator=g, device="cuda") < 0.06) if name == "k" else 1.0
            state[name], state[name + "_scales"] = _to_4_bits(torch.randn((*pool, DIM), generator=g, device="cuda") * size, LIMIT[case["dtype"]])
    if case["op"] == "read":
        return state
    if case["op"] == "attend":
        if case["accumulate"]:
            state["weights"] = torch.rand(pool, generator=g, device="cuda") * 4
        return dict(state, q=normal(batch, case["heads"], 1, DIM, size=2.0))
    state["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")
    if len(_dims(case)) > 1:
        state["coordinates"] = _coordinates((batch, new), len(_dims(case)), state["lengths"][:, None])
    if case["heads"]:
        state["q"] = normal(batch, case["heads"], new, DIM)
    return dict(state, new_k=normal(batch, kv_heads, new, DIM), new_v=normal(batch, kv_heads, new, DIM))


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    return {"rotary": _run_rotary, "append": _run_append, "held": _run_held, "read": _run_read, "attend": _run_attend}[state["case"]["op"]](state)


def _own_rotary(s):
    import flex_block_attn_amd as fba

    return fba.Rotary(s["turns"], s["axis"], len(_dims(s["case"])), s["case"]["interleaved"])


def _own_cache(s):
    import flex_block_attn_amd as fba

    if "k_scales" not in s:
        return fba.PagedCache(s["k"], s["v"])
    return fba.PagedCache4(s["k"], s["v"], s["k_scales"], s["v_scales"], getattr(torch, s["case"]["dtype"]), weights=s.get("weights"))


def _rotated(x, coordinates, s, double=False):
    """x (batch, heads, tokens, DIM), coordinates (batch, tokens, axes) -> rotated, in 32 bits or in 64"""
    angle = (coordinates.double()[..., s["axis"].long()] * s["frequency"])[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    x = x.double() if double else x.float()
    cos, sin = cos.to(x.dtype), sin.to(x.dtype)
    n = angle.shape[-1]
    if s["case"]["interleaved"]:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _run_rotary(s):
    case = s["case"]
    turn = (lambda t: t.transpose(1, 2)) if case["layout"] == "bshd" else (lambda t: t)
    with torch.set_grad_enabled(case["step"]):
        if own:
            import flex_block_attn_amd as fba

            q, k = fba.rotary_func(turn(s["q"]), turn(s["k"]), _own_rotary(s), coordinates=s["coordinates"])
        else:
            q, k = (_rotated(turn(x), s["coordinates"], s).to(x.dtype) for x in (s["q"], s["k"]))
    if not case["step"]:
        return q, k
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (turn(s["dq"]), turn(s["dk"]))))


def _slots(s):
    """Slots of the new tokens, and what they stand at."""
    slot = s["lengths"].long()[:, None] + torch.arange(s["case"]["new"], device="cuda")
    return slot, s["coordinates"] if "coordinates" in s else slot[..., None].expand(-1, -1, max(1, len(_dims(s["case"]))))


def _rows(s, slot):
    """Numbers of slots' rows in the pool: (batch, kv_heads, slots)."""
    page, kv_heads = s["case"]["page"], s["case"]["kv_heads"]
    return (s["table"].long().gather(1, slot // page)[:, None] * kv_heads + torch.arange(kv_heads, device="cuda")[:, None]) * page + (slot % page)[:, None]


def _write(pool, rows, written, values):
    """Rows of a pool; a token behind its sequence's count leaves what is at its place."""
    pool = pool.view(-1, pool.shape[-1])
    pool[rows] = torch.where(written[:, None, :, None], values, pool[rows])


def _run_append(s):
    if own:
        import flex_block_attn_amd as fba

        lengths, q = fba.cache_append_rotary(_own_cache(s), s["table"], s["lengths"], s["new_k"], s["new_v"], _own_rotary(s), q=s.get("q"), counts=s["counts"],
                                             coordinates=s.get("coordinates"))
    else:
        slot, at = _slots(s)
        rows, written = _rows(s, slot), torch.arange(s["case"]["new"], device="cuda") < s["counts"][:, None]
        _write(s["k"], rows, written, _rotated(s["new_k"], at, s).to(s["k"].dtype))
        _write(s["v"], rows, written, s["new_v"])
        q = _rotated(s["q"], at, s).to(s["q"].dtype) if "q" in s else None
        lengths = s["lengths"] + s["counts"]
    return s["k"], s["v"], lengths, q


def _power(e):
    """2^e, exactly: int32 between -126 and 127 -> float32"""
    return ((e.int() + 127) << 23).view(torch.float32)


def _to_4_bits(x, limit):
    """x (..., DIM) -> codes (..., DIM / 2), scales (..., DIM / 32), bytes both"""
    x = x.unflatten(-1, (DIM // 32, 32))
    most = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(most)
    e = torch.where(most > 0, exponent - 3 + (mantissa >= 0.875).int(), torch.full_like(exponent, -limit)).clamp(-limit, limit)
    t = x * _power(-e)[..., None]
    a = t.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    code = (code + 8 * (t < 0).to(torch.uint8)).flatten(-2)
    scales = torch.where(most.isfinite(), e + 127, torch.full_like(e, 255))
    return code[..., 0::2] + code[..., 1::2] * 16, scales.to(torch.uint8)


def _from_4_bits(codes, scales):
    """The values, in 32 bits."""
    step = torch.tensor(STEPS, device="cuda")
    step = torch.cat([step, -step])
    values = step[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    e = scales.int() - 127
    size = torch.where(e == 128, torch.full(e.shape, math.nan, device="cuda"), _power(e.clamp_max(127)))
    return (values.unflatten(-1, (DIM // 32, 32)) * size[..., None]).flatten(-2)


def _values(s, name, rows):
    """Rows of the pool as values in 32 bits."""
    pool = s[name].view(-1, s[name].shape[-1])[rows]
    return pool.float() if name + "_scales" not in s else _from_4_bits(pool, s[name + "_scales"].view(-1, DIM // 32)[rows])


def _read_back(s, lengths, slots):
    """Rows of all sequences, dense, zeros behind their lengths."""
    slot = torch.arange(slots, device="cuda")
    there = (slot < lengths[:, None])[:, None, :, None]
    rows = _rows(s, slot.expand(s["case"]["batch"], -1))
    return [torch.where(there, _values(s, name, rows), torch.zeros((), device="cuda")).to(getattr(torch, s["case"]["dtype"])) for name in ("k", "v")]


def _run_held(s):
    case = s["case"]
    slots = case["len"] + case["new"]
    if own:
        import flex_block_attn_amd as fba

        cache = _own_cache(s)
        if case["dims"]:
            lengths, _ = fba.cache_append_rotary(cache, s["table"], s["lengths"], s["new_k"], s["new_v"], _own_rotary(s), counts=s["counts"], coordinates=s.get("coordinates"))
        else:
            lengths = fba.cache_append(cache, s["table"], s["lengths"], s["new_k"], s["new_v"], counts=s["counts"])
        return (lengths, *fba.cache_read(cache, s["table"], lengths, slots))
    slot, at = _slots(s)
    rows, written = _rows(s, slot), torch.arange(case["new"], device="cuda") < s["counts"][:, None]
    k = _rotated(s["new_k"], at, s, double=True) if case["dims"] else s["new_k"].double()
    for name, x in (("k", k), ("v", s["new_v"].double())):
        codes, scales = _to_4_bits(x, LIMIT[case["dtype"]])
        _write(s[name], rows, written, codes)
        _write(s[name + "_scales"], rows, written, scales)
    lengths = s["lengths"] + s["counts"]
    return (lengths, *_read_back(s, lengths, slots))


def _run_read(s):
    if own:
        import flex_block_attn_amd as fba

        return fba.cache_read(_own_cache(s), s["table"], s["lengths"], s["case"]["len"])
    return _read_back(s, s["lengths"], s["case"]["len"])


def _run_attend(s):
    case = s["case"]
    window = case["window"] or None
    if own:
        import flex_block_attn_amd as fba

        o = fba.cache_attn_func(s["q"], _own_cache(s), s["table"], s["lengths"], window=window, sinks=case["sinks"], accumulate=case["accumulate"])
    else:
        o = _plain_attend(s, window)
    return (o, s["weights"]) if case["accumulate"] else o


def _plain_attend(s, window):
    case, q = s["case"], s["q"]
    B, H, Hk, most, sinks = case["batch"], case["heads"], case["kv_heads"], case["len"], case["sinks"]
    n = s["lengths"].long()[:, None]
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
    rows = _rows(s, slot)
    kf, vf = _values(s, "k", rows), _values(s, "v", rows)  # (B, Hk, slots, DIM)
    sc = (q.float().reshape(B, Hk, H // Hk, DIM) @ kf.transpose(-1, -2).contiguous()) * SCALE
    sc = sc.masked_fill(~seen[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    if "weights" in s:  # slots that are not seen add nothing
        s["weights"].view(-1).index_add_(0, rows.reshape(-1), p.sum(2).reshape(-1))
    return (p @ vf).reshape(B, H, 1, DIM).to(q.dtype)


# ---------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "held": _exact_held, "read": _exact_read, "attend": _exact_attend}[case["op"]](s)


def _turned(x, at, case, back=False):
    """Rows (tokens, DIM) that stand at (tokens, axes): every pair a complex number, times exp(i angle)."""
    x = x.double().clone()
    place = 0
    pairs = sum(_dims(case)) // 2
    for axis, d in enumerate(_dims(case)):
        j = torch.arange(d // 2, dtype=torch.float64, device="cuda")
        angle = at[:, axis, None].double() * case["theta"] ** (-2 * j / d)
        turn = torch.polar(torch.ones_like(angle), -angle if back else angle)
        i = place + torch.arange(d // 2, device="cuda")
        re, im = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + pairs)
        z = torch.complex(x[:, re], x[:, im]) * turn
        x[:, re], x[:, im] = z.real, z.imag
        place += d // 2
    return x


def _exact_rotary(s):
    """Head by head."""
    case = s["case"]
    found = []
    for name, back in (("q", False), ("k", False), ("dq", True), ("dk", True)):
        if back and not case["step"]:
            continue
        x = s[name].detach()
        heads_last = case["layout"] == "bshd"
        out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            for h in range(x.shape[2 if heads_last else 1]):
                at = (b, slice(None), h) if heads_last else (b, h)
                out[at] = _turned(x[at], s["coordinates"][b], case, back)
        found.append(out.transpose(1, 2) if heads_last and not back else out)
    return tuple(found)


def _places(s, b, n):
    slot = torch.arange(n, device="cuda")
    return s["table"][b].long()[slot // s["case"]["page"]], slot % s["case"]["page"]


def _stand(s, b, n, count):
    if "coordinates" in s:
        return s["coordinates"][b, :count]
    return torch.arange(n, n + count, device="cuda")[:, None]


def _exact_append(s):
    case = s["case"]
    k, v = s["k"].double(), s["v"].double()
    q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda") if case["heads"] else None
    for b, (n, count) in enumerate(zip(_lengths(case), _counts(case))):
        pages, at = (t[n:] for t in _places(s, b, n + count))
        for h in range(case["kv_heads"]):
            k[pages, h, at] = _turned(s["new_k"][b, h, :count], _stand(s, b, n, count), case)
            v[pages, h, at] = s["new_v"][b, h, :count].double()
        for h in range(case["heads"]):  # what is behind a count is turned too
            q[b, h] = _turned(s["q"][b, h], _stand(s, b, n, case["new"]), case)
    return k, v, None, q


def _held(x, limit):
    """Rows (n, DIM) in 64 bits -> the values that 4 bits hold of them: the nearer one of the two neighbours among a group's fifteen, of two alike the one with the even code."""
    groups = x.reshape(-1, 32)
    most = groups.abs().amax(1)
    e = torch.full_like(most, -float(limit))
    some = (most > 0) & torch.isfinite(most)
    binade = torch.floor(torch.log2(most[some]))
    binade = torch.where(torch.exp2(binade) > most[some], binade - 1, binade)
    binade = torch.where(torch.exp2(binade + 1) <= most[some], binade + 1, binade)
    e[some] = binade - 2 + (most[some] >= 1.75 * torch.exp2(binade)).double()
    unit = torch.exp2(e.clamp(-limit, limit))[:, None]
    steps = torch.tensor(STEPS, dtype=torch.float64, device="cuda")
    size = (groups.abs() / unit).contiguous()
    above = torch.bucketize(size, steps).clamp(1, 7)
    down, up = size - steps[above - 1], steps[above] - size
    code = torch.where((down < up) | ((down == up) & (above % 2 == 1)), above - 1, above)
    code = torch.where(size > 6, torch.full_like(code, 7), code)
    values = torch.where(groups < 0, -steps[code], steps[code]) * unit
    return torch.where(torch.isfinite(most)[:, None], values, torch.full_like(values, math.nan)).reshape(x.shape)


def _exact_values(s, name, b, h, n):
    """A head's first n rows of a sequence in 64 bits."""
    pages, at = _places(s, b, n)
    rows = s[name][pages, h, at]
    if name + "_scales" not in s:
        return rows.double()
    codes = torch.empty((n, DIM), dtype=torch.long, device="cuda")
    codes[:, 0::2], codes[:, 1::2] = rows.long() % 16, rows.long() // 16
    steps = torch.tensor([*STEPS, *(-x for x in STEPS)], dtype=torch.float64, device="cuda")
    return steps[codes] * torch.exp2(s[name + "_scales"][pages, h, at].double() - 127).repeat_interleave(32, 1)


def _exact_held(s):
    case = s["case"]
    out = [torch.zeros((case["batch"], case["kv_heads"], case["len"] + case["new"], DIM), dtype=torch.float64, device="cuda") for _ in range(2)]
    limit = LIMIT[case["dtype"]]
    for b, (n, count) in enumerate(zip(_lengths(case), _counts(case))):
        for h in range(case["kv_heads"]):
            for t, name in zip(out, ("k", "v")):
                t[b, h, :n] = _exact_values(s, name, b, h, n)
                new = s["new_" + name][b, h, :count].double()
                t[b, h, n:n + count] = _held(_turned(new, _stand(s, b, n, count), case) if name == "k" and case["dims"] else new, limit)
    return (None, *out)


def _exact_read(s):
    case = s["case"]
    out = [torch.zeros((case["batch"], case["kv_heads"], case["len"], DIM), dtype=torch.float64, device="cuda") for _ in range(2)]
    for b, n in enumerate(_lengths(case)):
        for h in range(case["kv_heads"]):
            for t, name in zip(out, ("k", "v")):
                t[b, h, :n] = _exact_values(s, name, b, h, n)
    return tuple(out)


def _exact_attend(s):
    case = s["case"]
    q = s["q"].double()
    G = case["heads"] // case["kv_heads"]
    o = torch.zeros_like(q)
    weights = s["weights"].double() if case["accumulate"] else None
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        slot = torch.arange(n, device="cuda")
        seen = (slot >= n - case["window"]) | (slot < case["sinks"]) if case["window"] else slot >= 0
        pages, at = _places(s, b, n)
        for h in range(case["kv_heads"]):
            kd, vd = _exact_values(s, "k", b, h, n), _exact_values(s, "v", b, h, n)
            weight = torch.softmax((q[b, h * G:(h + 1) * G, 0] @ kd.T * SCALE).masked_fill(~seen, -math.inf), -1)
            o[b, h * G:(h + 1) * G, 0] = weight @ vd
            if weights is not None:
                weights[pages, h, at] += weight.sum(0)
    return o if weights is None else (o, weights)
