"""The operators of a cache held in 8 bits, measured case by case.

A cache of keys and values may be held as 8-bit codes instead of the compute
type: a row (one position's key or value of one head) is ``head_dim`` codes and
one float32 scale,

    scale = max |x| / limit,   code = round(x / scale),   value = code * scale

(the scale rounded to float32, the code nearest to the exact quotient by it, of
two equally near the even one), with e4m3 codes (``"fp8"``, limit 448) or whole
numbers (``"int8"``, limit 127).
Three operators, as a step of the engine calls them:

* ``store``: the norm and rotation of a step's queries and keys, the keys and
  values written as codes, and the step's pages read back as values;
* ``read``: pages read back into the compute type, as the attention of a
  prompt's portion wants the context behind it;
* ``attend``: attention of one new token a request over the paged codes.

``own`` False computes them in elementary torch operations, True by the calls a
user makes of the framework.
"""
from __future__ import annotations

import math

import torch

own = False

LIMITS = {"fp8": 448.0, "int8": 127.0}
CODES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the cache traffic of a decode step of 8 requests at the 0.6B layer sizes: latency counts
        dict(name="store_decode_8", op="store", codes="fp8", dtype="bf16", tokens=8, requests=8, start=700, heads=16, kv_heads=8,
             head_dim=128, page=16, norm=True, rotate="half"),
        # ... of a 2,048-token prompt at the 8B layer sizes
        dict(name="store_prompt_2048", op="store", codes="fp8", dtype="bf16", tokens=2048, requests=1, start=0, heads=32,
             kv_heads=8, head_dim=128, page=16, norm=True, rotate="half"),
        # ... of five portions that begin inside a page, heads of 64 with neighbouring values turned, no norm
        dict(name="store_portions_int8", op="store", codes="int8", dtype="bf16", tokens=1733, requests=5, start=37, heads=15,
             kv_heads=5, head_dim=64, page=32, norm=False, rotate="pairs"),
        # ... of the float32 path without a position encoding: keys and values as they are projected
        dict(name="store_float32", op="store", codes="int8", dtype="f32", tokens=917, requests=3, start=5, heads=4, kv_heads=4,
             head_dim=128, page=16, norm=False, rotate="none"),
        # the context behind a portion of one request
        dict(name="read_2k", op="read", codes="fp8", dtype="bf16", requests=1, longest=2048, kv_heads=8, head_dim=128, page=16,
             window=0),
        # contexts of four requests, the longest of 32,000 positions
        dict(name="read_32k_ragged", op="read", codes="int8", dtype="bf16", requests=4, longest=32000, kv_heads=8, head_dim=128,
             page=64, window=0),
        # a decode step of one request, short context: latency
        dict(name="attend_1x500", op="attend", codes="fp8", dtype="bf16", requests=1, padding=0, longest=500, ragged=False,
             heads=16, kv_heads=8, head_dim=128, page=16, window=0, softcap=0.0, sink=False),
        # the decode step the framework's benchmark times: 8 requests over 2,048 positions
        dict(name="attend_8x2048", op="attend", codes="fp8", dtype="bf16", requests=8, padding=0, longest=2048, ragged=False,
             heads=16, kv_heads=8, head_dim=128, page=16, window=0, softcap=0.0, sink=False),
        # continuous batching: 64 requests of many lengths at the 8B layer sizes, a captured step's padding rows behind them
        dict(name="attend_61_ragged", op="attend", codes="int8", dtype="bf16", requests=61, padding=3, longest=8192, ragged=True,
             heads=32, kv_heads=8, head_dim=128, page=16, window=0, softcap=0.0, sink=False),
        # long contexts
        dict(name="attend_8x32000", op="attend", codes="fp8", dtype="bf16", requests=8, padding=0, longest=32000, ragged=False,
             heads=32, kv_heads=8, head_dim=128, page=16, window=0, softcap=0.0, sink=False),
        # heads of 64, seven to a key/value head, a window, a cap on the scores and a sink
        dict(name="attend_window_64", op="attend", codes="int8", dtype="bf16", requests=13, padding=0, longest=9001, ragged=True,
             heads=14, kv_heads=2, head_dim=64, page=32, window=1500, softcap=30.0, sink=True),
        # the float32 path
        dict(name="attend_float32", op="attend", codes="fp8", dtype="f32", requests=3, padding=0, longest=5003, ragged=True,
             heads=16, kv_heads=4, head_dim=128, page=16, window=0, softcap=0.0, sink=False),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["store", "read", "attend", "attend"])
    case = dict(op=op, codes=rng.choice(["fp8", "int8"]), dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]),
                kv_heads=rng.choice([1, 2, 3, 4, 8]), head_dim=rng.choice([64, 128]), page=rng.choice([8, 16, 32, 64]))
    width = case["kv_heads"] * case["head_dim"]
    if op == "store":
        tokens = spread(1, 4096 * 1024 // max(width, 1024))
        plain = case["dtype"] == "f32"
        case.update(tokens=tokens, requests=min(tokens, spread(1, 16)), start=rng.choice([0, rng.randrange(1, 3000)]),
                    heads=case["kv_heads"] * rng.choice([1, 2, 3, 4]), norm=False if plain else rng.random() < 0.7,
                    rotate="none" if plain else rng.choice(["half", "half", "pairs", "part"]))
        if not plain and rng.random() < 0.2:
            case["head_dim"] = 256 if width <= 512 else 128
    elif op == "read":
        longest = spread(1, 40000)
        case.update(requests=max(1, min(spread(1, 16), 80000 // longest)), longest=longest,
                    window=rng.choice([0, 0, spread(1, 4096)]))
    else:
        longest = spread(1, 40000)
        case.update(requests=max(1, min(spread(1, 64), 8 * 32000 // longest)), padding=rng.choice([0, 0, 1, 3]), longest=longest,
                    ragged=rng.random() < 0.7, heads=case["kv_heads"] * rng.choice([1, 2, 4, 5, 7, 8]),
                    window=rng.choice([0, 0, 0, spread(1, 4096)]), softcap=rng.choice([0.0, 0.0, 30.0]), sink=rng.random() < 0.3)
    return case


def _lengths(case):
    """How many positions each request holds when the operator has run."""
    if case["op"] == "store":   # portions of (nearly) equal size
        size, more = divmod(case["tokens"], case["requests"])
        return [case["start"] + size + (1 if i < more else 0) for i in range(case["requests"])]
    n, longest = case["requests"], case["longest"]
    if case["op"] == "attend" and not case["ragged"]:
        return [longest] * n
    return [max(1, longest - (i * longest) // n) for i in range(n)]


def _first_seen(case, length):
    return max(0, length - case["window"]) if case["window"] else 0


def work(case):
    element = 2 if case["dtype"] == "bf16" else 4
    kv, hd, lengths = case["kv_heads"], case["head_dim"], _lengths(case)
    row = hd + 4   # codes and scale of a key or a value
    if case["op"] == "store":
        tokens, heads = case["tokens"], case["heads"]
        skipped = case["start"] // case["page"] * case["page"]
        rows = 2 * kv * sum(n - skipped for n in lengths)
        turned = {"half": hd, "pairs": hd, "part": hd // 2, "none": 0}[case["rotate"]]
        return {"bytes": tokens * (2 * heads + 2 * kv) * hd * element + tokens * (4 * turned + 8) + tokens * 2 * kv * row
                + rows * (row + hd * element), "flops": tokens * (heads + 2 * kv) * hd * 8 + rows * hd}
    seen = sum(n - _first_seen(case, n) for n in lengths)
    if case["op"] == "read":
        return {"bytes": 2 * kv * seen * (row + hd * element), "flops": 2 * kv * seen * hd}
    return {"bytes": 2 * kv * seen * row + 2 * case["requests"] * case["heads"] * hd * element,
            "flops": 4 * case["heads"] * hd * seen}


# ------------------------------------------------------------------ the inputs
def _codes_of(x, kind):
    """Codes and scales of rows x [..., head_dim] in float32. The quotients, which may lie next to the middle between two
    codes, are taken in 64 bits."""
    scale = x.abs().amax(-1, keepdim=True) / torch.full((), LIMITS[kind], device=x.device)   # a division, not a product
    y = torch.where(scale > 0, x.double() / scale.double(), 0.0).clamp(-LIMITS[kind], LIMITS[kind])
    if kind == "fp8":
        # an e4m3 number has three bits behind the leading one, and no smaller step than 2^-9
        step = torch.ldexp(torch.ones_like(y), torch.frexp(y).exponent.clamp(min=-5) - 4)
        y = (y / step).round() * step
    return (y if kind == "fp8" else y.round()).float().to(CODES[kind]), scale.squeeze(-1)


def _pages(case, lengths, gen):
    """(how many pages the pool has, block tables [requests, width]): every request's pages anywhere in the pool."""
    page = case["page"]
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int64)
    table = torch.full((len(lengths), max(counts)), -1, dtype=torch.int32)
    at, order = 0, order.to(torch.int32).cpu()
    for i, count in enumerate(counts):
        table[i, :count] = order[at:at + count]
        at += count
    return pages, table.cuda()


def _pool(case, pages, table, lengths, gen):
    """Codes of normal values, some channels wider as in real keys; rows behind a request's last position, and pages that
    nobody holds, have what an earlier owner left there: scales that are no number."""
    shape = (pages, 2, case["kv_heads"], case["page"], case["head_dim"])
    codes = torch.empty(shape, dtype=CODES[case["codes"]], device="cuda")
    scales = torch.empty(shape[:4], dtype=torch.float32, device="cuda")
    wide = 1.0 + 3.0 * (torch.rand(case["head_dim"], generator=gen, device="cuda") > 0.95)
    step = max(1, (64 << 20) // (2 * case["kv_heads"] * case["page"] * case["head_dim"]))
    for at in range(0, pages, step):
        x = torch.randn((min(step, pages - at),) + shape[1:], generator=gen, device="cuda") * wide
        codes[at:at + step], scales[at:at + step] = _codes_of(x, case["codes"])
    held = torch.zeros((pages, case["page"]), dtype=torch.bool, device="cuda")
    at = torch.arange(table.shape[1] * case["page"], device="cuda")
    inside = at[None, :] < torch.tensor(lengths, device="cuda")[:, None]
    row = table.long().clamp(min=0)[:, at // case["page"]] * case["page"] + at % case["page"]
    held.view(-1)[row[inside]] = True
    scales.masked_fill_(~held[:, None, None, :], float("nan"))
    return codes, scales


def _to_read(table, begins, ends, page):
    """Page and row of the positions [begin, end) of every request, as a host that knows them lists them."""
    rows = torch.cat([torch.full((end - begin,), i) for i, (begin, end) in enumerate(zip(begins, ends))]).cuda()
    at = torch.cat([torch.arange(begin, end) for begin, end in zip(begins, ends)]).cuda()
    return table.long()[rows, at // page], at % page


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    lengths, dtype, page = _lengths(case), TYPES[case["dtype"]], case["page"]
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    kv, hd = case["kv_heads"], case["head_dim"]
    state = {"case": case}
    if case["op"] == "store":
        skipped = case["start"] // page * page       # what lies in pages that this step does not touch
        local = [n - skipped for n in lengths]
        pages, table = _pages(case, local, gen)
        codes, scales = _pool(case, pages, table, local, gen)
        heads, tokens = case["heads"], case["tokens"]
        qkv = torch.randn((tokens, (heads + 2 * kv) * hd), generator=gen, device="cuda").to(dtype)
        first = case["start"] - skipped
        rows = torch.cat([torch.full((n - first,), i, dtype=torch.int64) for i, n in enumerate(local)]).cuda()
        at = torch.cat([torch.arange(first, n) for n in local]).cuda()
        slots = table.long()[rows, at // page] * page + at % page
        positions = (at + skipped).to(torch.int32)
        cos = sin = None
        if case["rotate"] != "none":
            turned = hd // 2 if case["rotate"] == "part" else hd
            angle = (torch.arange(max(lengths), dtype=torch.float64, device="cuda")[:, None]
                     * 1e6 ** (-torch.arange(0, turned, 2, dtype=torch.float64, device="cuda") / turned))
            cos, sin = angle.cos().float(), angle.sin().float()
        weight = lambda: 1.0 + 0.1 * torch.randn(hd, generator=gen, device="cuda") if case["norm"] else None  # noqa: E731
        held, row = _to_read(table, [0] * len(local), local, page)
        state.update(codes=codes, scales=scales, table=table, held=held, row=row, q=qkv[:, :heads * hd], k=qkv[:, heads * hd:(heads + kv) * hd],
                     v=qkv[:, (heads + kv) * hd:], q_weight=weight(), k_weight=weight(), cos=cos, sin=sin,
                     slots=slots.to(torch.int32), positions=positions, rows=ints(range(len(local))),
                     first=ints([first] * len(local)), last=ints([n - 1 for n in local]),
                     q_out=torch.zeros((tokens, heads, hd), dtype=dtype, device="cuda"),
                     values=torch.zeros((pages, 2, kv, page, hd), dtype=dtype, device="cuda"))
        return state
    pages, table = _pages(case, lengths, gen)
    codes, scales = _pool(case, pages, table, lengths, gen)
    state.update(codes=codes, scales=scales, table=table)
    n = len(lengths)
    if case["op"] == "read":
        # from the first page that holds a position which the query at the last one sees
        held, row = _to_read(table, [_first_seen(case, length) // page * page for length in lengths], lengths, page)
        state.update(held=held, row=row, rows=ints(range(n)), last=ints([length - 1 for length in lengths]), first=ints([length - 1 for length in lengths]),
                     values=torch.zeros((pages, 2, kv, page, hd), dtype=dtype, device="cuda"))
        return state
    padding, heads = case["padding"], case["heads"]
    tokens = torch.randperm(n + padding, generator=gen, device="cuda")[:n].to(torch.int32)   # which row of q a request's token is
    positions = torch.zeros(n + padding, dtype=torch.int32, device="cuda")
    positions[tokens.long()] = ints(lengths) - 1
    state.update(q=(1.5 * torch.randn((n + padding, heads, hd), generator=gen, device="cuda")).to(dtype),
                 row_token=torch.cat([tokens, ints([-1] * padding)]), row_request=torch.cat([ints(range(n)), ints([0] * padding)]),
                 positions=positions, longest=max(lengths), out=torch.zeros((n + padding, heads, hd), dtype=dtype, device="cuda"),
                 sink=torch.randn(heads, generator=gen, device="cuda") if case["sink"] else None)
    return state


# ------------------------------------------------------------------ the plain forms
def _turn(x, cos, sin, positions, how):
    """Rotation of heads x [tokens, n, head_dim] in float32."""
    if how == "none":
        return x
    c, s = cos[positions.long()][:, None, :], sin[positions.long()][:, None, :]
    turned = 2 * cos.shape[1]
    part, rest = x[..., :turned], x[..., turned:]
    if how == "pairs":
        a, b = part[..., 0::2], part[..., 1::2]
        return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), rest], -1)
    a, b = part[..., :turned // 2], part[..., turned // 2:]
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1)


def _normed(x, weight):
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _rows(state, held, row):
    """Rows ``row`` of pages ``held``, [rows, 2, kv_heads, head_dim] in float32."""
    codes = state["codes"].view(torch.uint8)[held, :, :, row].view(state["codes"].dtype)
    return codes.float() * state["scales"][held, :, :, row].unsqueeze(-1)


def _plain_read(state):
    held, row = state["held"], state["row"]
    state["values"][held, :, :, row] = _rows(state, held, row).to(state["values"].dtype)
    return state["values"]


def _plain_store(state):
    case = state["case"]
    kv, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    tokens = state["q"].shape[0]
    heads_of = lambda x: x.float().view(tokens, -1, hd)  # noqa: E731
    turn = lambda x: _turn(x, state["cos"], state["sin"], state["positions"], case["rotate"])  # noqa: E731
    state["q_out"].copy_(turn(_normed(heads_of(state["q"]), state["q_weight"])))
    rows = torch.stack([turn(_normed(heads_of(state["k"]), state["k_weight"])), heads_of(state["v"])], 1)   # [tokens, 2, kv, hd]
    codes, scales = _codes_of(rows, case["codes"])
    held, row = state["slots"].long() // page, state["slots"].long() % page
    state["codes"].view(torch.uint8)[held, :, :, row] = codes.view(torch.uint8)
    state["scales"][held, :, :, row] = scales
    return {"q": state["q_out"], "values": _plain_read(state)}


def _plain_attend(state):
    case = state["case"]
    n, kv, hd, page = case["requests"], case["kv_heads"], case["head_dim"], case["page"]
    group = case["heads"] // kv
    held = state["table"].long().clamp(min=0)
    keys = held.shape[1] * page
    tokens = state["row_token"][:n].long()
    pos = state["positions"].long()[tokens]
    at = torch.arange(keys, device="cuda")
    seen = at[None, :] <= pos[:, None]
    if case["window"]:
        seen &= at[None, :] > pos[:, None] - case["window"]

    def rows(plane):   # [requests, kv_heads, keys, head_dim]
        scales = torch.where(seen[:, None, :], state["scales"][held][:, :, plane].transpose(1, 2).reshape(n, kv, keys), 0.0)
        values = state["codes"].view(torch.uint8)[held][:, :, plane].view(CODES[case["codes"]]).float()
        return torch.where(seen[:, None, :, None], values.transpose(1, 2).reshape(n, kv, keys, hd), 0.0) * scales.unsqueeze(-1)

    q = state["q"].float()[tokens].view(n, kv, group, hd)
    scores = torch.matmul(q, rows(0).transpose(-1, -2)) / math.sqrt(hd)
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    if state["sink"] is not None:
        total = total + torch.exp(state["sink"].view(1, kv, group, 1) - top)
    out = torch.matmul(weights, rows(1)) / total
    state["out"][tokens] = out.view(n, case["heads"], hd).to(state["out"].dtype)
    return state["out"]


def run(state):
    case = state["case"]
    if own:
        from metallix_b200 import ops
        pool = ops.QuantizedPool(state["codes"], state["scales"])
        if case["op"] == "attend":
            return ops.paged_attention_decode(
                state["q"], pool, state["out"], state["table"], state["row_token"], state["row_request"], state["positions"],
                1.0 / math.sqrt(case["head_dim"]), state["longest"], window=case["window"], softcap=case["softcap"],
                sink=state["sink"])
        if case["op"] == "read":
            return ops.read_cache(pool, state["values"], state["table"], state["rows"], state["first"], state["last"],
                                  window=case["window"])
        ops.qk_norm_rope_cache(state["q"], state["k"], state["v"], state["q_out"], pool, state["slots"], state["positions"],
                               state["q_weight"], state["k_weight"], state["cos"], state["sin"], EPS,
                               interleaved=case["rotate"] == "pairs")
        ops.read_cache(pool, state["values"], state["table"], state["rows"], state["first"], state["last"])
        return {"q": state["q_out"], "values": state["values"]}
    if case["op"] == "attend":
        return _plain_attend(state)
    if case["op"] == "store":
        return _plain_store(state)
    return _plain_read(state)


# ------------------------------------------------------------------ the definitions, in 64 bits
def _exact_codes(x, kind):
    """What rows x (float64) read back as: the nearest code, halves to even, times the scale."""
    limit = LIMITS[kind]
    scale = (x.abs().max(-1, keepdim=True).values / limit).float().double()   # kept in 32 bits
    y = x / torch.where(scale == 0, torch.ones_like(scale), scale)
    if kind == "int8":
        return torch.round(y) * scale
    exponent = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.pow(2.0, exponent - 3)
    return torch.round(y / step) * step * scale


def exact(case, seed):
    s = prepare(case, seed)
    page, hd = case["page"], case["head_dim"]
    table, lengths = s["table"].long().cpu(), _lengths(case)
    if case["op"] == "read":
        out = torch.zeros(s["values"].shape, dtype=torch.float64, device="cuda")
        for r, length in enumerate(lengths):
            seen_page = _first_seen(case, length) // page
            for p in range(seen_page, -(-length // page)):
                count, where = min(page, length - p * page), int(table[r, p])
                out[where, :, :, :count] = s["codes"][where, :, :, :count].double() * s["scales"][where, :, :, :count].double()[..., None]
        return out
    if case["op"] == "store":
        def heads(x, weight, turned):
            x = x.double().reshape(x.shape[0], -1, hd)
            if weight is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + EPS) * weight.double()
            if turned and s["cos"] is not None:
                half = s["cos"].shape[1]
                where = torch.arange(half, device="cuda")
                i, j = (2 * where, 2 * where + 1) if case["rotate"] == "pairs" else (where, where + half)
                c, sn = (t.double()[s["positions"].long()].unsqueeze(1) for t in (s["cos"], s["sin"]))
                y = x.clone()
                y[..., i] = x[..., i] * c - x[..., j] * sn
                y[..., j] = x[..., j] * c + x[..., i] * sn
                x = y
            return x
        out = torch.zeros(s["values"].shape, dtype=torch.float64, device="cuda")
        skipped = case["start"] // page * page
        for r, length in enumerate(lengths):   # what the pages held before the step
            n = case["start"] - skipped
            where = int(table[r, 0])
            out[where, :, :, :n] = s["codes"][where, :, :, :n].double() * s["scales"][where, :, :, :n].double()[..., None]
        held, row = s["slots"].long() // page, s["slots"].long() % page
        out[held, 0, :, row] = _exact_codes(heads(s["k"], s["k_weight"], True), case["codes"])
        out[held, 1, :, row] = _exact_codes(heads(s["v"], None, False), case["codes"])
        return {"q": heads(s["q"], s["q_weight"], True), "values": out}
    if sum(lengths) * case["heads"] * hd > 4e9:
        return None
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for r, length in enumerate(lengths):
        token, begin = int(s["row_token"][r]), _first_seen(case, length)
        at = torch.arange(begin, length)
        held, row = table[r, at // page].cuda(), (at % page).cuda()
        rows = s["codes"].view(torch.uint8)[held, :, :, row].view(CODES[case["codes"]]).double() * s["scales"][held, :, :, row].double()[..., None]
        keys, values = (rows[:, plane].repeat_interleave(group, 1) for plane in (0, 1))      # [keys, heads, head_dim]
        score = torch.einsum("hd,khd->hk", s["q"][token].double(), keys) / hd ** 0.5
        if case["softcap"]:
            score = case["softcap"] * torch.tanh(score / case["softcap"])
        if s["sink"] is not None:
            score = torch.cat([score, s["sink"].double()[:, None]], 1)
        weight = torch.softmax(score, 1)[:, :length - begin]
        out[token] = torch.einsum("hk,khd->hd", weight, values)
    return out
