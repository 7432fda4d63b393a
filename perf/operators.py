"""The operators that serve a model held in 4 bits, and the work that their speed is measured on.

- ``store``: keys and values of a step's tokens are quantised into the pages of a 4-bit cache as they are written, and the rows
  written are read back.
- ``attend``: attention over a 4-bit cache, for sequences that bring one token and for sequences that bring a portion of a prompt.
- ``linear``: the product of a few tokens with a 4-bit weight, stored in the activations' type, in float32, or with a SiLU gate.

What 4 bits hold: ``group`` neighbouring values share a minimum z and a step s, both float16, and a value is c s + z with c in 0 .. 15:
z = float16(min x), s = float16((max x - z) f) with f the float32 next to 1/15, the difference and the product in float32,
c = (x - z) / s rounded to the nearest, ties to even, and cut to 0 .. 15; s = 0 gives c = 0.  A group that holds a value beyond 60000, or one that is not finite, is
not a number as a whole.

Sizes are those of the engine's 1b, 8b and 14b layers and of its tiny models.  Inputs are normal (keys with the louder channels that
rotated keys have), pages are handed out in random order.
"""
import math

import torch

own = False
DEVICE = "cuda"
LIMIT = 60000.0


# ------------------------------------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------------------------------------
def store(dtype, d, kv_heads, group, seqs, tokens, past, spread=0.0, page=16):
    """``seqs`` sequences bring ``tokens`` tokens each (less by up to the share ``spread``) behind ``past`` others."""
    return {"kind": "store", "dtype": dtype, "d": d, "kv_heads": kv_heads, "group": group, "seqs": seqs, "tokens": tokens, "past": past,
            "spread": spread, "page": page}


def attend(dtype, d, heads, kv_heads, group, seqs, tokens, context, spread=0.0, window=0, page=16):
    """``seqs`` sequences bring ``tokens`` tokens each; with them they hold ``context`` tokens, less by up to the share ``spread``."""
    return {"kind": "attend", "dtype": dtype, "d": d, "heads": heads, "kv_heads": kv_heads, "group": group, "seqs": seqs, "tokens": tokens,
            "context": context, "spread": spread, "window": window, "page": page}


def linear(dtype, mode, tokens, rows, width, group):
    """x [tokens, width] times a weight of ``rows`` rows (twice as many with mode "gated")."""
    return {"kind": "linear", "dtype": dtype, "mode": mode, "tokens": tokens, "rows": rows, "width": width, "group": group}


def listed():
    cases = {
        # a decode step of a few users: one row of every head and sequence
        "store-decode": store("bfloat16", 128, 8, 64, seqs=8, tokens=1, past=2047),
        # a whole prompt goes into the cache
        "store-prompt": store("bfloat16", 128, 8, 64, seqs=1, tokens=2048, past=0),
        # the float32 path, portions of odd lengths that start in the middle of a page
        "store-float32": store("float32", 64, 4, 32, seqs=5, tokens=301, past=21, spread=0.9, page=32),
        # one user's stream of tokens
        "attend-1": attend("bfloat16", 128, 32, 8, 64, seqs=1, tokens=1, context=2048),
        # a busy server: the cache's bytes are what counts
        "attend-64": attend("bfloat16", 128, 32, 8, 64, seqs=64, tokens=1, context=8192),
        # requests of all ages, five query heads a key head, fine groups
        "attend-ragged": attend("bfloat16", 128, 40, 8, 32, seqs=21, tokens=1, context=9000, spread=0.95),
        # the float32 path with a window
        "attend-float32": attend("float32", 64, 16, 4, 32, seqs=4, tokens=1, context=700, spread=0.5, window=200),
        # a portion of a long document whose first 6,000 tokens are cached
        "attend-portion": attend("bfloat16", 128, 32, 8, 64, seqs=1, tokens=1733, context=7733),
        # one user's token through the product for queries, keys and values
        "linear-1": linear("bfloat16", "store", 1, 6144, 4096, 64),
        # a few users' tokens through the gated product of the feed-forward
        "linear-8-gated": linear("bfloat16", "gated", 8, 12288, 4096, 64),
        # a busy server's tokens through the feed-forward's second product
        "linear-64": linear("bfloat16", "float32", 64, 4096, 12288, 32),
        # the float32 path, an odd number of tokens and rows
        "linear-float32": linear("float32", "store", 5, 1003, 2048, 32),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "portion", "linear", "linear"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    d, group, page = rng.choice([64, 128, 128, 256]), rng.choice([32, 64]), rng.choice([16, 32, 64])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    if kind == "store":
        seqs = log_uniform(rng, 1, 64)
        return store(dtype, d, kv_heads, group, seqs, log_uniform(rng, 1, max(2, 4096 // seqs)), rng.randint(0, 300),
                     rng.choice([0.0, 0.5, 0.9]), page)
    if kind == "attend":
        seqs = log_uniform(rng, 1, 64)
        if dtype == "float32":
            seqs = min(seqs, 16)
        context = log_uniform(rng, 1, min(9000, 262144 // seqs))
        return attend(dtype, d, heads, kv_heads, group, seqs, 1, context, rng.choice([0.0, 0.5, 0.95]), rng.choice([0, 0, 128, 1000]), page)
    if kind == "portion":
        tokens = log_uniform(rng, 2, 1200)
        return attend(dtype, d, heads, kv_heads, group, rng.choice([1, 1, 2, 3]) if tokens < 500 else 1, tokens,
                      tokens + log_uniform(rng, 1, 4000) - 1, rng.choice([0.0, 0.3]), rng.choice([0, 0, 500]), page)
    mode = rng.choice(["store", "gated", "float32"])
    return linear(dtype, mode, log_uniform(rng, 1, 64), log_uniform(rng, 40, 9000), 64 * log_uniform(rng, 2, 100), group)


def lengths(case):
    """(tokens brought, tokens held after them) of every sequence."""
    n = case["seqs"]
    share = [1.0 - case["spread"] * i / max(n - 1, 1) for i in range(n)]
    if case["kind"] == "store":
        new = [max(1, int(case["tokens"] * s)) for s in share]
        return new, [case["past"] + k for k in new]
    held = [max(1, int(case["context"] * s)) for s in share]
    return [min(case["tokens"], h) for h in held], held


# ------------------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------------------
def normal(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * scale).to(getattr(torch, dtype))


def rows_of_cache(case, n, seed):
    """Keys and values [n, kv_heads, d] of n tokens, as the projections leave them: some channels of a key are louder than others."""
    shape = (n, case["kv_heads"], case["d"])
    loud = 1.0 + 3.0 * (torch.arange(case["d"], device=DEVICE) % 17 == 3)
    return (normal(shape, 16 * seed + 1, "float32") * loud).to(getattr(torch, case["dtype"])), normal(shape, 16 * seed + 2, case["dtype"], 0.5)


def tables(case, seed):
    """Block table [seqs, most pages] over pages in random order, and which sequence and position every token brought has."""
    new, held = lengths(case)
    per = [-(-h // case["page"]) for h in held]
    order = torch.randperm(sum(per), generator=torch.Generator().manual_seed(16 * seed + 3))
    table = torch.full((len(per), max(per)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(DEVICE), sum(per)


def places(first, counts):
    """Sequence and position of ``counts[b]`` tokens from position ``first[b]`` on, sequence after sequence (int32)."""
    seq = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    start = torch.tensor([0] + counts[:-1]).cumsum(0)
    pos = torch.arange(len(seq)) - start[seq] + torch.tensor(first)[seq]
    return seq.to(torch.int32).to(DEVICE), pos.to(torch.int32).to(DEVICE)


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    dtype = getattr(torch, case["dtype"])
    state = {"case": case}
    if case["kind"] == "linear":
        gated = case["mode"] == "gated"
        shape = (case["rows"] * (2 if gated else 1), case["width"])
        weight = normal(shape, 16 * seed + 5, "bfloat16", 0.02)
        state["x"] = normal((case["tokens"], case["width"]), 16 * seed + 4, case["dtype"])
        state["out"] = torch.empty((case["tokens"], case["rows"]), dtype=torch.float32 if case["mode"] == "float32" else dtype, device=DEVICE)
        if own:
            from carbon_engine_b200 import ops_int4
            state["weight"] = ops_int4.Int4Weight.quantize(weight, case["group"], gated=gated)
        else:
            state["weight"] = quantise(weight, case["group"])
        return state
    new, held = lengths(case)
    table, pages = tables(case, seed)
    before = [h - n for h, n in zip(held, new)]
    state.update(table=table, slots=int32(range(len(new))), status=int32([0]))
    state["seq"], state["pos"] = places(before, new)
    shape = (pages, case["kv_heads"], case["page"])
    if own:
        from carbon_engine_b200 import ops_int4
        state["pages"] = ops_int4.Int4Pages(pages, case["kv_heads"], case["page"], case["d"], case["group"], device=DEVICE)
    if case["kind"] == "store":
        # a step's keys and values lie side by side in the rows of one product
        k, v = rows_of_cache(case, sum(new), seed)
        both = torch.cat([k.flatten(1), v.flatten(1)], dim=1)
        state["k"], state["v"] = (both[:, i * k[0].numel():(i + 1) * k[0].numel()].unflatten(1, k.shape[1:]) for i in (0, 1))
        state["k_back"], state["v_back"] = torch.empty_like(k), torch.empty_like(v)
        if not own:
            state["codes"] = [torch.zeros(shape + (case["d"] // 2,), dtype=torch.uint8, device=DEVICE) for _ in range(2)]
            state["steps"] = [torch.zeros(shape + (case["d"] // case["group"], 2), dtype=torch.float16, device=DEVICE) for _ in range(2)]
        return state
    # what earlier steps and the tokens at hand have left in the cache
    seq, pos = places([0] * len(held), held)
    k, v = rows_of_cache(case, sum(held), seed)
    if own:
        ops_int4.kv_write(state["pages"], k, v, pos, seq, state["slots"], table, state["status"])
    else:
        state["codes"], state["steps"] = [], []
        page, slot = table[seq.long(), pos.long() // case["page"]].long(), pos.long() % case["page"]
        for rows in (k, v):
            codes, steps = quantise(rows, case["group"])
            state["codes"].append(torch.zeros(shape + codes.shape[2:], dtype=torch.uint8, device=DEVICE))
            state["steps"].append(torch.zeros(shape + steps.shape[2:], dtype=torch.float16, device=DEVICE))
            state["codes"][-1][page, :, slot], state["steps"][-1][page, :, slot] = codes, steps
    state["q"] = normal((sum(new), case["heads"], case["d"]), 16 * seed + 6, case["dtype"])
    state["out"] = torch.empty_like(state["q"])
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state["starts"], state["held"], state["new"] = int32(starts), int32(held), int32(new)
    # one-token sequences are taken as such; the others in runs of 64 tokens
    state["decoding"] = len(new) if max(new) == 1 else 0
    state["tiles"] = None if max(new) == 1 else int32([(b, at) for b, n in enumerate(new) for at in range(0, n, 64)])
    return state


# ------------------------------------------------------------------------------------------------------------------------------
# the plain forms, and the framework's calls
# ------------------------------------------------------------------------------------------------------------------------------
def quantise(x, group):
    """Codes (two a byte, the lower one first) and (step, minimum) of the groups along the last axis.  Codes in 64 bits: a value may lie
    next to the border between two."""
    x = x.unflatten(-1, (-1, group))
    lo, hi = x.amin(-1).float(), x.amax(-1).float()
    z = lo.half()
    s = ((hi - z.float()) * torch.tensor(1.0 / 15.0, dtype=torch.float32, device=x.device)).half()
    bad = ~((x.float().abs() <= LIMIT).all(-1))
    s, z = s.masked_fill(bad, math.nan), z.masked_fill(bad, math.nan)
    code = ((x.double() - z.double()[..., None]) / s.double()[..., None]).round().clamp(0, 15)
    code = torch.where((s > 0)[..., None], code, torch.zeros_like(code)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.stack([s, z], dim=-1)


def values(codes, steps):
    """What codes and (step, minimum) stand for, in float32 along the last axis."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).float().unflatten(-1, (steps.shape[-2], -1))
    return (c * steps[..., 0:1].float() + steps[..., 1:2].float()).flatten(-2)


def run(state):
    return {"store": run_store, "attend": run_attend, "linear": run_linear}[state["case"]["kind"]](state)


def run_store(state):
    case = state["case"]
    if own:
        from carbon_engine_b200 import ops_int4
        where = (state["pos"], state["seq"], state["slots"], state["table"], state["status"])
        ops_int4.kv_write(state["pages"], state["k"], state["v"], *where)
        ops_int4.kv_read(state["pages"], state["k_back"], state["v_back"], *where)
        return {"k": state["k_back"], "v": state["v_back"]}
    pos = state["pos"].long()
    page = state["table"][state["slots"][state["seq"].long()].long(), pos // case["page"]].long()
    slot = pos % case["page"]
    out = {}
    for name, x, codes, steps in zip("kv", (state["k"], state["v"]), state["codes"], state["steps"]):
        codes[page, :, slot], steps[page, :, slot] = quantise(x, case["group"])
        out[name] = values(codes[page, :, slot], steps[page, :, slot]).to(x.dtype)
    return out


def run_attend(state):
    case = state["case"]
    scale = 1.0 / math.sqrt(case["d"])
    if own:
        from carbon_engine_b200 import ops_int4
        ops_int4.attention(state["q"], state["pages"], state["out"], state["slots"], state["starts"], state["held"], state["table"],
                           state["status"], n_decode=state["decoding"], max_ctx=case["context"], tiles=state["tiles"],
                           window=case["window"], scale=scale)
        return state["out"]
    new, held, starts = state["new"].long(), state["held"].long(), state["starts"].long()
    n, heads, kv_heads = case["tokens"], case["heads"], case["kv_heads"]
    k, v = (values(codes[state["table"].clamp(min=0).long()], steps[state["table"].clamp(min=0).long()]).transpose(1, 2).flatten(2, 3)
            for codes, steps in zip(state["codes"], state["steps"]))                     # [seqs, kv_heads, keys, d]
    i = torch.arange(n, device=DEVICE)
    rows = torch.minimum(starts[:-1, None] + i, starts[1:, None] - 1)                    # a sequence with fewer tokens repeats its last
    q = state["q"].float()[rows].unflatten(2, (kv_heads, -1)).permute(0, 2, 3, 1, 4)     # [seqs, kv_heads, heads of it, tokens, d]
    scores = (q.flatten(2, 3) @ k.transpose(2, 3) * scale).unflatten(2, (-1, n))
    at = (held - new)[:, None] + torch.minimum(i, new[:, None] - 1)
    key = torch.arange(k.shape[2], device=DEVICE)
    seen = key <= at[..., None]
    if case["window"]:
        seen &= key > at[..., None] - case["window"]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (-1, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [seqs, tokens, heads, d]
    return o[i < new[:, None]].to(state["q"].dtype)


def run_linear(state):
    case = state["case"]
    if own:
        from carbon_engine_b200 import ops, ops_int4
        mode = {"store": ops.GEMM_STORE, "gated": ops.GEMM_SWIGLU, "float32": ops.GEMM_STORE_F32}[case["mode"]]
        ops_int4.matmul(state["x"], state["weight"], state["out"], mode)
        return state["out"]
    y = state["x"].float() @ values(*state["weight"]).T
    if case["mode"] == "gated":
        gate, up = y.chunk(2, dim=1)
        y = gate / (1.0 + (-gate).exp()) * up
    return y.to(state["out"].dtype)


def work(case):
    """Each input read once, each output written once: 4 bits a value and (step, minimum) a group, activations in their own type."""
    el = 2 if case["dtype"] == "bfloat16" else 4
    bits = 0.5 + 4.0 / case["group"]
    if case["kind"] == "linear":
        rows = case["rows"] * (2 if case["mode"] == "gated" else 1)
        out = case["tokens"] * case["rows"] * (4 if case["mode"] == "float32" else el)
        return {"bytes": rows * case["width"] * bits + case["tokens"] * case["width"] * el + out, "flops": 2 * case["tokens"] * rows * case["width"]}
    new, held = lengths(case)
    row = 2 * case["kv_heads"] * case["d"]                    # values of a token's key and value
    if case["kind"] == "store":                               # read, held, read back and written: a difference, a product and a sum each
        return {"bytes": sum(new) * row * (2 * el + 2 * bits), "flops": 6 * sum(new) * row}
    keys = pairs = 0
    for n, h in zip(new, held):
        first = max(0, h - n + 1 - case["window"]) if case["window"] else 0
        keys += h - first
        pairs += sum(min(p + 1, case["window"] or p + 1) for p in range(h - n, h))
    return {"bytes": keys * row * bits + 2 * sum(new) * case["heads"] * case["d"] * el, "flops": 4 * pairs * case["heads"] * case["d"]}


# ------------------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------------------------------------
def held_values(x, group):
    """The values that 4 bits hold for x, in float64: of z + n s, n = 0 .. 15, the one next to x (n even where two are as near)."""
    rows = x.reshape(-1, group)
    least, most = rows.min(dim=1).values.to(torch.float32), rows.max(dim=1).values.to(torch.float32)
    z = least.to(torch.float16).double()
    # (the product of two float32 numbers is exact in float64)
    f = float(torch.tensor(1.0 / 15.0, dtype=torch.float32))
    s = (torch.sub(most, z.to(torch.float32)).double() * f).to(torch.float32).to(torch.float16).double()
    y = rows.double()
    t = (y - z[:, None]) / torch.where(s > 0, s, torch.ones_like(s))[:, None]
    whole = torch.floor(t)
    rest = t - whole
    whole += ((rest > 0.5) | ((rest == 0.5) & (whole % 2 == 1))).double()
    whole = torch.minimum(torch.maximum(whole, torch.zeros_like(whole)), torch.full_like(whole, 15.0))
    return (whole * s[:, None] + z[:, None]).reshape(x.shape)


def exact(case, seed):
    if case["kind"] == "linear":
        gated = case["mode"] == "gated"
        w = normal((case["rows"] * (2 if gated else 1), case["width"]), 16 * seed + 5, "bfloat16", 0.02)
        x = normal((case["tokens"], case["width"]), 16 * seed + 4, case["dtype"]).double()
        parts = []
        for at in range(0, len(w), 2048):
            parts.append(x @ held_values(w[at:at + 2048], case["group"]).T)
        y = torch.cat(parts, dim=1)
        return torch.sigmoid(y[:, :case["rows"]]) * y[:, :case["rows"]] * y[:, case["rows"]:] if gated else y
    new, held = lengths(case)
    if case["kind"] == "store":
        k, v = rows_of_cache(case, sum(new), seed)
        return {"k": held_values(k, case["group"]), "v": held_values(v, case["group"])}
    k, v = rows_of_cache(case, sum(held), seed)
    q = normal((sum(new), case["heads"], case["d"]), 16 * seed + 6, case["dtype"]).double()
    each = case["heads"] // case["kv_heads"]
    out = torch.empty_like(q)
    row = first = 0
    for n, h in zip(new, held):
        keys, vals = (held_values(t[first:first + h], case["group"]) for t in (k, v))
        where = torch.arange(h - n, h, device=DEVICE)
        far = where[:, None] - torch.arange(h, device=DEVICE)[None, :]
        hidden = (far < 0) | (far >= (case["window"] or h + 1))
        for head in range(case["heads"]):
            score = q[row:row + n, head] @ keys[:, head // each].T / math.sqrt(case["d"])
            out[row:row + n, head] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=1) @ vals[:, head // each]
        row, first = row + n, first + h
    return out
