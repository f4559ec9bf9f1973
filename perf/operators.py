"""The serving operators as they are measured: cases, inputs, calls, plain forms and 64-bit definitions.

Three operators of one low-precision decoder layer: keys and values rotated and appended to a
paged cache (16-bit or 4-bit), attention over that cache, and the linear layers around them in
8-bit integers.  ``own`` chooses between the plain forms (elementary torch operations) and the
calls a user makes of this package.

A 4-bit cache row (one token of one head) stands for low + code * scale with codes 0..15: low is
the row's smallest value, scale is (largest - smallest) / 15 rounded to the row's 16-bit type,
and a code is (value - low) / scale rounded to the nearest whole number, ties to the even one.
The values that are quantised are the rotated keys (or the values) rounded to that type.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step's append: a token of each of 64 sequences, 32 query heads on 8 K/V heads
        {"name": "append16 decode", "op": "append", "tokens": 64, "seqs": 64, "heads": 32, "kv": 8,
         "dim": 128, "rot": 128, "block": 16, "bits": 16, "dtype": "bfloat16",
         "interleaved": False, "order": "head"},
        # a prefill of ragged prompts, adjacent-pair rotation of half the head, token-major pages
        {"name": "append16 prefill", "op": "append", "tokens": 16385, "seqs": 8, "heads": 32,
         "kv": 32, "dim": 128, "rot": 64, "block": 64, "bits": 16, "dtype": "float16",
         "interleaved": True, "order": "token"},
        # a decode step's append into the 4-bit cache at a large batch
        {"name": "append4 decode", "op": "append", "tokens": 256, "seqs": 256, "heads": 32,
         "kv": 8, "dim": 128, "rot": 128, "block": 32, "bits": 4, "dtype": "float16",
         "interleaved": False, "order": "head"},
        # a prefill into the 4-bit cache
        {"name": "append4 prefill", "op": "append", "tokens": 32768, "seqs": 16, "heads": 32,
         "kv": 8, "dim": 128, "rot": 128, "block": 64, "bits": 4, "dtype": "bfloat16",
         "interleaved": False, "order": "head"},
        # one user with a short context: latency is all there is
        {"name": "attend16 one user", "op": "attend", "seqs": 1, "queries": 1, "keys": 1000,
         "heads": 32, "kv": 8, "dim": 128, "block": 16, "bits": 16, "dtype": "bfloat16",
         "order": "head"},
        # a served batch on 16-bit pages, small heads, token-major pages, odd group of 7
        {"name": "attend16 batch", "op": "attend", "seqs": 64, "queries": 1, "keys": 4096,
         "heads": 28, "kv": 4, "dim": 64, "block": 32, "bits": 16, "dtype": "float16",
         "order": "token"},
        # one user of the 4-bit cache with a few thousand keys
        {"name": "attend4 one user", "op": "attend", "seqs": 1, "queries": 1, "keys": 4097,
         "heads": 32, "kv": 8, "dim": 128, "block": 32, "bits": 4, "dtype": "bfloat16",
         "order": "head"},
        # a few very long contexts, the reason for four bits
        {"name": "attend4 long", "op": "attend", "seqs": 8, "queries": 1, "keys": 131072,
         "heads": 32, "kv": 8, "dim": 128, "block": 64, "bits": 4, "dtype": "bfloat16",
         "order": "head"},
        # append and attention together, several drafted tokens per sequence
        {"name": "step4 drafted", "op": "step", "seqs": 48, "queries": 4, "keys": 8192,
         "heads": 32, "kv": 8, "dim": 128, "rot": 128, "block": 64, "bits": 4,
         "dtype": "bfloat16", "interleaved": False, "order": "head"},
        # a linear layer of a decode step: the weight is read once for a few tokens
        {"name": "linear8 decode", "op": "linear", "rows": 8, "out": 14336, "in": 4096,
         "dtype": "bfloat16", "bias": False, "act": "none"},
        # a ragged prefill
        {"name": "linear8 ragged", "op": "linear", "rows": 4097, "out": 11008, "in": 4096,
         "dtype": "bfloat16", "bias": True, "act": "gelu_tanh"},
        # the largest product
        {"name": "linear8 square", "op": "linear", "rows": 8192, "out": 8192, "in": 8192,
         "dtype": "float16", "bias": True, "act": "none"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["bfloat16", "float16"])
    op = rng.choice(["append", "attend", "attend", "step", "linear"])
    if op == "linear":
        rows = _spread(rng, 1, 8192)
        return {"op": op, "rows": rows, "out": 16 * _spread(rng, 8, 896),
                "in": 16 * _spread(rng, 16, 512), "dtype": dtype,
                "bias": rng.random() < 0.5, "act": rng.choice(["none", "gelu_tanh"])}
    bits = rng.choice([4, 4, 16])
    kv = rng.choice([1, 2, 4, 8, 8])
    case = {"op": op, "heads": kv * rng.choice([1, 2, 4, 5, 7, 8]), "kv": kv,
            "dim": rng.choice([64, 128, 128]), "block": rng.choice([16, 32, 48, 64, 128]),
            "bits": bits, "dtype": dtype, "order": rng.choice(["head", "head", "token"])}
    if op != "attend":
        case["rot"] = rng.choice([case["dim"], case["dim"], case["dim"] // 2])
        case["interleaved"] = rng.random() < 0.3
    if op == "append":
        case["tokens"] = _spread(rng, 1, 20000)
        case["seqs"] = min(case["tokens"], _spread(rng, 1, 128))
        return case
    case["seqs"] = _spread(rng, 1, 128)
    case["keys"] = _spread(rng, 16, min(131072, 700000 // case["seqs"]))
    case["queries"] = rng.choice([1, 1, 1, 2, 5]) if case["keys"] > 16 else 1
    return case


def _lengths(case):
    """Ragged context lengths: the longest is case["keys"], the others down to a third of it."""
    rng = random.Random(case["keys"] * 1000 + case["seqs"])
    n, top = case["seqs"], case["keys"]
    low = max(case["queries"], top // 3, 1)
    return [top] + [rng.randint(min(low, top), top) for _ in range(n - 1)]


def _queries(case):
    """Query tokens per sequence: 1, or ragged up to case["queries"] (at least one)."""
    rng = random.Random(case["keys"] + 7 * case["seqs"])
    top = case["queries"]
    return [top] + [rng.randint(1, top) for _ in range(case["seqs"] - 1)]


def _prompt_spans(case):
    """(start position, tokens) of each sequence of an append; a prefill starts some sequences
    behind an earlier part and ends with a few padding tokens that belong to none."""
    n, total = case["seqs"], case["tokens"]
    rng = random.Random(total * 1000 + n)
    if total == n:
        return [(rng.randint(0, 4095), 1) for _ in range(n)], 0
    pad = min(5, total - n)
    cuts = sorted(rng.sample(range(1, total - pad), n - 1)) if n > 1 else []
    edges = [0] + cuts + [total - pad]
    return [(rng.choice([0, 0, rng.randint(1, 500)]), edges[i + 1] - edges[i]) for i in range(n)], pad


# ----------------------------------------------------------------------------------- the inputs
def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _tables(gen, lengths, block):
    """Page table with the pages of all sequences in a random order, -1 behind each last page."""
    counts = [-(-n // block) for n in lengths]
    total = sum(counts)
    width = max(counts) + 1
    order = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for z, n in enumerate(counts):
        table[z, :n] = order[at:at + n]
        at += n
    return table, total


def _paged(case, pages, last, dtype):
    """An empty paged tensor [pages, kv, block, last] whose memory is head- or token-major."""
    if case["order"] == "head":
        return torch.empty((pages, case["kv"], case["block"], last), dtype=dtype, device=DEV)
    return torch.empty((pages, case["block"], case["kv"], last), dtype=dtype, device=DEV).transpose(1, 2)


def _fill_cache(case, gen, pages, dtype, state):
    """A cache with contents: rows with a common offset per channel, as keys have."""
    for side, shift in (("k", 1.0), ("v", 0.2)):
        dim = case["dim"]
        offset = torch.randn((1, case["kv"], 1, dim), generator=gen, device=DEV) * shift
        if case["bits"] == 16:
            cache = _paged(case, pages, dim, dtype)
            step = max(1, (1 << 26) // (case["kv"] * case["block"] * dim))
            for p in range(0, pages, step):
                part = cache[p:p + step]
                part.copy_(torch.randn(part.shape, generator=gen, device=DEV) + offset)
        else:
            cache = _paged(case, pages, dim // 2, torch.uint8)
            params = _paged(case, pages, 2, dtype)
            cache.copy_(torch.randint(0, 256, cache.shape, generator=gen, device=DEV, dtype=torch.uint8))
            spread = torch.rand(params.shape[:3], generator=gen, device=DEV)
            params[..., 0].copy_(0.2 + 0.2 * spread)
            params[..., 1].copy_(-3.0 - spread)
            state[side + "_params"] = params
        state[side + "_cache"] = cache


def _angles(case, top, state):
    half = case["rot"] // 2
    rate = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    angle = torch.arange(top, dtype=torch.float64, device=DEV)[:, None] * rate[None]
    state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()


def _new_tokens(case, gen, tokens, dtype, state):
    for name, heads in (("q", case["heads"]), ("k", case["kv"]), ("v", case["kv"])):
        state[name] = _normal(gen, (tokens, heads, case["dim"]), dtype)
    state["q_out"] = torch.empty_like(state["q"])
    if case["bits"] == 4:   # what the cache stands for, for the prompt's own attention
        state["k_out"], state["v_out"] = torch.empty_like(state["k"]), torch.empty_like(state["v"])


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "linear":
        m, n, k = case["rows"], case["out"], case["in"]
        state["x"] = _normal(gen, (m, k), dtype)
        state["w"] = torch.randint(-127, 128, (n, k), generator=gen, device=DEV, dtype=torch.int8)
        state["w_scale"] = (0.5 + torch.rand(n, generator=gen, device=DEV)) / (73.0 * math.sqrt(k))
        state["bias"] = _normal(gen, (n,), dtype, 0.1) if case["bias"] else None
        state["x8"] = torch.empty((m, k), dtype=torch.int8, device=DEV)
        state["x_scale"] = torch.empty(m, dtype=torch.float32, device=DEV)
        state["y"] = torch.empty((m, n), dtype=dtype, device=DEV)
        return state
    if case["op"] == "append":
        spans, pad = _prompt_spans(case)
        state["table"], pages = _tables(gen, [s + n for s, n in spans], case["block"])
        seq = [z for z, (_, n) in enumerate(spans) for _ in range(n)] + [-1] * pad
        pos = [s + i for s, n in spans for i in range(n)] + [0] * pad
        _angles(case, max(s + n for s, n in spans), state)
        _fill_cache(case, gen, pages, dtype, state)
    else:
        lengths, counts = _lengths(case), _queries(case)
        state["table"], pages = _tables(gen, lengths, case["block"])
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        state["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        state["spans"] = list(zip(starts[:-1], counts, lengths))
        _fill_cache(case, gen, pages, dtype, state)
        tokens = starts[-1]
        state["out"] = torch.empty((tokens, case["heads"], case["dim"]), dtype=dtype, device=DEV)
        state["lse"] = torch.empty((tokens, case["heads"]), dtype=torch.float32, device=DEV)
        if own:
            from compiler_b200 import ops
            size = ops.attention_paged_workspace(tokens, case["heads"], case["kv"], case["dim"])
            state["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEV)
        if case["op"] == "attend":
            state["q"] = _normal(gen, (tokens, case["heads"], case["dim"]), dtype)
            return state
        seq = [z for z, n in enumerate(counts) for _ in range(n)]
        pos = [lengths[z] - n + i for z, n in enumerate(counts) for i in range(n)]
        _angles(case, max(lengths), state)
    state["live"] = sum(z >= 0 for z in seq)
    state["seq"] = torch.tensor(seq, dtype=torch.int32, device=DEV)
    state["pos"] = torch.tensor(pos, dtype=torch.int32, device=DEV)
    _new_tokens(case, gen, len(seq), dtype, state)
    return state


# ------------------------------------------------------------------------------------- the runs
def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_append(s):
    from compiler_b200 import ops
    ops.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["seq"], s["pos"],
                  k_params=s.get("k_params"), v_params=s.get("v_params"), cos=s["cos"],
                  sin=s["sin"], interleaved=s["case"]["interleaved"], q=s["q"], q_out=s["q_out"],
                  k_out=s.get("k_out"), v_out=s.get("v_out"), stream=_stream())


def _own_attend(s, q):
    from compiler_b200 import ops
    ops.attention_paged(q, s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["out"],
                        s["workspace"], k_params=s.get("k_params"), v_params=s.get("v_params"),
                        cu_seqlens_q=s["starts"], lse=s["lse"], stream=_stream())


def _own_linear(s):
    from compiler_b200 import ops
    from compiler_b200.runtime import abi
    act = {"none": abi.ACT_NONE, "gelu_tanh": abi.ACT_GELU_TANH}[s["case"]["act"]]
    ops.quantize_rows(s["x"], s["x8"], s["x_scale"], stream=_stream())
    ops.linear_int8(s["x8"], s["x_scale"], s["w"], s["w_scale"], s["y"], bias=s["bias"], act=act,
                    stream=_stream())


def _rotated(x, cos, sin, rot, interleaved):
    """x [T, heads, dim] in 64 bits, cos / sin [T, rot / 2]; the same in 64 bits."""
    part, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
    c, s = cos[:, None].double(), sin[:, None].double()
    first, second = a * c - b * s, b * c + a * s
    if interleaved:
        part = torch.stack((first, second), dim=-1).flatten(-2)
    else:
        part = torch.cat((first, second), dim=-1)
    return torch.cat((part, rest), dim=-1)


def _nearest(x, dtype):
    """64-bit values rounded once to the nearest value of a 16-bit type, still in 64 bits."""
    digits, lowest = (8, -125) if dtype == torch.bfloat16 else (11, -13)
    _, exponent = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), exponent.clamp(min=lowest) - digits)
    return torch.round(x / step) * step


def _four_bits(x, dtype):
    """Rows x [..., dim] (64 bits, values of `dtype`) -> codes, scale, low."""
    low, high = x.amin(-1), x.amax(-1)
    scale = _nearest((high - low) / 15.0, dtype)
    code = torch.round((x - low[..., None]) / scale[..., None]).clamp(0, 15)
    code = torch.where(scale[..., None] > 0, code, torch.zeros_like(code))
    return code, scale, low


def _plain_append(s):
    case, dtype = s["case"], TYPES[s["case"]["dtype"]]
    block = case["block"]
    live = s["seq"] >= 0
    position = s["pos"].long()
    cos, sin = s["cos"][position], s["sin"][position]
    page = s["table"][s["seq"].clamp(min=0).long(), position // block].long()[live]
    slot = (position % block)[live]
    new = {"q": _rotated(s["q"].double(), cos, sin, case["rot"], case["interleaved"]),
           "k": _rotated(s["k"].double(), cos, sin, case["rot"], case["interleaved"]),
           "v": s["v"].double()}
    live_rows = live[:, None, None]
    s["q_out"].copy_(torch.where(live_rows, _nearest(new["q"], dtype), s["q_out"].double()))
    for side in ("k", "v"):
        rows = _nearest(new[side], dtype)
        if case["bits"] == 16:
            s[side + "_cache"][page, :, slot] = rows[live].to(dtype)
        else:
            code, scale, low = _four_bits(rows, dtype)
            code8 = code.to(torch.uint8)
            s[side + "_cache"][page, :, slot] = (code8[..., 0::2] | (code8[..., 1::2] << 4))[live]
            s[side + "_params"][page, :, slot] = torch.stack((scale, low), dim=-1)[live].to(dtype)
            rows = low[..., None] + code * scale[..., None]
            s[side + "_out"].copy_(torch.where(live_rows, rows, s[side + "_out"].double()))


def _plain_rows(s, side, z, length):
    """The cached rows of one sequence as 32-bit values [kv, length, dim]."""
    block = s["case"]["block"]
    pages = s["table"][z, :-(-length // block)].long()
    rows = s[side + "_cache"][pages].transpose(1, 2).flatten(0, 1)[:length]
    if s["case"]["bits"] == 4:
        params = s[side + "_params"][pages].transpose(1, 2).flatten(0, 1)[:length].float()
        codes = torch.stack((rows & 15, rows >> 4), dim=-1).flatten(-2).float()
        return (params[..., 1:] + codes * params[..., :1]).transpose(0, 1)
    return rows.float().transpose(0, 1)


def _plain_attend(s, q):
    case = s["case"]
    kv, dim, group = case["kv"], case["dim"], case["heads"] // case["kv"]
    for z, (start, count, length) in enumerate(s["spans"]):
        keys, values = _plain_rows(s, "k", z, length), _plain_rows(s, "v", z, length)
        rows = q[start:start + count].float().view(count, kv, group, dim).permute(1, 0, 2, 3)
        score = torch.matmul(rows.reshape(kv, count * group, dim), keys.transpose(1, 2)) / math.sqrt(dim)
        row = torch.arange(count * group, device=DEV) // group
        hidden = torch.arange(length, device=DEV)[None] > (length - count + row)[:, None]
        score = score.masked_fill(hidden[None], -math.inf)
        top = score.amax(-1, keepdim=True)
        weight = torch.exp(score - top)
        total = weight.sum(-1, keepdim=True)
        result = torch.matmul(weight, values) / total
        state = (top + torch.log(total)).view(kv, count, group)
        s["out"][start:start + count] = result.view(kv, count, group, dim).permute(1, 0, 2, 3).reshape(
            count, case["heads"], dim).to(s["out"].dtype)
        s["lse"][start:start + count] = state.permute(1, 0, 2).reshape(count, case["heads"])


def _plain_linear(s):
    x = s["x"].float()
    scale = x.abs().amax(-1) / 127.0
    code = torch.round(x.double() / scale.double()[:, None])
    code = torch.where(scale[:, None] > 0, code, torch.zeros_like(code))
    total = torch.matmul(code, s["w"].double().t())
    y = (total * scale.double()[:, None] * s["w_scale"].double()).float()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["act"] == "gelu_tanh":
        y = 0.5 * y * (1.0 + torch.tanh(0.79788456 * (y + 0.044715 * y * y * y)))
    s["y"].copy_(y)


def run(state):
    op = state["case"]["op"]
    if op == "linear":
        (_own_linear if own else _plain_linear)(state)
        return state["y"]
    if op == "attend":
        (_own_attend if own else _plain_attend)(state, state["q"])
        return {"out": state["out"], "lse": state["lse"]}
    (_own_append if own else _plain_append)(state)
    done = {"q": state["q_out"]}
    if state["case"]["bits"] == 4:   # codes as the values they stand for
        done["k"], done["v"] = state["k_out"], state["v_out"]
    if op == "append":
        done = {name: rows[:state["live"]] for name, rows in done.items()}
        if state["case"]["bits"] == 16:
            done["k_cache"], done["v_cache"] = state["k_cache"], state["v_cache"]
        return done
    (_own_attend if own else _plain_attend)(state, state["q_out"])
    return {"out": state["out"], "lse": state["lse"], **done}


# ------------------------------------------------------------------------------ the work of each
def work(case):
    if case["op"] == "linear":
        m, n, k = case["rows"], case["out"], case["in"]
        size = m * k * 2 + n * k + n * 4 + m * n * 2 + (n * 2 if case["bias"] else 0)
        return {"bytes": size, "flops": 2 * m * n * k}
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    row = dim * 2 if case["bits"] == 16 else dim // 2 + 4   # a cached row of one head
    size, flops = 0, 0
    if case["op"] != "attend":
        tokens = (sum(n for _, n in _prompt_spans(case)[0]) if case["op"] == "append"
                  else sum(_queries(case)))
        # q, k, v read; the rotated q and the cached rows (4 bits: their values too) written; angles
        size += tokens * (2 * heads * dim * 2 + 2 * kv * dim * 2 + 2 * kv * row + case["rot"] * 4 + 8)
        if case["bits"] == 4:
            size += tokens * 2 * kv * dim * 2
        flops += tokens * (heads + kv) * case["rot"] * 3
    if case["op"] != "append":
        lengths, counts = _lengths(case), _queries(case)
        size += sum(lengths) * kv * 2 * row + sum(counts) * heads * (2 * dim * 2 + 4)
        size += sum(-(-n // case["block"]) for n in lengths) * 4
        flops += sum(4 * c * heads * n * dim for c, n in zip(counts, lengths))
    return {"bytes": size, "flops": flops}


# --------------------------------------------------------------- the definitions, in 64 bits
def _cut(x, dtype):
    """Nearest value of a 16-bit type, ties to even, by the bits of the 64-bit number."""
    drop = 45 if dtype == torch.bfloat16 else 42
    bits = x.contiguous().view(torch.int64)
    kept = (bits + ((1 << (drop - 1)) - 1) + ((bits >> drop) & 1)) & ~((1 << drop) - 1)
    value = kept.view(torch.float64)
    if dtype == torch.float16:   # below 2^-14 the steps of float16 are 2^-24
        value = torch.where(x.abs() < 2.0 ** -14, torch.round(x * 2.0 ** 24) * 2.0 ** -24, value)
    return value


def _turn(s, name):
    """The rotation as a complex product."""
    case = s["case"]
    x, rot = s[name].double(), case["rot"]
    position = s["pos"].long()
    angle = torch.complex(s["cos"][position].double(), s["sin"][position].double())[:, None]
    head = x[..., :rot]
    if case["interleaved"]:
        pair = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous())
        turned = torch.view_as_real(pair * angle).reshape(head.shape)
    else:
        pair = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous())
        turned = torch.cat(((pair * angle).real, (pair * angle).imag), dim=-1)
    return torch.cat((turned, x[..., rot:]), dim=-1)


def _stands_for(rows, dtype):
    """The values that the 4-bit cache stands for after rows [..., dim] were put in."""
    rows = _cut(rows, dtype)
    low = rows.min(-1, keepdim=True).values
    scale = _cut((rows.max(-1, keepdim=True).values - low) / 15, dtype)
    code = torch.where(scale > 0, ((rows - low) / scale).round(), torch.zeros_like(rows)).clamp(0, 15)
    return low + scale * code


def _exact_append(s):
    case, dtype = s["case"], TYPES[s["case"]["dtype"]]
    rows = {"q": _turn(s, "q"), "k": _turn(s, "k"), "v": s["v"].double()}
    if case["bits"] == 4:
        rows["k"], rows["v"] = _stands_for(rows["k"], dtype), _stands_for(rows["v"], dtype)
    return rows


def _exact_attend(s, q, fresh):
    """Attention by one query token at a time; `fresh` replaces the appended rows."""
    case = s["case"]
    kv, block, group = case["kv"], case["block"], case["heads"] // case["kv"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device=DEV)
    for z, (start, count, length) in enumerate(s["spans"]):
        where = torch.arange(length, device=DEV)
        page, slot = s["table"][z][where // block].long(), where % block
        side = {}
        for name in ("k", "v"):
            rows = s[name + "_cache"][page, :, slot]
            if case["bits"] == 4:
                params = s[name + "_params"][page, :, slot].double()
                both = torch.empty((length, kv, case["dim"]), dtype=torch.float64, device=DEV)
                both[..., 0::2], both[..., 1::2] = rows % 16, rows // 16
                rows = both * params[..., 0:1] + params[..., 1:2]
            else:
                rows = rows.double()
            if fresh is not None:
                rows[length - count:] = fresh[name][start:start + count]
            side[name] = rows
        for i in range(count):
            seen = length - count + i + 1
            row = q[start + i].double().view(kv, group, -1)
            score = torch.einsum("hgd,nhd->hgn", row, side["k"][:seen]) * case["dim"] ** -0.5
            lse[start + i] = torch.logsumexp(score, -1).flatten()
            share = torch.softmax(score, -1)
            out[start + i] = torch.einsum("hgn,nhd->hgd", share, side["v"][:seen]).reshape(case["heads"], -1)
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    dtype = TYPES[case["dtype"]]
    if case["op"] == "linear":
        x = s["x"].double()
        scale = (x.abs().max(-1, keepdim=True).values.float() / 127).double()
        code = torch.where(scale > 0, (x / scale).round(), torch.zeros_like(x))
        y = (code @ s["w"].double().T) * scale * s["w_scale"].double()[None]
        if case["bias"]:
            y += s["bias"].double()
        if case["act"] == "gelu_tanh":
            y = y * torch.sigmoid(2 * 0.79788456 * (y + 0.044715 * y ** 3))
        return y
    if case["op"] == "attend":
        return _exact_attend(s, s["q"], None)
    rows = _exact_append(s)
    if case["op"] == "append":
        tail = s["live"]
        done = {name: x[:tail] for name, x in rows.items()}
        if case["bits"] == 16:
            page = s["table"][s["seq"][:tail].long(), s["pos"][:tail].long() // case["block"]].long()
            for name in ("k", "v"):
                cache = s[name + "_cache"].double()
                cache[page, :, s["pos"][:tail].long() % case["block"]] = done.pop(name)
                done[name + "_cache"] = cache
        return done
    # the attention of a step reads what the operators hand on: q and the 16-bit rows rounded
    fresh = rows if case["bits"] == 4 else {n: _cut(rows[n], dtype) for n in ("k", "v")}
    done = rows if case["bits"] == 4 else {"q": rows["q"]}
    return {**_exact_attend(s, _cut(rows["q"], dtype), fresh), **done}
