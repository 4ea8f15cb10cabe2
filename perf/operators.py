"""The operators around a paged key/value cache, as measurable cases: rotary embedding with the append to the cache (in 16 bits, or
quantised to 8 or 4 as it is written), reading the cache back, and attention of new tokens over it.

A case is a dict of plain values.  ``prepare`` makes what a serving program holds before the call, ``run`` is one call (in plain
torch operations, or, with ``own`` set, through ``mlxl3_b200.kv``), ``work`` what the call cannot do without, ``exact`` the result
from the definition in 64 bits.

The cache is a pool of pages, keys and values each [pages, kv_heads, page_size, head_dim]; token t of sequence b lies in row
t % page_size of page table[b, t // page_size].  Sequence b brings the rows row_start[b] .. row_start[b + 1] of the call, its last tokens:
row i of n is token length[b] - n + i.  8 and 4 bits: one 32-bit scale s = max|x| / m per vector (m = 127 or 7) and codes
round(x * m / max|x|); 4-bit codes are stored as code + 8, the even dimension in the low half of the byte.

Kinds:
  append     q and k rotated by their positions, q to a buffer of its own, k and v into the cache; a quantised cache is then read
             back, because what it holds is known by its values only
  read       rows of the sequences out of the cache
  attention  softmax(q k^T * scale) v of every new token over the tokens up to its own (with a window: the last `window` of them)
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
LIMIT = {8: 127, 4: 7}
BLOCK = 4096                                   # vectors of a pool that are made at a time


def listed():
    return [
        # the next token of one conversation: the projections' output into the cache
        {"name": "append-1token", "kind": "append", "dtype": "f16", "bits": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "batch": 1, "new_min": 1, "new_max": 1, "length_min": 2048, "length_max": 2048,
         "rotated": 128, "interleaved": False, "theta": 500000.0, "stretch": 1.0, "shape": 1},
        # one step of 64 conversations, bf16, half of each head rotated in neighbouring pairs, the cache in 8 bits
        {"name": "append-64seqs-8bit", "kind": "append", "dtype": "bf16", "bits": 8, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "batch": 64, "new_min": 1, "new_max": 1, "length_min": 200, "length_max": 9000,
         "rotated": 64, "interleaved": True, "theta": 10000.0, "stretch": 1.0, "shape": 2},
        # prompts of ragged length, one of them late in a long context with stretched frequencies
        {"name": "append-prompts", "kind": "append", "dtype": "f16", "bits": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "batch": 3, "new_min": 1500, "new_max": 4100, "length_min": 4100, "length_max": 100000,
         "rotated": 128, "interleaved": False, "theta": 500000.0, "stretch": 8.0, "shape": 3},
        # a prompt into a cache of 4 bits
        {"name": "append-prompt-4bit", "kind": "append", "dtype": "f16", "bits": 4, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "batch": 1, "new_min": 4000, "new_max": 4000, "length_min": 4000, "length_max": 4000,
         "rotated": 128, "interleaved": False, "theta": 500000.0, "stretch": 1.0, "shape": 4},
        # short ragged sequences taken out of an 8-bit cache for inspection
        {"name": "read-8bit", "kind": "read", "dtype": "f16", "out": "f32", "bits": 8, "heads": 16, "kv_heads": 4, "head_dim": 64, "page": 16,
         "batch": 5, "new_min": 37, "new_max": 700, "length_min": 700, "length_max": 2000, "shape": 5},
        # one long conversation taken out of a 4-bit cache, to be kept elsewhere
        {"name": "read-4bit-long", "kind": "read", "dtype": "bf16", "out": "bf16", "bits": 4, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 64, "batch": 1, "new_min": 60001, "new_max": 60001, "length_min": 60001, "length_max": 60001, "shape": 6},
        # decode of one token at the context of this repository's decoder
        {"name": "attention-1token", "kind": "attention", "dtype": "f16", "bits": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "batch": 1, "new_min": 1, "new_max": 1, "length_min": 2048, "length_max": 2048, "window": 0, "shape": 7},
        # one step of 64 conversations of ragged length in small pages
        {"name": "attention-64seqs", "kind": "attention", "dtype": "bf16", "bits": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "batch": 64, "new_min": 1, "new_max": 1, "length_min": 300, "length_max": 12000, "window": 0, "shape": 8},
        # long conversations in a 4-bit cache
        {"name": "attention-4bit-long", "kind": "attention", "dtype": "f16", "bits": 4, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "batch": 16, "new_min": 1, "new_max": 1, "length_min": 20000, "length_max": 60000, "window": 0, "shape": 9},
        # 16 draft tokens of each of eight conversations verified at once, five query heads to a key head, an 8-bit cache
        {"name": "attention-verify-8bit", "kind": "attention", "dtype": "bf16", "bits": 8, "heads": 40, "kv_heads": 8, "head_dim": 128,
         "page": 32, "batch": 8, "new_min": 16, "new_max": 16, "length_min": 1000, "length_max": 12000, "window": 0, "shape": 10},
        # a prompt read in one piece
        {"name": "attention-prompt", "kind": "attention", "dtype": "f16", "bits": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "batch": 1, "new_min": 4096, "new_max": 4096, "length_min": 4096, "length_max": 4096, "window": 0, "shape": 11},
        # a step that mixes chunks of prompts with single tokens: small heads, seven query heads to a key head, a sliding window
        {"name": "attention-mixed", "kind": "attention", "dtype": "bf16", "bits": 16, "heads": 28, "kv_heads": 4, "head_dim": 64, "page": 16,
         "batch": 24, "new_min": 1, "new_max": 700, "length_min": 700, "length_max": 9000, "window": 1024, "shape": 12},
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    """One more case of the same ranges that costs no more than the largest listed one."""
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("append", "read", "attention")}
    while True:
        kind = rng.choice(["append", "append", "read", "attention", "attention", "attention", "attention"])
        kv_heads = rng.choice([1, 2, 3, 4, 5, 8])
        case = {"kind": kind, "dtype": rng.choice(["f16", "bf16"]), "bits": rng.choice([16, 16, 8, 4]), "kv_heads": kv_heads,
                "heads": kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8]), "head_dim": rng.choice([64, 128, 128]),
                "page": rng.choice([16, 32, 64, 128, 24, 256]), "batch": _log_uniform(rng, 1, 64), "shape": rng.randrange(1 << 30)}
        if kind == "attention" and rng.random() < 0.4:
            case["new_min"] = case["new_max"] = 1
        else:
            case["new_min"], case["new_max"] = sorted(_log_uniform(rng, 1, 4096) for _ in range(2))
        case["length_min"], case["length_max"] = sorted(_log_uniform(rng, case["new_max"], 60000) for _ in range(2))
        if kind == "append":
            case["interleaved"] = rng.random() < 0.5
            case["rotated"] = rng.choice([case["head_dim"], case["head_dim"], case["head_dim"] // 2, 16, 48])
            case["theta"] = rng.choice([10000.0, 500000.0, 1000000.0])
            case["stretch"] = rng.choice([1.0, 1.0, 4.0, 8.0])
        elif kind == "read":
            case["out"] = rng.choice(["f16", "bf16", "f32"])
        else:
            case["window"] = rng.choice([0, 0, 0, 100, 1024, 4096])
        if _cost(case) <= most[kind]:
            return case


# ---- shapes ---------------------------------------------------------------------------------------------------------


def _shape(case):
    """(new tokens, length) of every sequence, spread over the case's ranges."""
    rng = random.Random(case["shape"])
    news = [_log_uniform(rng, case["new_min"], case["new_max"]) for _ in range(case["batch"])]
    lengths = [max(n, rng.randint(case["length_min"], case["length_max"])) for n in news]
    return news, lengths


def _vector_bytes(case):
    """Bytes of one head's vector in the cache, with its scale."""
    d, bits = case["head_dim"], case["bits"]
    return d * 2 if bits == 16 else d * bits // 8 + 4


def _visible(n, length, window):
    """(keys seen, summed over the n last tokens; keys that any of them sees)."""
    first = length - n
    if not window:
        return n * first + n * (n + 1) // 2, length
    return sum(min(first + i + 1, window) for i in range(n)), length - max(0, first - window + 1)


def work(case):
    news, lengths = _shape(case)
    rows, d, h, g = sum(news), case["head_dim"], case["heads"], case["kv_heads"]
    vector = _vector_bytes(case)
    if case["kind"] == "append":
        # q read and written, k and v read and written to the cache; read back where it is quantised
        moved = rows * (2 * h * d * 2 + 2 * g * d * 2 + 2 * g * vector)
        if case["bits"] != 16:
            moved += rows * 2 * g * (vector + 2 * d)
        return {"bytes": moved, "flops": rows * (h + g) * case["rotated"] * 3}
    if case["kind"] == "read":
        size = 4 if case["out"] == "f32" else 2
        return {"bytes": rows * 2 * g * (vector + size * d), "flops": rows * 2 * g * d}
    pairs = keys = 0
    for n, length in zip(news, lengths):
        a, b = _visible(n, length, case["window"])
        pairs, keys = pairs + a, keys + b
    return {"bytes": 2 * rows * h * d * 2 + keys * 2 * g * vector, "flops": 4 * pairs * h * d}


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.4e15


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _turns(case):
    """Turns per position of every rotated pair, in 64 bits: theta^(-2i/rotated) / 2 pi, divided by `stretch` for a longer context."""
    i = torch.arange(case["rotated"] // 2, dtype=torch.float64)
    return case["theta"] ** (-2.0 * i / case["rotated"]) / (2.0 * math.pi) / case["stretch"]


def _pool(case, pages, generator):
    """Keys or values of a whole pool: N(0, 1) in 16 bits, or their codes and scales."""
    d, bits = case["head_dim"], case["bits"]
    shape = (pages, case["kv_heads"], case["page"])
    if bits == 16:
        out = torch.empty(shape + (d,), dtype=DTYPES[case["dtype"]], device="cuda")
        for at in range(0, pages, BLOCK):
            out[at:at + BLOCK] = torch.randn(out[at:at + BLOCK].shape, device="cuda", generator=generator, dtype=out.dtype)
        return out, None
    out = torch.empty(shape + (d * bits // 8,), dtype=torch.int8 if bits == 8 else torch.uint8, device="cuda")
    limit = LIMIT[bits]
    for at in range(0, pages, BLOCK):
        x = torch.randn(out[at:at + BLOCK].shape[:3] + (d,), device="cuda", generator=generator, dtype=torch.float16)
        code = (x * (limit / 2.7)).round_().clamp_(-limit, limit).to(torch.int8)
        out[at:at + BLOCK] = code if bits == 8 else ((code[..., 0::2] + 8) | ((code[..., 1::2] + 8) << 4)).to(torch.uint8)
    scale = (torch.rand(shape, device="cuda", generator=generator) + 0.5) * (2.7 / limit)
    return out, scale


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    news, lengths = _shape(case)
    dtype, d = DTYPES[case["dtype"]], case["head_dim"]
    rows, page = sum(news), case["page"]
    counts = [-(-n // page) for n in lengths]
    # an append touches only the pages of its own tokens: the others exist in the table, not in the pool
    firsts = [(n - k) // page if case["kind"] == "append" else 0 for n, k in zip(lengths, news)]
    pages = sum(c - f for c, f in zip(counts, firsts)) + 3
    order = torch.randperm(pages, generator=generator, device="cuda").to(torch.int32)
    table = torch.zeros((case["batch"], max(counts)), dtype=torch.int32, device="cuda")
    at = 0
    for b, (c, f) in enumerate(zip(counts, firsts)):
        table[b, f:c] = order[at:at + c - f]
        at += c - f
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    state = {"case": case, "news": news, "lengths": lengths, "starts": starts, "table": table, "pages": pages,
             "row_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
             "length": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    # the place of every row's token: page and row of the page
    positions = torch.cat([torch.arange(n - k, n) for n, k in zip(lengths, news)]).cuda()
    sequence = torch.repeat_interleave(torch.arange(case["batch"]), torch.tensor(news)).cuda()
    state["positions"], state["sequence"] = positions, sequence
    state["k"], state["k_scale"] = _pool(case, pages, generator)
    state["v"], state["v_scale"] = _pool(case, pages, generator)

    def rows_of(heads, factor=1.0):
        return (torch.randn((rows, heads, d), device="cuda", generator=generator) * factor).to(dtype)
    if case["kind"] == "append":
        state["q"], state["new_k"], state["new_v"] = rows_of(case["heads"]), rows_of(case["kv_heads"], 1.5), rows_of(case["kv_heads"])
        state["turns"] = _turns(case).cuda()
        state["q_out"] = torch.empty_like(state["q"])
    elif case["kind"] == "attention":
        state["q"] = rows_of(case["heads"], 2.5)               # scores of a few units: attention that prefers some keys
        state["out"] = torch.empty_like(state["q"])
    if case["kind"] == "read" or (case["kind"] == "append" and case["bits"] != 16):
        kind = DTYPES[case.get("out", case["dtype"])]
        state["k_rows"] = torch.empty((rows, case["kv_heads"], d), dtype=kind, device="cuda")
        state["v_rows"] = torch.empty_like(state["k_rows"])
    if own:
        _handles(state)
    return state


# ---- the framework's calls --------------------------------------------------------------------------------------------


def _handles(state):
    import mlxl3_b200 as ex
    from mlxl3_b200 import kv
    ex.init(torch.cuda.current_device())
    case = state["case"]
    codes = {"f16": ex.F16, "bf16": ex.BF16, "f32": ex.F32}
    scales = [0 if s is None else s.data_ptr() for s in (state["k_scale"], state["v_scale"])]
    state["cache"] = kv.KvCache(state["pages"], case["page"], case["kv_heads"], case["head_dim"], codes[case["dtype"]], case["bits"],
                                state["k"].data_ptr(), state["v"].data_ptr(), *scales)
    state["batch"] = kv.KvBatch(state["row_start"].data_ptr(), state["length"].data_ptr(), state["table"].data_ptr(), case["batch"],
                                state["table"].shape[1], state["starts"][-1])
    state["out_code"] = codes[case.get("out", case["dtype"])]
    if case["kind"] == "append":
        state["rope"] = kv.Rope(state["turns"].data_ptr(), case["rotated"], case["interleaved"])
    elif case["kind"] == "attention":
        state["max_new"] = max(state["news"])
        state["workspace"] = kv.new_attention_workspace(state["cache"], state["batch"], case["heads"], state["max_new"])


def _run_own(state):
    import mlxl3_b200 as ex
    from mlxl3_b200 import kv
    case, cache, batch = state["case"], state["cache"], state["batch"]
    stream = ex.Stream(torch.cuda.current_stream().cuda_stream)
    if case["kind"] == "attention":
        kv.attention(cache, batch, state["q"].data_ptr(), case["heads"], case["head_dim"] ** -0.5, state["out"].data_ptr(), state["workspace"],
                     max_new=state["max_new"], window=case["window"], stream=stream)
        return state["out"]
    if case["kind"] == "append":
        kv.append(cache, batch, state["new_k"].data_ptr(), state["new_v"].data_ptr(), state["rope"], d_q=state["q"].data_ptr(),
                  heads=case["heads"], d_q_out=state["q_out"].data_ptr(), stream=stream)
        if case["bits"] == 16:
            return state["q_out"], state["k"], state["v"]
    kv.read(cache, batch, state["out_code"], state["k_rows"].data_ptr(), state["v_rows"].data_ptr(), stream=stream)
    if case["kind"] == "append":
        return state["q_out"], state["k_rows"], state["v_rows"]
    return state["k_rows"], state["v_rows"]


# ---- the plain form -----------------------------------------------------------------------------------------------------


def _rotate(x, cos, sin, interleaved):
    """Pairs of the first 2 * cos.shape[-1] dimensions turned: neighbours, or the two halves."""
    r = 2 * cos.shape[-1]
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2], out[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        out[..., :r // 2], out[..., r // 2:r] = a * cos - b * sin, a * sin + b * cos
    return out


def _quantise(x, bits):
    """Codes and scales of 64-bit vectors (a value next to the border between two codes decides which)."""
    m = LIMIT[bits]
    most = x.abs().amax(-1, keepdim=True)
    code = torch.where(most > 0, (x * m) / most, torch.zeros_like(x)).round().to(torch.int8)
    scale = (most / m).squeeze(-1).float()
    return (code if bits == 8 else ((code[..., 0::2] + 8) | ((code[..., 1::2] + 8) << 4)).to(torch.uint8)), scale


def _values(stored, scale, bits):
    """32-bit values of stored vectors."""
    if bits == 16:
        return stored.float()
    if bits == 4:
        stored = torch.stack(((stored & 15).to(torch.int8) - 8, (stored >> 4).to(torch.int8) - 8), -1).flatten(-2)
    return stored.float() * scale.unsqueeze(-1)


def _run_plain(state):
    case = state["case"]
    page, bits = case["page"], case["bits"]
    places = state["table"][state["sequence"], state["positions"] // page].long(), state["positions"] % page
    if case["kind"] == "append":
        turns = state["positions"].double().unsqueeze(-1) * state["turns"]
        angle = 2.0 * math.pi * (turns - turns.round())
        cos, sin = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)
        state["q_out"].copy_(_rotate(state["q"].float(), cos.float(), sin.float(), case["interleaved"]))
        if bits == 16:
            state["k"][places[0], :, places[1]] = _rotate(state["new_k"].float(), cos.float(), sin.float(), case["interleaved"]).to(state["k"].dtype)
            state["v"][places[0], :, places[1]] = state["new_v"]
            return state["q_out"], state["k"], state["v"]
        for name, x in (("k", _rotate(state["new_k"].double(), cos, sin, case["interleaved"])), ("v", state["new_v"].double())):
            code, scale = _quantise(x, bits)
            state[name][places[0], :, places[1]] = code
            state[name + "_scale"][places[0], :, places[1]] = scale
    if case["kind"] in ("append", "read"):
        for name in ("k", "v"):
            scale = None if bits == 16 else state[name + "_scale"][places[0], :, places[1]]
            state[name + "_rows"].copy_(_values(state[name][places[0], :, places[1]], scale, bits))
        held = (state["k_rows"], state["v_rows"])
        return (state["q_out"], *held) if case["kind"] == "append" else held
    g, d = case["kv_heads"], case["head_dim"]
    group = case["heads"] // g
    for b, (n, length) in enumerate(zip(state["news"], state["lengths"])):
        low = max(0, length - n - case["window"] + 1) if case["window"] else 0
        used = state["table"][b, low // page:-(-length // page)].long()
        skip = low - low // page * page

        def gathered(name):
            scale = None if bits == 16 else state[name + "_scale"][used]
            return _values(state[name][used], scale, bits).transpose(0, 1).reshape(g, -1, d)[:, skip:skip + length - low]
        keys, values = gathered("k"), gathered("v")
        rows = slice(state["starts"][b], state["starts"][b] + n)
        q = state["q"][rows].float().reshape(n, g, group, d).permute(1, 2, 0, 3).reshape(g, group * n, d)
        scores = torch.matmul(q, keys.transpose(1, 2)).mul_(d ** -0.5).reshape(g, group, n, -1)
        key = torch.arange(low, length, device="cuda")
        own_position = torch.arange(length - n, length, device="cuda").unsqueeze(-1)
        hidden = key > own_position
        if case["window"]:
            hidden |= key <= own_position - case["window"]
        scores.masked_fill_(hidden, -math.inf)
        scores -= scores.amax(-1, keepdim=True)
        scores.exp_()
        scores /= scores.sum(-1, keepdim=True)
        out = torch.matmul(scores.reshape(g, group * n, -1), values)
        state["out"][rows] = out.reshape(g, group, n, d).permute(2, 0, 1, 3).reshape(n, g * group, d).to(state["out"].dtype)
    return state["out"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------


def _stored(s, name):
    """What the rows of the call hold in the cache, [rows, kv_heads, head_dim] in 64 bits."""
    out = []
    for b, (n, length) in enumerate(zip(s["news"], s["lengths"])):
        out.append(_sequence(s, name, b, length - n, length).transpose(0, 1))
    return torch.cat(out)


def _sequence(s, name, b, low, high):
    """Keys or values low..high-1 of one sequence, [kv_heads, tokens, head_dim] in 64 bits."""
    case = s["case"]
    token = torch.arange(low, high, device="cuda")
    at, row = s["table"][b][token // case["page"]].long(), token % case["page"]
    pool = s[name].transpose(1, 2)                                         # [pages, page, kv_heads, ...]
    held = pool[at, row]
    if case["bits"] == 4:
        wide = torch.empty(held.shape[:-1] + (case["head_dim"],), dtype=torch.float64, device="cuda")
        wide[..., 0::2], wide[..., 1::2] = held % 16, held // 16
        held = wide - 8
    if case["bits"] != 16:
        held = held.double() * s[name + "_scale"].transpose(1, 2)[at, row].double()[..., None]
    return held.double().transpose(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    d, bits = case["head_dim"], case["bits"]
    if case["kind"] == "read":
        return _stored(s, "k"), _stored(s, "v")
    if case["kind"] == "append":
        r = case["rotated"]
        turned = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                             2 * math.pi * torch.remainder(s["positions"].double()[:, None] * s["turns"], 1.0))[:, None]

        def rotated(x):
            x = x.double()
            head = x[..., :r]
            if case["interleaved"]:
                pairs = torch.view_as_complex(head.unflatten(-1, (r // 2, 2)).contiguous()) * turned
                head = torch.view_as_real(pairs).flatten(-2)
            else:
                pairs = torch.complex(head[..., :r // 2].contiguous(), head[..., r // 2:].contiguous()) * turned
                head = torch.cat((pairs.real, pairs.imag), -1)
            return torch.cat((head, x[..., r:]), -1)
        q, k, v = rotated(s["q"]), rotated(s["new_k"]), s["new_v"].double()
        if bits == 16:
            out = []
            page = s["table"][s["sequence"], s["positions"] // case["page"]].long()
            for name, x in (("k", k), ("v", v)):
                pool = s[name].double().transpose(1, 2).contiguous()
                pool[page, s["positions"] % case["page"]] = x
                out.append(pool.transpose(1, 2).contiguous())
            return q, *out
        m = LIMIT[bits]
        held = []
        for x in (k, v):
            top = x.abs().max(-1, keepdim=True).values
            held.append(torch.round(x * m / top).nan_to_num(0.0) * (top / m).float().double())
        return q, *held
    group = case["heads"] // case["kv_heads"]
    result = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (n, length) in enumerate(zip(s["news"], s["lengths"])):
        low = max(0, length - n + 1 - case["window"]) if case["window"] else 0
        keys, values = _sequence(s, "k", b, low, length), _sequence(s, "v", b, low, length)
        at = torch.arange(low, length, device="cuda")
        for first in range(0, n, 512):
            last = min(n, first + 512)
            position = torch.arange(length - n + first, length - n + last, device="cuda")[:, None]
            seen = (at <= position) & ((at > position - case["window"]) if case["window"] else True)
            rows = slice(s["starts"][b] + first, s["starts"][b] + last)
            for h in range(case["heads"]):
                score = (s["q"][rows, h].double() @ keys[h // group].T / math.sqrt(d)).where(seen, -math.inf)
                result[rows, h] = torch.softmax(score, -1) @ values[h // group]
    return result
