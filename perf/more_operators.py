"""More operators of a server that answers many requests from one GPU: their plain forms, and the calls
that a program makes of them.

A case is a plain dict; `listed()` gives the named ones and `draw()` more of the same ranges. The
operators:

append8     rotary positions of q and k, and k and v into their slots of a paged cache of 8-bit values with
            a scale per row and kv head (muyo_paged_rope_append_q8kv)
attention8  attention of one new token per sequence over such a cache (muyo_paged_attention_decode_q8kv)
prefix      attention of one new token per sequence, all of which go on from the same first keys, over a
            paged fp16 cache (muyo_paged_attention_prefix_f16kv)
sample      the next token of each row of logits by its own temperature, top-k, top-p and min-p, from
            given random numbers (muyo_sample_rows_f32)

Head layouts, widths and vocabularies are those of the two configurations that the binding names
(QWEN25_05B, QWEN25_7B).
"""
import math
import random

import torch

own = False  # False: the plain forms below; True: the library's entry points

MODELS = {
    "0.5b": dict(heads=14, kv_heads=2, head_dim=64, vocab=151936),
    "7b": dict(heads=28, kv_heads=4, head_dim=128, vocab=152064),
}
ROPE_BASE = 1e6
HALF, INTERLEAVED = 0, 1
INT8, E4M3 = 0, 1
LARGEST = {INT8: 127.0, E4M3: 448.0}


def listed():
    return [
        # One chat's token: a layer's rope and append, all latency.
        dict(name="append8_token", kind="append8", model="0.5b", tokens=1, position=301, page_size=16, pages=256,
             format=INT8, layout=HALF, rotary=64, scaling="none", stacked=True),
        # A decode step of many long chats, positions scaled past the trained context.
        dict(name="append8_step", kind="append8", model="7b", tokens=253, position=100003, page_size=64, pages=1024,
             format=E4M3, layout=HALF, rotary=128, scaling="yarn", stacked=True),
        # Prompts of several requests in one pass, half of each head rotated, pairs side by side.
        dict(name="append8_prompts", kind="append8", model="7b", tokens=8191, position=0, page_size=16, pages=2048,
             format=INT8, layout=INTERLEAVED, rotary=64, scaling="linear", stacked=False),
        # One chat, the first tokens of an answer.
        dict(name="attention8_short", kind="attention8", model="0.5b", queries=1, keys=302, spread="same",
             page_size=16, window=0, format=INT8),
        # One chat late in a long document.
        dict(name="attention8_long", kind="attention8", model="7b", queries=1, keys=32749, spread="same",
             page_size=64, window=0, format=E4M3),
        # A server's step: chats of all lengths side by side.
        dict(name="attention8_ragged", kind="attention8", model="7b", queries=64, keys=16384, spread="even",
             page_size=16, window=0, format=INT8),
        # A few chats after a system prompt.
        dict(name="prefix_few", kind="prefix", model="0.5b", queries=3, prefix=1009, keys=100, spread="even",
             page_size=16),
        # A server's step: chats of all lengths about one document.
        dict(name="prefix_chats", kind="prefix", model="7b", queries=64, prefix=8190, keys=2000, spread="log",
             page_size=16),
        # Many answers to one long prompt.
        dict(name="prefix_answers", kind="prefix", model="7b", queries=250, prefix=16381, keys=500, spread="even",
             page_size=64),
        # One chat's next token, with a chat's usual settings.
        dict(name="sample_token", kind="sample", vocab=151936, rows=1, settings="chat", masked=0.0),
        # A batch's step: every request has settings of its own.
        dict(name="sample_step", kind="sample", vocab=152064, rows=61, settings="mixed", masked=0.0),
        # Many answers to one prompt, drawn from most of the distribution.
        dict(name="sample_answers", kind="sample", vocab=151936, rows=500, settings="nucleus", masked=0.0),
    ]


def _log_int(rng, low, high):
    """An integer of [low, high], spread over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["append8", "attention8", "prefix", "sample"])
    page_size = rng.choice([16, 32, 64, 128])
    model = rng.choice(["0.5b", "7b"])
    if kind == "append8":
        tokens = _log_int(rng, 1, 8191)
        rotary = rng.choice([64, 32, 24, 20]) if model == "0.5b" else rng.choice([128, 96, 64, 36])
        return dict(kind=kind, model=model, tokens=tokens, position=rng.choice([0, _log_int(rng, 1, 200000)]),
                    page_size=page_size, pages=max(64, 2 * tokens // page_size + rng.randint(1, 100)),
                    format=rng.choice([INT8, E4M3]), layout=rng.choice([HALF, INTERLEAVED]), rotary=rotary,
                    scaling=rng.choice(["none", "linear", "yarn"]), stacked=rng.random() < 0.5)
    if kind == "attention8":
        keys = _log_int(rng, 1, 32768)
        return dict(kind=kind, model=model, queries=_log_int(rng, 1, max(1, min(256, 500000 // keys))), keys=keys,
                    spread=rng.choice(["same", "even", "log"]), page_size=page_size,
                    window=rng.choice([0, 0, _log_int(rng, 1, 4096)]), format=rng.choice([INT8, E4M3]))
    if kind == "prefix":
        queries, keys = _log_int(rng, 1, 250), _log_int(rng, 1, 2000)
        return dict(kind=kind, model=model, queries=queries, prefix=_log_int(rng, 16, 16384), keys=keys,
                    spread=rng.choice(["same", "even", "log"]) if queries * keys < 125000 else "log",
                    page_size=page_size)
    return dict(kind=kind, vocab=rng.choice([151936, 152064, _log_int(rng, 1000, 152064)]), rows=_log_int(rng, 1, 450),
                settings=rng.choice(["chat", "mixed", "nucleus", "plain"]), masked=rng.choice([0.0, 0.0, 0.9]))


# --------------------------------------------------------------------------------------------
# Inputs: everything from the seed alone, made on the GPU.

def _generator(seed, what):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + what * 7919 + 29) % (1 << 60))


def _rand(seed, what, shape, std=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=_generator(seed, what), device="cuda").mul_(std).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(count, page_size):
    return -(-count // page_size)


def _key_counts(case):
    """Keys in the cache of each query's own sequence, the new token's included."""
    n, keys = case["queries"], case["keys"]
    if case["spread"] == "same":
        return [keys] * n
    if case["spread"] == "even":
        return [1 + int((i + 0.5) / n * (keys - 1)) for i in range(n)]
    return [max(1, min(keys, int(keys ** ((i + 0.5) / n)))) for i in range(n)]


def _settings(case):
    """(temperature, top_k, top_p, min_p) of each row; top_k 0, top_p 1 and min_p 0 are off."""
    chat, nucleus, plain = (0.7, 40, 0.95, 0.0), (1.0, 0, 0.95, 0.0), (1.0, 0, 1.0, 0.0)
    kinds = {
        "chat": [chat],
        "nucleus": [nucleus, (0.8, 0, 0.9, 0.0), nucleus, (1.2, 0, 0.98, 0.01)],
        "plain": [plain, (1.5, 0, 1.0, 0.0)],
        "mixed": [chat, nucleus, (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.05), plain, (0.6, 20, 0.95, 0.0),
                  (1.3, 1000, 0.99, 0.001), (0.9, 1, 1.0, 0.0), (1.0, 30000, 1.0, 0.0)],
    }[case["settings"]]
    return [kinds[r % len(kinds)] for r in range(case["rows"])]


def _turns(case):
    """Turns per position of each rotated pair, and the factor on the rotated values: the positions
    as they are, interpolated, or YaRN's blend of the two by wavelength (its ramp from 32 to 1 turns in
    a trained context of 32768, stretched fourfold)."""
    rotary = case["rotary"]
    j = torch.arange(rotary // 2, dtype=torch.float64)
    turns = torch.pow(torch.tensor(ROPE_BASE, dtype=torch.float64), -2.0 * j / rotary) / (2 * math.pi)
    if case["scaling"] == "linear":
        return turns / 4.0, 1.0
    if case["scaling"] == "yarn":
        def pair(turning):
            return rotary * math.log(32768 / (turning * 2 * math.pi)) / (2 * math.log(ROPE_BASE))

        low, high = max(0.0, math.floor(pair(32))), min(rotary - 1.0, math.ceil(pair(1)))
        keep = 1.0 - ((j - low) / max(0.001, high - low)).clamp(0.0, 1.0)
        return turns * keep + turns / 4.0 * (1.0 - keep), 1.138629436111989  # 1 + ln(4) / 10
    return turns, 1.0


CODE_TYPE = {INT8: torch.int8, E4M3: torch.float8_e4m3fn}


def _codes(seed, what, shape, form):
    """A cache row's values in units of its scale: normal ones, the largest near the end of the type."""
    x = _rand(seed, what, shape, LARGEST[form] / 3.2).clamp_(-LARGEST[form], LARGEST[form])
    return x.round_().to(torch.int8) if form == INT8 else x.to(torch.float8_e4m3fn)


def _scales(seed, what, shape, form):
    """Rows of values of about one, some larger than others."""
    x = torch.randn(shape, generator=_generator(seed, what), device="cuda")
    return x.mul_(0.25).exp_().mul_(3.2 / LARGEST[form])


def prepare(case, seed):
    kind = case["kind"]
    s = dict(case, kind=kind)
    order = random.Random(seed * 31 + 11)
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = _rand(seed, 1, (rows, vocab), 2.5)
        # A few tokens stand out of each row, by more or less.
        likely = torch.randint(0, vocab, (rows, 24), generator=_generator(seed, 2), device="cuda")
        logits.scatter_add_(1, likely, _rand(seed, 3, (rows, 24), 4.0) + 9.0)
        if case["masked"]:  # a grammar that allows few of the tokens next
            drop = torch.rand((rows, vocab), generator=_generator(seed, 4), device="cuda") < case["masked"]
            logits.masked_fill_(drop, -math.inf)
        settings = _settings(case)
        order.shuffle(settings)
        column = list(zip(*settings))
        s.update(logits=logits, temperature=torch.tensor(column[0], device="cuda"), top_k=_ints(column[1]),
                 top_p=torch.tensor(column[2], device="cuda"), min_p=torch.tensor(column[3], device="cuda"),
                 random=torch.rand(rows, generator=_generator(seed, 5), device="cuda", dtype=torch.float64),
                 tokens=torch.empty(rows, dtype=torch.int32, device="cuda"), logprobs=torch.empty(rows, device="cuda"))
        return s
    m = MODELS[case["model"]]
    heads, kv, hd, size = m["heads"], m["kv_heads"], m["head_dim"], case["page_size"]
    s.update(heads=heads, kv_heads=kv, head_dim=hd, scale=1.0 / math.sqrt(hd))
    if kind == "append8":
        tokens, pages, form = case["tokens"], case["pages"], case["format"]
        qdim, kdim = heads * hd, kv * hd
        width = qdim + 2 * kdim
        qkv = _rand(seed, 1, (tokens, width))
        parts = torch.split(qkv, [qdim, kdim, kdim], 1)
        if not case["stacked"]:
            parts = [p.contiguous() for p in parts]
        turns, magnitude = _turns(case)
        step = torch.arange(tokens, device="cuda")
        positions = case["position"] + (step if case["position"] == 0 else -(step * 97) % (case["position"] + 1))
        slots = torch.randperm(pages * size, generator=_generator(seed, 2), device="cuda")[:tokens]
        s.update(q=parts[0], k=parts[1], v=parts[2], magnitude=float(torch.tensor(magnitude, dtype=torch.float32)),
                 turns=turns.cuda(), positions=positions.to(torch.int32), slots=slots.to(torch.int32),
                 q_out=torch.empty((tokens, heads, hd), device="cuda"),
                 kcache=_codes(seed, 3, (pages, kv, size, hd), form), kscales=_scales(seed, 4, (pages, kv, size), form),
                 vcache=_codes(seed, 5, (pages, kv, size, hd), form), vscales=_scales(seed, 6, (pages, kv, size), form))
        return s
    keys = _key_counts(case)
    order.shuffle(keys)
    held = list(keys)
    if kind == "prefix":
        held.append(case["prefix"])  # a sequence like the others
    counts = [_pages(n, size) for n in held]
    pages, width = sum(counts), max(counts)
    ids = torch.randperm(pages, generator=_generator(seed, 1), device="cuda").to(torch.int32)
    have = _ints(counts)
    column = torch.arange(width, device="cuda")
    first = torch.cumsum(have, 0) - have
    table = torch.where(column < have[:, None], ids[(first[:, None] + column).clamp(max=pages - 1)], -1)
    rows = list(range(len(keys)))
    order.shuffle(rows)  # the batch's order is not the tables'
    s.update(q=_rand(seed, 2, (len(keys), heads, hd), 2.0), tables=table.to(torch.int32).contiguous(), pages=pages,
             width=width, sequence=_ints(rows), positions=_ints([keys[r] - 1 for r in rows]), longest=max(keys),
             out=torch.empty((len(keys), heads, hd), device="cuda"))
    if kind == "prefix":
        s.update(shared=_ints([len(keys), case["prefix"]]),
                 kcache=_rand(seed, 3, (pages, kv, size, hd), dtype=torch.float16),
                 vcache=_rand(seed, 4, (pages, kv, size, hd), dtype=torch.float16))
        return s
    form = case["format"]
    s.update(kcache=_codes(seed, 3, (pages, kv, size, hd), form), kscales=_scales(seed, 4, (pages, kv, size), form),
             vcache=_codes(seed, 5, (pages, kv, size, hd), form), vscales=_scales(seed, 6, (pages, kv, size), form))
    return s


# --------------------------------------------------------------------------------------------
# One pass.

def run(s):
    kind = s["kind"]
    if own:
        return {"append8": _own_append, "attention8": _own_attention, "prefix": _own_prefix,
                "sample": _own_sample}[kind](s)
    return {"append8": _plain_append, "attention8": _plain_attention, "prefix": _plain_prefix,
            "sample": _plain_sample}[kind](s)


def _plain_rotate(x, cos, sin, layout, rotary):
    """x [tokens][heads][head_dim], its first `rotary` values rotated in pairs."""
    turned, rest = x[..., :rotary], x[..., rotary:]
    if layout == HALF:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_quantise(y, form):
    """Codes and scales of rows y in 64 bits: a value next to a border between two codes is not moved over it."""
    scales = (y.abs().amax(-1) / LARGEST[form]).float()
    scaled = y / scales.double()[..., None]
    if form == INT8:
        return scaled.round().clamp(-127, 127).to(torch.int8), scales
    # Steps of an eighth of the value's power of two, of 2^-9 below 2^-6; what is rounded is then exact in the type.
    step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))) - 3)
    return ((scaled / step).round() * step).clamp(-448, 448).to(torch.float32).to(torch.float8_e4m3fn), scales


def _plain_append(s):
    tokens, hd, size, layout, rotary = s["tokens"], s["head_dim"], s["page_size"], s["layout"], s["rotary"]
    turn = torch.frac(s["positions"].double()[:, None, None] * s["turns"]) * (2 * math.pi)
    cos, sin = turn.cos() * s["magnitude"], turn.sin() * s["magnitude"]
    q = _plain_rotate(s["q"].reshape(tokens, s["heads"], hd), cos.float(), sin.float(), layout, rotary)
    k = _plain_rotate(s["k"].reshape(tokens, s["kv_heads"], hd).double(), cos, sin, layout, rotary)
    v = s["v"].reshape(tokens, s["kv_heads"], hd).double()
    slots = s["slots"].long()
    at = slots // size, slice(None), slots % size
    for y, cache, scales in ((k, s["kcache"], s["kscales"]), (v, s["vcache"], s["vscales"])):
        codes, scale = _plain_quantise(y, s["format"])
        cache.view(torch.int8)[at] = codes.view(torch.int8)
        scales[at] = scale
    return dict(q=q, kcache=s["kcache"], vcache=s["vcache"], kscales=s["kscales"], vscales=s["vscales"])


def _rows(cache, scales, pages, form):
    """The rows of pages [...][n] as f32 [...][kv_heads][n * page_size][head_dim]."""
    rows = cache.view(torch.int8)[pages].view(CODE_TYPE[form]).float() * scales[pages][..., None]
    rows = rows.transpose(-4, -3)
    return rows.reshape(*rows.shape[:-3], -1, rows.shape[-1])


def _plain_attention(s):
    queries, heads, kv, hd, size = s["queries"], s["heads"], s["kv_heads"], s["head_dim"], s["page_size"]
    pages = s["tables"][s["sequence"].long()].long().clamp(min=0)
    k = _rows(s["kcache"], s["kscales"], pages, s["format"])
    q = s["q"].reshape(queries, kv, heads // kv, hd).transpose(2, 3).contiguous()
    scores = (k @ q) * s["scale"]
    del k
    at, last = torch.arange(scores.shape[2], device="cuda"), s["positions"][:, None]
    seen = at <= last
    if s["window"]:
        seen = seen & (at > last - s["window"])
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    weights = torch.exp(scores - scores.amax(2, keepdim=True))
    total = weights.sum(2).unsqueeze(-1)
    v = _rows(s["vcache"], s["vscales"], pages, s["format"])
    out = weights.transpose(2, 3).contiguous() @ v / total
    return out.reshape(queries, heads, hd)


def _plain_prefix(s):
    queries, heads, kv, hd, size = s["queries"], s["heads"], s["kv_heads"], s["head_dim"], s["page_size"]
    group, prefix = heads // kv, s["prefix"]
    first = s["tables"][s["shared"][0].long()].long()[:_pages(prefix, size)]
    own_pages = s["tables"][s["sequence"].long(), :_pages(s["longest"], size)].long().clamp(min=0)

    def rows(cache, pages):
        x = cache[pages].float().transpose(-4, -3)
        return x.reshape(*x.shape[:-3], -1, hd)

    q = s["q"].reshape(queries, kv, group, hd)
    together = q.transpose(0, 1).reshape(kv, queries * group, hd)
    k = rows(s["kcache"], first)[:, :prefix].transpose(1, 2).contiguous()
    shared = ((together @ k) * s["scale"]).reshape(kv, queries, group, prefix)
    mine = (q @ rows(s["kcache"], own_pages).transpose(2, 3).contiguous()) * s["scale"]  # [queries][kv][group][keys]
    seen = torch.arange(mine.shape[3], device="cuda") <= s["positions"][:, None]
    mine = mine.masked_fill(~seen[:, None, None, :], -math.inf)
    top = torch.maximum(shared.amax(3).transpose(0, 1), mine.amax(3))
    shared = torch.exp(shared - top.transpose(0, 1)[..., None])
    mine = torch.exp(mine - top[..., None])
    total = shared.sum(3).transpose(0, 1) + mine.sum(3)
    out = shared.reshape(kv, queries * group, prefix) @ rows(s["vcache"], first)[:, :prefix].contiguous()
    out = out.reshape(kv, queries, group, hd).transpose(0, 1) + mine @ rows(s["vcache"], own_pages)
    return (out / total[..., None]).reshape(queries, heads, hd)


def _plain_sample(s):
    x, vocab = s["logits"], s["vocab"]
    greedy = s["temperature"] <= 0
    heat = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    value, index = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits stay in the order of their index
    # Weights and their sums in 64 bits: a random number next to a border between two tokens is not moved over it.
    weight = torch.exp((value.double() - value[:, :1].double()) / heat)
    mass = torch.cumsum(weight, 1)
    k = torch.where(greedy, 1, torch.where(s["top_k"] > 0, s["top_k"], vocab)).long().clamp(max=vocab)[:, None]
    whole = mass.gather(1, k - 1)
    p = s["top_p"].double()[:, None]
    kept = torch.arange(vocab, device="cuda") < k
    kept &= (mass - weight < p * whole) | (p >= 1)
    kept &= weight >= s["min_p"].double()[:, None]
    kept[:, 0] = True
    weight = torch.where(kept, weight, 0.0)
    weight = torch.zeros_like(weight).scatter_(1, index, weight)  # by rising index
    mass = torch.cumsum(weight, 1)
    total = mass[:, -1:]
    last = (torch.arange(vocab, device="cuda") * (weight > 0)).amax(1)
    token = torch.minimum((mass <= s["random"][:, None] * total).sum(1), last)
    logprobs = torch.log(weight.gather(1, token[:, None]) / total)[:, 0]
    return dict(tokens=token.int(), logprobs=logprobs.float())


# The library, in its own terms.

_library = None


def _load():
    global _library
    if _library is None:
        import os
        import sys

        sys.path.insert(0, os.path.join(os.getcwd(), "muyo-llm_amd"))
        import muyo_hip

        _library = muyo_hip, muyo_hip.load()
    return _library


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _space(s, size):
    """The workspace that a program keeps beside its buffers."""
    s["space"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    return s["space"]


def _own_append(s):
    mh, lib = _load()
    mh.check(lib.muyo_paged_rope_append_q8kv(
        s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["q"].stride(0), s["k"].stride(0), s["v"].stride(0),
        s["q_out"].data_ptr(), s["kcache"].data_ptr(), s["vcache"].data_ptr(), s["kscales"].data_ptr(),
        s["vscales"].data_ptr(), s["positions"].data_ptr(), s["slots"].data_ptr(), s["tokens"], s["heads"],
        s["kv_heads"], s["head_dim"], s["pages"], s["page_size"], s["format"], s["layout"], s["rotary"],
        s["turns"].data_ptr(), s["magnitude"], _stream()))
    return dict(q=s["q_out"], kcache=s["kcache"], vcache=s["vcache"], kscales=s["kscales"], vscales=s["vscales"])


def _own_attention(s):
    mh, lib = _load()
    space = s.get("space")
    if space is None:
        space = _space(s, lib.muyo_paged_attention_decode_q8kv_workspace_bytes(s["queries"], s["heads"],
                                                                               s["kv_heads"], s["head_dim"]))
    mh.check(lib.muyo_paged_attention_decode_q8kv(
        s["q"].data_ptr(), s["kcache"].data_ptr(), s["vcache"].data_ptr(), s["kscales"].data_ptr(),
        s["vscales"].data_ptr(), s["out"].data_ptr(), s["tables"].data_ptr(), s["queries"], s["width"],
        s["sequence"].data_ptr(), s["positions"].data_ptr(), s["queries"], s["heads"], s["kv_heads"], s["head_dim"],
        s["pages"], s["page_size"], s["format"], s["window"], s["scale"], space.data_ptr(), space.numel(), _stream()))
    return s["out"]


def _own_prefix(s):
    mh, lib = _load()
    space = s.get("space")
    if space is None:
        space = _space(s, lib.muyo_paged_attention_prefix_f16kv_workspace_bytes(s["queries"], s["heads"],
                                                                                s["kv_heads"], s["head_dim"]))
    mh.check(lib.muyo_paged_attention_prefix_f16kv(
        s["q"].data_ptr(), s["kcache"].data_ptr(), s["vcache"].data_ptr(), s["out"].data_ptr(),
        s["tables"].data_ptr(), s["queries"] + 1, s["width"], s["sequence"].data_ptr(), s["positions"].data_ptr(),
        s["queries"], s["shared"].data_ptr(), s["heads"], s["kv_heads"], s["head_dim"], s["pages"], s["page_size"],
        s["scale"], space.data_ptr(), space.numel(), _stream()))
    return s["out"]


def _own_sample(s):
    mh, lib = _load()
    space = s.get("space")
    if space is None:
        space = _space(s, lib.muyo_sample_rows_workspace_bytes(s["rows"], s["vocab"]))
    mh.check(lib.muyo_sample_rows_f32(
        s["logits"].data_ptr(), s["vocab"], s["rows"], s["vocab"], s["temperature"].data_ptr(), s["top_k"].data_ptr(),
        s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["random"].data_ptr(), s["tokens"].data_ptr(),
        s["logprobs"].data_ptr(), space.data_ptr(), space.numel(), _stream()))
    return dict(tokens=s["tokens"], logprobs=s["logprobs"])


# --------------------------------------------------------------------------------------------
# What a pass cannot do without.

def work(case):
    kind = case["kind"]
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": 4 * rows * vocab + 32 * rows, "flops": 5 * rows * vocab}
    m = MODELS[case["model"]]
    heads, kv, hd = m["heads"], m["kv_heads"], m["head_dim"]
    if kind == "append8":
        return {"bytes": case["tokens"] * (8 * heads * hd + 8 * kv * hd + 2 * kv * (hd + 4) + 8),
                "flops": case["tokens"] * (case["rotary"] * 3 * (heads + kv) + 4 * kv * hd)}
    if kind == "attention8":
        keys = sum(min(n, case["window"] or n) for n in _key_counts(case))
        return {"bytes": 2 * kv * (hd + 4) * keys + 8 * heads * hd * case["queries"], "flops": 4 * heads * hd * keys}
    keys, queries = sum(_key_counts(case)), case["queries"]
    return {"bytes": 4 * kv * hd * (keys + case["prefix"]) + 8 * heads * hd * queries,
            "flops": 4 * heads * hd * (keys + queries * case["prefix"])}


# --------------------------------------------------------------------------------------------
# The same results in 64 bits.

def _e4m3_values():
    """What each byte stands for: sign, four bits of exponent, three of fraction."""
    values = []
    for byte in range(256):
        exponent, fraction = byte >> 3 & 15, byte & 7
        size = fraction * 2.0 ** -9 if exponent == 0 else (8 + fraction) * 2.0 ** (exponent - 10)
        values.append(math.nan if byte & 127 == 127 else -size if byte & 128 else size)
    return torch.tensor(values, dtype=torch.float64, device="cuda")


def _decoded(cache, form):
    return cache.double() if form == INT8 else _e4m3_values()[cache.view(torch.uint8).long()]


def _exact_append(case, s):
    half, tokens, form, size = case["rotary"] // 2, case["tokens"], case["format"], case["page_size"]
    heads, kv, hd = s["heads"], s["kv_heads"], s["head_dim"]
    if case["layout"] == HALF:
        first, second = torch.arange(half), torch.arange(half) + half
    else:
        first, second = 2 * torch.arange(half), 2 * torch.arange(half) + 1
    turn = torch.polar(torch.full((tokens, half), s["magnitude"], dtype=torch.float64, device="cuda"),
                       2 * math.pi * torch.frac(s["positions"].double()[:, None] * s["turns"]))[:, None]

    def rotated(x, count):
        x = x.double().reshape(tokens, count, hd).clone()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    out = dict(q=rotated(s["q"], heads))
    slots = s["slots"].long()
    at = slots // size, slice(None), slots % size
    for what, y in (("k", rotated(s["k"], kv)), ("v", s["v"].double().reshape(tokens, kv, hd))):
        scales = s[what + "scales"].double()
        scales[at] = y.abs().amax(-1) / LARGEST[form]
        codes = None  # whole numbers
        if form == E4M3:
            # Between the type's values: the number of midpoints below a size is the place of the nearest.
            values = _e4m3_values()[:127]
            scaled = y / scales[at].float().double()[..., None]
            nearest = values[torch.searchsorted((values[1:] + values[:-1]) / 2, scaled.abs().contiguous())]
            codes = _decoded(s[what + "cache"], form)
            codes[at] = torch.where(scaled < 0, -nearest, nearest)
        out[what + "cache"], out[what + "scales"] = codes, scales
    return {key: out[key] for key in ("q", "kcache", "vcache", "kscales", "vscales")}


def _exact_sample(case, s):
    out = []
    given = zip(s["temperature"].tolist(), s["top_k"].tolist(), s["top_p"].tolist(), s["min_p"].tolist(),
                s["random"].tolist())
    for row, (heat, top_k, top_p, min_p, u) in zip(s["logits"], given):
        if heat <= 0:
            out.append(torch.zeros((), dtype=torch.float64, device="cuda"))
            continue
        lp = torch.log_softmax(row.double() / heat, 0)
        fall = torch.sort(lp, descending=True).values
        count = min(top_k, fall.numel()) if top_k > 0 else fall.numel()
        mass = torch.cumsum(torch.softmax(fall[:count], 0), 0)
        if top_p < 1:
            count = min(count, 1 + int((mass < top_p).sum()))
        if min_p > 0:
            count = min(count, int((fall - fall[0] >= math.log(min_p)).sum()))
        count = max(count, 1)
        least = fall[count - 1]
        keep = lp > least
        ties = torch.nonzero(lp == least)[:count - int(keep.sum()), 0]
        keep[ties] = True
        lp = torch.log_softmax(torch.where(keep, lp, -math.inf), 0)
        at = torch.nonzero(keep)[:, 0]
        reached = torch.cumsum(lp[at].exp(), 0)
        token = at[min(int((reached <= u * reached[-1]).sum()), at.numel() - 1)]
        out.append(lp[token])
    return dict(tokens=None, logprobs=torch.stack(out))


def exact(case, seed):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind == "sample":
        return _exact_sample(case, s)
    if kind == "append8":
        return _exact_append(case, s)
    heads, kv, hd, size = s["heads"], s["kv_heads"], s["head_dim"], case["page_size"]
    prefix, window, tables = case.get("prefix", 0), case.get("window", 0), s["tables"].long()
    out = torch.empty((case["queries"], heads, hd), dtype=torch.float64, device="cuda")

    def keys_of(row, first, last):
        at = torch.arange(first, last, device="cuda")
        page = tables[row][at // size]
        found = []
        for what in "kv":
            x = s[what + "cache"].view(torch.int8 if kind == "attention8" else torch.float16)[page, :, at % size]
            if kind == "attention8":
                x = _decoded(x, case["format"]) * s[what + "scales"][page, :, at % size].double()[..., None]
            found.append(x.double())
        return found  # [keys][kv][hd] each

    if prefix:
        shared = keys_of(case["queries"], 0, prefix)
    for i, (row, last) in enumerate(zip(s["sequence"].tolist(), s["positions"].tolist())):
        k, v = keys_of(row, max(0, last + 1 - window) if window else 0, last + 1)
        if prefix:
            k, v = torch.cat([shared[0], k]), torch.cat([shared[1], v])
        for g in range(kv):
            q = s["q"][i].double().reshape(kv, heads // kv, hd)[g]
            scores = (k[:, g].contiguous() @ q.t().contiguous()) * s["scale"]
            out[i].reshape(kv, heads // kv, hd)[g] = torch.softmax(scores, 0).t().contiguous() @ v[:, g].contiguous()
    return out
