"""The operators of a server that answers many requests from one GPU: their plain forms, and the calls
that a program makes of them.

A case is a plain dict; `listed()` gives the named ones and `draw()` more of the same ranges. The
operators:

plan       pages for the sequences of a step: block tables, the ring of free pages, and each new
           token's sequence, position and slot (muyo_paged_plan)
append     rotary positions of q and k, and k and v into their slots of a paged fp16 cache
           (muyo_paged_rope_append_f16kv)
attention  attention of one new token per sequence over the pages (muyo_paged_attention_decode_f16kv)
logprobs   log probabilities of given tokens, their ranks, the entropy and the most likely tokens of
           each row of logits (muyo_token_logprobs_f32)

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


def listed():
    return [
        # Every decode step of a server: each sequence grows by one token.
        dict(name="plan_step", kind="plan", sequences=64, longest=2048, page_size=16, share_new=0.0, share_done=0.0,
             prompt=0, scarce=False),
        # A step that also ends some sequences and admits prompts: many tokens, pages both ways.
        dict(name="plan_prompts", kind="plan", sequences=256, longest=8192, page_size=16, share_new=0.25,
             share_done=0.1, prompt=4096, scarce=False),
        # One chat's token: a layer's rope and append, all latency.
        dict(name="append_token", kind="append", model="0.5b", tokens=1, position=301, page_size=16, pages=256,
             layout=HALF, rotary=64, scaling="none", stacked=True),
        # A decode step of many long chats, positions scaled past the trained context.
        dict(name="append_step", kind="append", model="7b", tokens=253, position=100003, page_size=64, pages=1024,
             layout=HALF, rotary=128, scaling="yarn", stacked=True),
        # Prompts of several requests in one pass, half of each head rotated, pairs side by side.
        dict(name="append_prompts", kind="append", model="7b", tokens=8191, position=0, page_size=16, pages=2048,
             layout=INTERLEAVED, rotary=64, scaling="linear", stacked=False),
        # One chat, the first tokens of an answer.
        dict(name="attention_short", kind="attention", model="0.5b", queries=1, keys=302, spread="same",
             page_size=16, window=0),
        # One chat late in a long document.
        dict(name="attention_long", kind="attention", model="7b", queries=1, keys=32749, spread="same",
             page_size=64, window=0),
        # A server's step: chats of all lengths side by side.
        dict(name="attention_ragged", kind="attention", model="7b", queries=64, keys=16384, spread="even",
             page_size=16, window=0),
        # Many short chats of the small model, each seeing its last 500 keys.
        dict(name="attention_window", kind="attention", model="0.5b", queries=250, keys=2048, spread="log",
             page_size=32, window=500),
        # The token that one chat has just sampled, with twenty alternatives.
        dict(name="logprobs_token", kind="logprobs", vocab=151936, rows=1, top=20),
        # The same of a batch of chats.
        dict(name="logprobs_step", kind="logprobs", vocab=152064, rows=61, top=5),
        # A scored prompt: every position's logits.
        dict(name="logprobs_prompt", kind="logprobs", vocab=151936, rows=1000, top=1),
    ]


def _log_int(rng, low, high):
    """An integer of [low, high], spread over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "append", "attention", "attention", "logprobs"])
    page_size = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        share = rng.choice([0.0, 0.1, 0.25])
        return dict(kind=kind, sequences=_log_int(rng, 1, 512), longest=_log_int(rng, 64, 8192), page_size=page_size,
                    share_new=share, share_done=rng.choice([0.0, 0.1]), prompt=_log_int(rng, 16, 2048) if share else 0,
                    scarce=rng.random() < 0.3)
    model = rng.choice(["0.5b", "7b"])
    if kind == "append":
        tokens = _log_int(rng, 1, 8191)
        rotary = rng.choice([64, 32, 24]) if model == "0.5b" else rng.choice([128, 96, 64, 32])
        return dict(kind=kind, model=model, tokens=tokens, position=rng.choice([0, _log_int(rng, 1, 200000)]),
                    page_size=page_size, pages=max(64, 2 * tokens // page_size + rng.randint(1, 100)),
                    layout=rng.choice([HALF, INTERLEAVED]), rotary=rotary,
                    scaling=rng.choice(["none", "linear", "yarn"]), stacked=rng.random() < 0.5)
    if kind == "attention":
        keys = _log_int(rng, 1, 32768)
        return dict(kind=kind, model=model, queries=_log_int(rng, 1, max(1, min(256, 500000 // keys))), keys=keys,
                    spread=rng.choice(["same", "even", "log"]), page_size=page_size,
                    window=rng.choice([0, 0, _log_int(rng, 1, 4096)]))
    return dict(kind=kind, vocab=rng.choice([151936, 152064, _log_int(rng, 1000, 152064)]), rows=_log_int(rng, 1, 900),
                top=rng.randint(0, 20))


# --------------------------------------------------------------------------------------------
# Inputs: everything from the seed alone, made on the GPU.

def _generator(seed, what):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + what * 7919 + 17) % (1 << 60))


def _rand(seed, what, shape, std=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=_generator(seed, what), device="cuda").mul_(std).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _requests(case):
    """(length, target) of a plan's sequences, before they are put into the seed's order."""
    n, pairs = case["sequences"], []
    new, done = round(case["share_new"] * n), round(case["share_done"] * n)
    for i in range(n):
        length = 1 + int((i + 0.5) / n * (case["longest"] - 1))
        if i < new:
            pairs.append((0, 1 + int((i + 0.5) / new * case["prompt"])))
        elif i < new + done:
            pairs.append((length, 0))
        else:
            pairs.append((length, length + 1))
    return pairs


def _pages(count, page_size):
    return -(-count // page_size)


def _key_counts(case):
    """Keys in the cache of each query's sequence, the new token's included."""
    n, keys = case["queries"], case["keys"]
    if case["spread"] == "same":
        return [keys] * n
    if case["spread"] == "even":
        return [1 + int((i + 0.5) / n * (keys - 1)) for i in range(n)]
    return [max(1, min(keys, int(keys ** ((i + 0.5) / n)))) for i in range(n)]


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
        return turns * keep + turns / 4.0 * (1.0 - keep), 1.0 + 0.1 * math.log(4.0)
    return turns, 1.0


def prepare(case, seed):
    kind = case["kind"]
    s = dict(case, kind=kind)
    order = random.Random(seed * 31 + 7)
    if kind == "plan":
        pairs = _requests(case)
        order.shuffle(pairs)
        size = case["page_size"]
        held = sum(_pages(a, size) for a, _ in pairs)
        needed = sum(max(0, _pages(b, size) - _pages(a, size)) for a, b in pairs)
        free = needed // 2 if case["scarce"] else needed + held // 8 + 1
        pages, width = held + free, _pages(max(max(a, b) for a, b in pairs), size)
        ids = torch.randperm(pages, generator=_generator(seed, 1), device="cuda").to(torch.int32)
        lengths = _ints([a for a, _ in pairs])
        have = -(-lengths // size)
        first = torch.cumsum(have, 0) - have
        column = torch.arange(width, device="cuda")
        table = torch.where(column < have[:, None], ids[(first[:, None] + column).clamp(max=pages - 1)], -1)
        head = order.randrange(pages)
        ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        ring[(head + torch.arange(free, device="cuda")) % pages] = ids[held:]
        tokens = sum(max(0, b - a) for a, b in pairs) + 5  # a step's lists have room to spare
        s.update(lengths=lengths, targets=_ints([b for _, b in pairs]), tables=table.to(torch.int32).contiguous(),
                 free_pages=ring, pool=_ints([head, free]), pages=pages, width=width, tokens=tokens,
                 granted=torch.empty(len(pairs), dtype=torch.int32, device="cuda"),
                 pool_out=torch.empty(2, dtype=torch.int32, device="cuda"),
                 starts=torch.empty(len(pairs) + 1, dtype=torch.int32, device="cuda"),
                 lists=[torch.empty(tokens, dtype=torch.int32, device="cuda") for _ in range(3)])
        return s
    if kind == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        logits = _rand(seed, 1, (rows, vocab), 3.0)
        given = torch.randint(0, vocab, (rows,), generator=_generator(seed, 2), device="cuda")
        # A sampled token stands out of its row more often than not.
        logits[torch.arange(rows, device="cuda"), given] += _rand(seed, 3, (rows,), 4.0) + 10.0
        s.update(logits=logits, tokens=given.to(torch.int32), logprobs=torch.empty(rows, device="cuda"),
                 entropy=torch.empty(rows, device="cuda"), ranks=torch.empty(rows, dtype=torch.int32, device="cuda"),
                 top_ids=torch.empty((rows, top), dtype=torch.int32, device="cuda"),
                 top_logprobs=torch.empty((rows, top), device="cuda"))
        return s
    m = MODELS[case["model"]]
    heads, kv, hd, size = m["heads"], m["kv_heads"], m["head_dim"], case["page_size"]
    s.update(heads=heads, kv_heads=kv, head_dim=hd, scale=1.0 / math.sqrt(hd))
    if kind == "append":
        tokens, pages = case["tokens"], case["pages"]
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
        s.update(q=parts[0], k=parts[1], v=parts[2], magnitude=magnitude, turns=turns.cuda(),
                 positions=positions.to(torch.int32), slots=slots.to(torch.int32),
                 q_out=torch.empty((tokens, heads, hd), device="cuda"),
                 kcache=_rand(seed, 3, (pages, kv, size, hd), dtype=torch.float16),
                 vcache=_rand(seed, 4, (pages, kv, size, hd), dtype=torch.float16))
        return s
    keys = _key_counts(case)
    order.shuffle(keys)
    counts = [_pages(n, size) for n in keys]
    pages, width = sum(counts), max(counts)
    ids = torch.randperm(pages, generator=_generator(seed, 1), device="cuda").to(torch.int32)
    have = _ints(counts)
    column = torch.arange(width, device="cuda")
    first = torch.cumsum(have, 0) - have
    table = torch.where(column < have[:, None], ids[(first[:, None] + column).clamp(max=pages - 1)], -1)
    rows = list(range(len(keys)))
    order.shuffle(rows)  # the batch's order is not the tables'
    s.update(q=_rand(seed, 2, (len(keys), heads, hd), 2.0), tables=table.to(torch.int32).contiguous(), pages=pages,
             width=width, sequence=_ints(rows), positions=_ints([keys[r] - 1 for r in rows]),
             kcache=_rand(seed, 3, (pages, kv, size, hd), dtype=torch.float16),
             vcache=_rand(seed, 4, (pages, kv, size, hd), dtype=torch.float16),
             out=torch.empty((len(keys), heads, hd), device="cuda"))
    return s


# --------------------------------------------------------------------------------------------
# One pass.

def run(s):
    kind = s["kind"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attention": _own_attention,
                "logprobs": _own_logprobs}[kind](s)
    return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention,
            "logprobs": _plain_logprobs}[kind](s)


def _plain_plan(s):
    size, pages, tokens = s["page_size"], s["pages"], s["tokens"]
    lengths, targets = s["lengths"].long(), s["targets"].long()
    head, free = s["pool"][0].long(), s["pool"][1].long()
    have, want = -(-lengths // size), -(-targets // size)
    new = (targets - lengths).clamp(min=0)
    fits = torch.cumsum(new, 0) <= tokens
    need = torch.where(fits, (want - have).clamp(min=0), 0)
    taken = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (taken <= free))
    granted = torch.where(ok, targets, lengths)
    new = torch.where(ok, new, 0)
    starts = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0))
    back = torch.where(ok, (have - want).clamp(min=0), 0)
    given = torch.cumsum(back, 0)
    column = torch.arange(s["width"], device="cuda")
    have, want = have[:, None], want[:, None]
    take = ok[:, None] & (column >= have) & (column < want)
    tables = torch.where(take, s["free_pages"][(head + (taken - need)[:, None] + column - have) % pages], s["tables"])
    # Pages given back go behind the ring's last; entries that are not go to a place past its end.
    leave = ok[:, None] & (column >= want) & (column < have)
    at = torch.where(leave, (head + free + (given - back)[:, None] + column - want) % pages, pages)
    ring = torch.cat([s["free_pages"], s["free_pages"][:1]]).scatter(0, at.flatten(), s["tables"].flatten())[:pages]
    used = torch.where(ok, need, 0).sum()
    pool = torch.stack([(head + used) % pages, free - used + back.sum()])
    token = torch.arange(tokens, device="cuda")
    sequence = torch.searchsorted(starts[1:], token, right=True)
    there = sequence < lengths.numel()
    sequence = sequence.clamp(max=lengths.numel() - 1)
    position = torch.where(there, token - starts[sequence] + lengths[sequence], 0)
    page = tables[sequence, position // size].long()
    slot = torch.where(there & (page >= 0) & (page < pages), page * size + position % size, -1)
    return dict(tables=tables, free_pages=ring, pool=pool.int(), granted=granted.int(), starts=starts.int(),
                sequence=torch.where(there, sequence, -1).int(), positions=torch.where(there, position, -1).int(),
                slots=slot.int())


def _plain_rotate(x, cos, sin, layout, rotary):
    """x [tokens][heads][head_dim], its first `rotary` values rotated in pairs."""
    turned, rest = x[..., :rotary], x[..., rotary:]
    if layout == HALF:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_append(s):
    tokens, hd, size, layout, rotary = s["tokens"], s["head_dim"], s["page_size"], s["layout"], s["rotary"]
    # Angles in 64 bits: a far position's turns are many, and only their fraction counts.
    angle = s["positions"].double()[:, None, None] * s["turns"] * (2 * math.pi)
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    q = _plain_rotate(s["q"].reshape(tokens, s["heads"], hd), cos, sin, layout, rotary)
    k = _plain_rotate(s["k"].reshape(tokens, s["kv_heads"], hd), cos, sin, layout, rotary)
    v = s["v"].reshape(tokens, s["kv_heads"], hd)
    slots = s["slots"].long()
    s["kcache"][slots // size, :, slots % size] = k.half()
    s["vcache"][slots // size, :, slots % size] = v.half()
    return dict(q=q, kcache=s["kcache"], vcache=s["vcache"])


def _plain_attention(s):
    queries, heads, kv, hd, size = s["queries"], s["heads"], s["kv_heads"], s["head_dim"], s["page_size"]
    group = heads // kv
    pages = s["tables"][s["sequence"].long()].long().clamp(min=0)
    keys = pages.shape[1] * size
    k = s["kcache"][pages].float().transpose(1, 2).reshape(queries, kv, keys, hd)
    q = s["q"].reshape(queries, kv, group, hd).transpose(2, 3).contiguous()
    scores = (k @ q) * s["scale"]
    del k
    at, last = torch.arange(keys, device="cuda"), s["positions"][:, None]
    seen = at <= last
    if s["window"]:
        seen = seen & (at > last - s["window"])
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    weights = torch.exp(scores - scores.amax(2, keepdim=True))
    total = weights.sum(2).unsqueeze(-1)
    v = s["vcache"][pages].float().transpose(1, 2).reshape(queries, kv, keys, hd)
    out = weights.transpose(2, 3).contiguous() @ v / total
    return out.reshape(queries, heads, hd)


def _plain_logprobs(s):
    x, vocab, top = s["logits"], s["vocab"], s["top"]
    shifted = x - x.amax(1, keepdim=True)
    weights = torch.exp(shifted)
    total = weights.sum(1)
    log_total = torch.log(total)
    entropy = log_total - (weights * shifted).sum(1) / total
    given = s["tokens"].long()[:, None]
    logprobs = shifted.gather(1, given)[:, 0] - log_total
    # One whole number a logit that orders them: the value, then the lower index.
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 20) - torch.arange(vocab, device="cuda")
    ranks = (order > order.gather(1, given)).sum(1)
    ids = torch.topk(order, top, 1).indices
    return dict(logprobs=logprobs, ranks=ranks.int(), entropy=entropy, top_ids=ids.int(),
                top_logprobs=shifted.gather(1, ids) - log_total[:, None])


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


def _own_plan(s):
    mh, lib = _load()
    sequence, positions, slots = s["lists"]
    mh.check(lib.muyo_paged_plan(s["lengths"].data_ptr(), s["targets"].data_ptr(), s["sequences"],
                                 s["tables"].data_ptr(), s["width"], s["free_pages"].data_ptr(), s["pool"].data_ptr(),
                                 s["pages"], s["page_size"], s["tokens"], s["granted"].data_ptr(),
                                 s["pool_out"].data_ptr(), s["starts"].data_ptr(), sequence.data_ptr(),
                                 positions.data_ptr(), slots.data_ptr(), _stream()))
    return dict(tables=s["tables"], free_pages=s["free_pages"], pool=s["pool_out"], granted=s["granted"],
                starts=s["starts"], sequence=sequence, positions=positions, slots=slots)


def _own_append(s):
    mh, lib = _load()
    mh.check(lib.muyo_paged_rope_append_f16kv(
        s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["q"].stride(0), s["k"].stride(0), s["v"].stride(0),
        s["q_out"].data_ptr(), s["kcache"].data_ptr(), s["vcache"].data_ptr(), s["positions"].data_ptr(),
        s["slots"].data_ptr(), s["tokens"], s["heads"], s["kv_heads"], s["head_dim"], s["pages"], s["page_size"],
        s["layout"], s["rotary"], s["turns"].data_ptr(), s["magnitude"], _stream()))
    return dict(q=s["q_out"], kcache=s["kcache"], vcache=s["vcache"])


def _space(s, size):
    """The workspace that a program keeps beside its buffers."""
    if "space" not in s:
        s["space"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    return s["space"]


def _own_attention(s):
    mh, lib = _load()
    space = s.get("space")
    if space is None:
        space = _space(s, lib.muyo_paged_attention_decode_f16kv_workspace_bytes(s["queries"], s["heads"],
                                                                                s["kv_heads"], s["head_dim"]))
    mh.check(lib.muyo_paged_attention_decode_f16kv(
        s["q"].data_ptr(), s["kcache"].data_ptr(), s["vcache"].data_ptr(), s["out"].data_ptr(),
        s["tables"].data_ptr(), s["queries"], s["width"], s["sequence"].data_ptr(), s["positions"].data_ptr(),
        s["queries"], s["heads"], s["kv_heads"], s["head_dim"], s["pages"], s["page_size"], s["window"], s["scale"],
        space.data_ptr(), space.numel(), _stream()))
    return s["out"]


def _own_logprobs(s):
    mh, lib = _load()
    space = s.get("space")
    if space is None:
        space = _space(s, lib.muyo_token_logprobs_workspace_bytes(s["rows"], s["vocab"], s["top"]))
    mh.check(lib.muyo_token_logprobs_f32(
        s["logits"].data_ptr(), s["vocab"], s["rows"], s["vocab"], s["tokens"].data_ptr(), s["logprobs"].data_ptr(),
        s["ranks"].data_ptr(), s["entropy"].data_ptr(), s["top"], s["top_ids"].data_ptr(),
        s["top_logprobs"].data_ptr(), space.data_ptr(), space.numel(), _stream()))
    return dict(logprobs=s["logprobs"], ranks=s["ranks"], entropy=s["entropy"], top_ids=s["top_ids"],
                top_logprobs=s["top_logprobs"])


# --------------------------------------------------------------------------------------------
# What a pass cannot do without.

def work(case):
    kind = case["kind"]
    if kind == "plan":
        pairs, size = _requests(case), case["page_size"]
        moved = sum(abs(_pages(b, size) - _pages(a, size)) for a, b in pairs)
        tokens = sum(max(0, b - a) for a, b in pairs)
        return {"bytes": 4 * (4 * len(pairs) + 2 * moved + 3 * tokens), "flops": 0}
    if kind == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": 4 * rows * (vocab + 4 + 2 * top), "flops": 5 * rows * vocab}
    m = MODELS[case["model"]]
    heads, kv, hd = m["heads"], m["kv_heads"], m["head_dim"]
    if kind == "append":
        return {"bytes": case["tokens"] * hd * (8 * heads + 8 * kv + 4 * kv) + 8 * case["tokens"],
                "flops": case["tokens"] * case["rotary"] * 3 * (heads + kv)}
    keys = sum(min(n, case["window"] or n) for n in _key_counts(case))
    return {"bytes": 4 * kv * hd * keys + 8 * heads * hd * case["queries"], "flops": 4 * heads * hd * keys}


# --------------------------------------------------------------------------------------------
# The same results in 64 bits.

def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if kind == "logprobs":
        out = dict(logprobs=[], ranks=None, entropy=[], top_ids=None, top_logprobs=[])
        for row, given in zip(s["logits"], s["tokens"].tolist()):
            x = row.double()
            lp = x - torch.logsumexp(x, 0)
            out["logprobs"].append(lp[given])
            out["entropy"].append(-(lp.exp() * lp).sum())
            out["top_logprobs"].append(torch.sort(lp, descending=True).values[:case["top"]])
        return {k: v if v is None else torch.stack(v) for k, v in out.items()}
    heads, kv, hd, size = s["heads"], s["kv_heads"], s["head_dim"], case["page_size"]
    if kind == "append":
        half, tokens = case["rotary"] // 2, case["tokens"]
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

        kcache, vcache, slots = s["kcache"].double(), s["vcache"].double(), s["slots"].long()
        kcache[slots // size, :, slots % size] = rotated(s["k"], kv)
        vcache[slots // size, :, slots % size] = s["v"].double().reshape(tokens, kv, hd)
        return dict(q=rotated(s["q"], heads), kcache=kcache, vcache=vcache)
    out = torch.empty((case["queries"], heads, hd), dtype=torch.float64, device="cuda")
    for i, (row, last) in enumerate(zip(s["sequence"].tolist(), s["positions"].tolist())):
        first = max(0, last + 1 - case["window"]) if case["window"] else 0
        at = torch.arange(first, last + 1, device="cuda")
        page = s["tables"][row].long()[at // size]
        k, v = (c[page, :, at % size].double() for c in (s["kcache"], s["vcache"]))  # [keys][kv][hd]
        for g in range(kv):
            q = s["q"][i].double().reshape(kv, heads // kv, hd)[g]
            scores = (k[:, g].contiguous() @ q.t().contiguous()) * s["scale"]
            out[i].reshape(kv, heads // kv, hd)[g] = torch.softmax(scores, 0).t().contiguous() @ v[:, g].contiguous()
    return out
