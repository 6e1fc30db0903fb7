"""The serving operators over a cache in 4 bits and of prompts, as a user's program calls them.

Keys and values held in 4 bits (``paged_append`` to a ``QuantizedCache``, and
``paged_read`` of what it stands for), the attention of one new token per
sequence over them, the same over a 16-bit cache with scores that are capped,
biased by distance or windowed, and the attention of prompts' rows over
themselves (``prompt_attention``) or over a cache (``paged_prompt``).  ``run``
computes them in plain torch operations, or with ``own`` set through the
framework's entry points; ``exact`` computes them in 64 bits.  Head layouts,
dims, page sizes and rotary bases are those of the benchmark's and the model
configurations (32 query / 8 KV heads and 28 / 4, head dim 128, base 500000 and
a yarn-scaled 1000000) and generic ones beside them.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GATHER = 1 << 28  # elements of keys, or of scores, that the plain forms hold at a time
GROUP = 32        # dims that share a scale and a zero
LARGEST = 4096.0   # magnitudes past it are not held

BASE = dict(base=500000.0, factor=1.0)
LINEAR = dict(base=10000.0, factor=4.0)  # positions slowed by the factor


def _case(kind, name, **over):
    case = dict(kind=kind, name=name, heads=8, group=4, dim=128, page=16, dtype="bf16",
                softcap=0.0, window=0, slopes=False, order=1)
    case.update(over)
    return case


def listed():
    return [
        # one decode step of 64 sequences: each one's new token to its page, and
        # the new tokens as the cache holds them
        _case("append", "append4_step_b64", batch=64, low=40, high=6000, new="step", **BASE),
        # several users' prompts at once behind what came before, and their rows
        # read back for the prompts' own attention
        _case("append", "append4_prompts_24k", batch=7, low=501, high=9001, new="part", page=64,
              heads=4, group=7, dtype="fp16", order=2, **LINEAR),
        # one short chat from the cache in 4 bits: launches and the chain of
        # loads count
        _case("decode4", "decode4_b1_2003", batch=1, low=2003, high=2003, empty=0),
        # a serving batch of chats and documents, some places of the batch idle
        _case("decode4", "decode4_b64_ragged", batch=64, low=30, high=16384, empty=5, order=4),
        # wide heads in the other type, scores capped
        _case("decode4", "decode4_b24_d256_cap", batch=24, low=500, high=12000, empty=0, heads=4,
              group=2, dim=256, page=32, dtype="fp16", softcap=50.0, order=5),
        # eight of the benchmark's long contexts
        _case("decode4", "decode4_b8_128k", batch=8, low=131001, high=131072, empty=0, page=32,
              order=6),
        # the 16-bit cache: a layer that sees the last 4096 tokens, scores capped
        _case("decode", "decode_b32_window_cap", batch=32, low=1000, high=30000, empty=2,
              softcap=30.0, window=4096, order=7),
        # the 16-bit cache: scores biased by distance, as many KV heads as query
        # heads
        _case("decode", "decode_b48_slopes_d64", batch=48, low=100, high=4000, empty=0, heads=16,
              group=1, dim=64, slopes=True, order=8),
        # one short question's own attention: latency
        _case("prompt", "prompt_b1_37", batch=1, low=37, high=37, new="all", paged=False,
              prefix=False),
        # documents packed into one batch, bidirectional over each one's
        # beginning, scores biased by distance, heads of 64
        _case("prompt", "prompt_documents_prefix_d64", batch=23, low=101, high=3001, new="all",
              paged=False, prefix=True, heads=12, group=1, dim=64, slopes=True, order=9),
        # one long document's prompt
        _case("prompt", "prompt_16k", batch=1, low=16384, high=16384, new="all", paged=False,
              prefix=False),
        # the next turns of a few chats, each over its own pages: few rows, a
        # long axis
        _case("prompt", "prompt_turns_b3", batch=3, low=20000, high=90000, new=33, paged=True,
              prefix=False, heads=4, group=7, page=64, order=10),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("append", "decode4", "decode4", "decode", "prompt", "prompt"))
    heads, group, dim = rng.choice(((8, 4, 128), (8, 4, 128), (4, 7, 128), (8, 4, 64), (2, 8, 256),
                                    (16, 1, 64), (4, 2, 96), (1, 16, 128), (3, 5, 160)))
    over = dict(heads=heads, group=group, dim=dim, page=rng.choice((16, 16, 32, 64, 128)),
                dtype=rng.choice(("bf16", "bf16", "fp16")), order=rng.randint(1, 1 << 20))
    scores = dict(softcap=rng.choice((0.0, 0.0, 30.0, 50.0)), slopes=rng.random() < 0.3,
                  window=rng.choice((0, 0, 0, 1024, 4096)))
    if kind == "append":
        # about as many values at most as the listed prompts have
        most = (1 << 24) // (heads * dim)
        batch = _log(rng, 1, 64)
        low, high = sorted(_log(rng, 1, most // batch + 1) for _ in range(2))
        case = _case(kind, "", batch=batch, low=low, high=high,
                     new=rng.choice(("step", "part", "all")), **over,
                     **rng.choice((BASE, LINEAR)))
    elif kind == "prompt":
        # at most the longest listed prompt's products
        batch = _log(rng, 1, 16)
        most = math.isqrt((1 << 39) // (batch * heads * group * dim))
        low, high = sorted(_log(rng, 1, min(most, 8192)) for _ in range(2))
        case = _case(kind, "", batch=batch, low=low, high=high, paged=rng.random() < 0.5,
                     prefix=rng.random() < 0.3, new="all", **over, **scores)
        if case["paged"]:
            case["new"] = rng.choice(("all", "part", 1 + _log(rng, 1, 100)))
    else:
        batch = _log(rng, 1, 128)
        most = max(64, min(131072, (1 << 28) // (batch * heads * dim)))
        low, high = sorted(_log(rng, 1, most) for _ in range(2))
        case = _case(kind, "", batch=batch, low=low, high=high,
                     empty=rng.choice((0, 0, min(2, batch - 1))), **over, **scores)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    """Visible tokens of each sequence, how many of them are new to it, and the
    tokens of its beginning that all of its rows see."""
    rng = random.Random(case["order"])
    lengths = [_log(rng, case["low"], case["high"]) for _ in range(case["batch"])]
    for b in rng.sample(range(case["batch"]), case.get("empty", 0)):
        lengths[b] = 0
    new = case.get("new", "step")
    if new == "step":
        count = [1] * len(lengths)
    elif new == "all":
        count = list(lengths)
    elif new == "part":
        count = [rng.randint(1, n) for n in lengths]
    else:
        count = [min(new, n) for n in lengths]
    prefix = [rng.randint(0, n) if case.get("prefix") else 0 for n in lengths]
    return lengths, count, prefix


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _table(case, lengths, gen):
    """The number of pages, and the (batch, blocks) table: pages in random
    order, a few unused, entries past a sequence's end -1 as an allocator
    leaves them."""
    page = case["page"]
    blocks = [-(-n // page) for n in lengths]
    count = sum(blocks) + 3
    order = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), max(blocks) + 2), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n]
        at += n
    return count, table


def _seven_bits(x):
    """Nonnegative fp16 numbers, rounded up to 7 significant bits."""
    return ((x.view(torch.int16) + 15) & -16).view(torch.float16)


def _quantize(x):
    """(.., dim) rows in 4 bits: codes (.., dim) uint8, and each group's scale
    (of 7 significant bits, rounded up) and zero (.., dim / 32, 2) fp16."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    scale, zero = _seven_bits(((high - low) / 15.0).half()), low.half()
    held = torch.maximum(low.abs(), high.abs()) <= LARGEST  # (false for NaN)
    scale, zero = (torch.where(held, t, torch.nan) for t in (scale, zero))
    step = scale.float()[..., None]
    codes = ((x - zero.float()[..., None]) / step).round().clamp(0.0, 15.0)
    codes = torch.where(step > 0, codes, 0.0).to(torch.uint8)
    return codes.flatten(-2), torch.stack((scale, zero), -1)


def _values(codes, scales):
    """What 4-bit rows stand for, in 32 bits."""
    scale, zero = scales.float().unbind(-1)
    codes = codes.float().unflatten(-1, (-1, GROUP))
    return (codes * scale[..., None] + zero[..., None]).flatten(-2)


def _toward(case, query, lengths, table, keys, gen):
    """One token of every hundred lies along its head's queries, so that the
    softmax has peaks."""
    first = torch.arange(0, max(int(lengths.max()), 1), 100, device="cuda")
    place = first + torch.randint(0, 100, (case["batch"], len(first)), generator=gen,
                                  device="cuda")
    seq, pick = (place < lengths[:, None]).nonzero(as_tuple=True)
    place = place[seq, pick]
    mean = query.unflatten(1, (case["heads"], case["group"])).float().mean(2) * 2.0
    noise = _normal(gen, (len(seq), case["heads"], case["dim"]), torch.float32)
    at = table[seq, place // case["page"]].long()
    keys[at, :, place % case["page"]] = (mean[seq] + noise).to(keys.dtype)


def _inputs(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed * 1000003 + 71)
    dtype, heads, dim = DTYPES[case["dtype"]], case["heads"], case["dim"]
    lengths, new, prefix = _lengths(case)
    starts = np.concatenate(([0], np.cumsum(new))).tolist()
    state = dict(host_lengths=lengths, host_new=new, host_starts=starts, host_prefix=prefix,
                 lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                 starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 prefix=torch.tensor(prefix, dtype=torch.int32, device="cuda"))
    if case["slopes"]:
        q_heads = heads * case["group"]
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / q_heads) for h in range(q_heads)],
                                       dtype=torch.float32, device="cuda")
    rows = sum(new) if case["kind"] in ("append", "prompt") else case["batch"]
    state["query"] = _normal(gen, (rows, heads * case["group"], dim), dtype)
    if case["kind"] == "append" or case["kind"] == "prompt" and not case["paged"]:
        state["key"], state["value"] = (_normal(gen, (rows, heads, dim), dtype) for _ in range(2))
    if case["kind"] == "prompt" and not case["paged"]:
        return state
    count, state["table"] = _table(case, lengths, gen)
    shape = (count, heads, case["page"], dim)
    if case["kind"] == "append":
        # pages as earlier calls left them: the new rows are all that is asked
        state["codes"] = [torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(2)]
        state["scales"] = [torch.zeros((*shape[:3], dim // GROUP, 2), dtype=torch.float16,
                                       device="cuda") for _ in range(2)]
        return state
    keys, values = _normal(gen, shape, dtype), _normal(gen, shape, dtype)
    if case["kind"] in ("decode", "decode4"):
        _toward(case, state["query"], state["lengths"], state["table"], keys, gen)
    if case["kind"] != "decode4":
        state["keys"], state["values"] = keys, values
        return state
    state["codes"], state["scales"] = [], []
    for pool in (keys, values):
        pieces = [_quantize(x) for x in pool.split(max(1, GATHER // (shape[1] * shape[2] * dim)))]
        state["codes"].append(torch.cat([c for c, _ in pieces]))
        state["scales"].append(torch.cat([s for _, s in pieces]))
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["kind"] == "append":
        state["rates"] = torch.from_numpy(_rates(case)).cuda()
    if own:
        package = os.path.abspath("refinekv-release_amd")  # (the working folder is the root)
        if package not in sys.path:
            sys.path.insert(0, package)
        import refinekv

        state["refinekv"], state["workspace"] = refinekv, {}
        if case["kind"] == "append":
            state["rotary"] = refinekv.Rotary(refinekv.RotaryConfig(
                head_dim=case["dim"], base=case["base"], factor=case["factor"],
                scaling="linear" if case["factor"] != 1.0 else "none"), device="cuda")
        if "codes" in state:
            state["cache"] = refinekv.QuantizedCache.packed(
                *state["codes"], *state["scales"], state["table"], state["lengths"],
                dtype=DTYPES[case["dtype"]])
        elif "keys" in state:
            state["cache"] = refinekv.PagedCache(state["keys"], state["values"], state["table"],
                                                 state["lengths"])
        state["options"] = dict(softcap=case["softcap"] or None, window=case["window"] or None,
                                slopes=state.get("slopes"), workspace=state["workspace"])
        if case.get("prefix"):
            state["options"]["prefix"] = state["prefix"]
    return state


# ---------------------------------------------------------------------------
# The operators, plain
# ---------------------------------------------------------------------------

def _rates(case):
    """Radians per position of each pair."""
    return case["base"] ** (-np.arange(0, case["dim"], 2, dtype=np.float64) / case["dim"]) \
        / case["factor"]


def _rotate(x, positions, rates):
    angles = positions.double()[:, None] * rates
    c, s = angles.cos().float()[:, None], angles.sin().float()[:, None]
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1).to(x.dtype)


def _plain_append(state):
    case = state["case"]
    starts, lengths, page = state["starts"].long(), state["lengths"].long(), case["page"]
    token = torch.arange(state["host_starts"][-1], device="cuda")
    seq = torch.searchsorted(starts[1:], token, right=True)
    position = lengths[seq] - starts[seq + 1] + token
    query = _rotate(state["query"], position, state["rates"])
    at, row = state["table"][seq, position // page].long(), position % page
    out = [query]
    rows = _rotate(state["key"], position, state["rates"]), state["value"]
    for codes, scales, x in zip(state["codes"], state["scales"], rows):
        codes[at, :, row], scales[at, :, row] = _quantize(x)
        out.append(_values(codes[at, :, row], scales[at, :, row]).to(x.dtype))
    return tuple(out)


def _scores(state, scores, distance, slopes):
    """Scores, capped and biased; distance and slopes broadcast to them."""
    case = state["case"]
    if case["softcap"]:
        scores = torch.tanh(scores / case["softcap"]) * case["softcap"]
    if case["slopes"]:
        scores = scores - slopes * distance.abs().float()
    return scores


def _weigh(scores, visible, v):
    scores = scores.masked_fill(~visible, -torch.inf)
    p = (scores - scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)).exp()
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, (p @ v) / total, 0.0)


def _plain_decode(state):
    case, table, lengths = state["case"], state["table"], state["lengths"]
    heads, group, dim, page = case["heads"], case["group"], case["dim"], case["page"]
    blocks = max(1, -(-max(state["host_lengths"]) // page))
    together = max(1, GATHER // (blocks * page * heads * dim))
    distance = lengths[:, None] - 1 - torch.arange(blocks * page, device="cuda")
    visible = distance >= 0
    if case["window"]:
        visible &= distance < case["window"]
    slopes = state["slopes"].view(heads, group, 1) if case["slopes"] else None
    outputs = []
    for b in range(0, case["batch"], together):
        take = slice(b, b + together)
        at = table[take, :blocks].clamp_min(0).long()
        if case["kind"] == "decode4":
            pools = [_values(c[at], s[at]) for c, s in zip(state["codes"], state["scales"])]
        else:
            pools = [state[x][at].float() for x in ("keys", "values")]
        # (n, blocks, heads, page, dim) -> (n, heads, tokens, dim)
        k, v = (x.transpose(1, 2).flatten(2, 3) for x in pools)
        q = state["query"][take].float().unflatten(1, (heads, group))
        scores = (q @ k.transpose(2, 3).contiguous()) * dim ** -0.5
        scores = _scores(state, scores, distance[take, None, None], slopes)
        out = _weigh(scores, visible[take, None, None], v)
        outputs.append(out.flatten(1, 2).to(state["query"].dtype))
    return torch.cat(outputs)


def _plain_prompt(state):
    case = state["case"]
    heads, group, dim, page = case["heads"], case["group"], case["dim"], case["page"]
    slopes = state["slopes"].view(heads, group, 1, 1) if case["slopes"] else None
    out = torch.empty_like(state["query"])
    for b, n in enumerate(state["host_lengths"]):
        first, end = state["host_starts"][b:b + 2]
        if case["paged"]:
            at = state["table"][b, :-(-n // page)].long()
            k, v = (state[x][at].transpose(0, 1).flatten(1, 2)[:, :n].float()
                    for x in ("keys", "values"))
        else:
            k, v = (state[x][first:end].transpose(0, 1).float() for x in ("key", "value"))
        k, v = k[:, None].transpose(2, 3).contiguous(), v[:, None].contiguous()
        token = torch.arange(n, device="cuda")
        together = max(1, GATHER // (n * heads * group))
        for row in range(first, end, together):
            take = slice(row, min(row + together, end))
            position = n - end + torch.arange(take.start, take.stop, device="cuda")
            distance = position[:, None] - token
            visible = (distance >= 0) | (token < state["host_prefix"][b])
            if case["window"]:
                visible &= distance < case["window"]
            # (rows, heads * group, dim) -> (heads, group, rows, dim)
            q = state["query"][take].float().unflatten(1, (heads, group)).permute(1, 2, 0, 3)
            scores = _scores(state, (q @ k) * dim ** -0.5, distance, slopes)
            seen = _weigh(scores, visible, v)
            out[take] = seen.permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
    return out


def run(state):
    case = state["case"]
    if own:
        refinekv = state["refinekv"]
        if case["kind"] == "append":
            starts = None if case["new"] == "step" else state["starts"]
            query = refinekv.paged_append(state["key"], state["value"], state["cache"],
                                          query=state["query"], rotary=state["rotary"],
                                          token_starts=starts)
            keys, values = refinekv.paged_read(state["cache"], state["key"].shape[0],
                                               token_starts=starts)
            return query, keys, values
        if case["kind"] != "prompt":
            return refinekv.paged_decode(state["query"], state["cache"], **state["options"])
        if case["paged"]:
            return refinekv.paged_prompt(state["query"], state["cache"],
                                         token_starts=state["starts"], **state["options"])
        return refinekv.prompt_attention(state["query"], state["key"], state["value"],
                                         token_starts=state["starts"], **state["options"])
    if case["kind"] == "append":
        return _plain_append(state)
    return _plain_prompt(state) if case["kind"] == "prompt" else _plain_decode(state)


def _pairs(case, n, new, prefix):
    """Visible (row, token) pairs of a sequence of n tokens, `new` of them rows."""
    position = np.arange(n - new, n, dtype=np.int64)
    first = np.maximum(position + 1 - case["window"], 0) if case["window"] else position * 0
    return int((np.maximum(position + 1, prefix) - first).clip(0).sum())


def work(case):
    heads, group, dim = case["heads"], case["group"], case["dim"]
    held = dim / 2 + dim // GROUP * 4  # bytes of a head's row in 4 bits
    lengths, new, prefix = _lengths(case)
    if case["kind"] == "append":
        rows = sum(new) * heads
        # rows and queries in, the cache's rows and turned queries out, the rows read back
        return {"bytes": rows * ((group + 2) * dim * 2 + group * dim * 2 + 2 * held + 2 * dim * 2),
                "flops": rows * dim * (3 * (group + 1) + 2 * 6)}
    if case["kind"] == "prompt":
        pairs = sum(_pairs(case, n, m, p) for n, m, p in zip(lengths, new, prefix))
        rows, seen = sum(new) * heads * group * dim, sum(lengths) * heads * dim
        return {"bytes": rows * 2 * 2 + seen * 2 * 2, "flops": pairs * heads * group * dim * 4}
    seen = sum(min(n, case["window"] or n) for n in lengths) * heads
    return {"bytes": seen * 2 * (held if case["kind"] == "decode4" else dim * 2)
            + case["batch"] * heads * group * dim * 2 * 2
            + sum(-(-n // case["page"]) for n in lengths) * 4,
            "flops": seen * dim * group * 4}


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------

def _held64(x):
    """What rows stand for once they are held in 4 bits."""
    groups = x.double().reshape(*x.shape[:-1], -1, GROUP)
    zero = groups.min(-1, keepdim=True).values.half().double()
    span = groups.max(-1, keepdim=True).values - groups.min(-1, keepdim=True).values
    scale = (span / 15).half().double()
    unit = torch.exp2(torch.floor(torch.log2(scale.clamp_min(2.0 ** -14))) - 6)
    scale = torch.ceil(scale / unit) * unit
    steps = torch.where(scale > 0, (groups - zero) / scale.clamp_min(1e-30), 0 * groups)
    return (zero + scale * torch.round(steps).clamp(0, 15)).reshape(x.shape)


def _turn64(case, x, positions):
    """As a product of complex numbers, rounded to the rows' type."""
    half = case["dim"] // 2
    rates = [math.exp(-2.0 * i / case["dim"] * math.log(case["base"])) / case["factor"]
             for i in range(half)]
    rates = torch.tensor(rates, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       positions.double()[:, None] * rates)[:, None]
    wide = x.double()
    turned = torch.complex(wide[..., :half].contiguous(), wide[..., half:].contiguous()) * turn
    return torch.cat((turned.real, turned.imag), -1)


def _rows64(state, name, b, h):
    """Sequence b's keys or values of head h."""
    case, n = state["case"], state["host_lengths"][b]
    take = state["table"][b, :-(-n // case["page"])].long()
    if case["kind"] == "decode4":
        k = 0 if name == "keys" else 1
        codes = state["codes"][k][take, h].double().flatten(0, 1)[:n]
        both = state["scales"][k][take, h].double().flatten(0, 1)[:n]
        both = both.repeat_interleave(GROUP, dim=1)
        return both[..., 1] + both[..., 0] * codes
    return state[name][take, h].flatten(0, 1)[:n].double()


def _attend64(state, q, k, v, position, prefix, h):
    """Query rows of one head at their positions over its keys."""
    case = state["case"]
    x = (q.double() @ k.T) / math.sqrt(case["dim"])
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    there = torch.arange(len(k), device="cuda")[None]
    here = position[:, None]
    if case["slopes"]:
        x = x - float(state["slopes"][h]) * (here - there).abs()
    hidden = (there > here) & (there >= prefix)
    if case["window"]:
        hidden |= there <= here - case["window"]
    return torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v


def exact(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    dtype, group = DTYPES[case["dtype"]], case["group"]
    if case["kind"] == "append":
        positions = torch.cat([torch.arange(n - m, n, device="cuda")
                               for n, m in zip(state["host_lengths"], state["host_new"])])
        key = _turn64(case, state["key"], positions).to(dtype)
        return (_turn64(case, state["query"], positions), _held64(key), _held64(state["value"]))
    out = torch.zeros(state["query"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(state["host_lengths"]):
        if n == 0:
            continue
        if case["kind"] == "prompt":
            first, end = state["host_starts"][b:b + 2]
        else:
            first, end = b, b + 1
        for h in range(case["heads"]):
            if case["kind"] == "prompt" and not case["paged"]:
                k, v = state["key"][first:end, h].double(), state["value"][first:end, h].double()
            else:
                k, v = _rows64(state, "keys", b, h), _rows64(state, "values", b, h)
            for q in range(h * group, (h + 1) * group):
                for row in range(first, end, 4096):
                    rows = torch.arange(row, min(row + 4096, end), device="cuda")
                    out[rows, q] = _attend64(state, state["query"][rows, q], k, v, n - end + rows,
                                             state["host_prefix"][b], q)
    return out
