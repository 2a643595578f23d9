"""Representative calls of the paged-cache operators, and how to time and check one.

They are what a decoder layer runs between its linears, on a key/value cache that is held in pages
and a prefix that every request of the batch shares:

* ``slots`` (``paged_slots``): one step's bookkeeping from the requests' lengths: block tables with
  pages taken off a free list, the cache slot and the position of every new token, token offsets.
* ``rotary`` (``rotary``): rotary positions of the queries and keys of a layer, or the inverse
  rotation (the gradient's direction).
* ``store`` (``rotary_store``): the same with the keys and values written to their cache slots.
* ``attention`` (``paged_attention``): queries of one or more tokens a request against the shared
  prefix and the request's own pages, causal within the request.

Lengths, sizes and layouts are the case's; the seed makes values, page orders and free lists.
"""

from __future__ import annotations

import functools
import math
import random

import torch

own = False

# ------------------------------------------------------------------- cases


def _slots(name, requests, new, length, page, columns):
    return {"name": name, "op": "slots", "requests": requests, "new": new, "length": length, "page": page,
            "columns": columns, "mix": 1}


def _rotary(name, op, tokens, heads, kv, dim, rotated, layout, dtype, reach, inverse=False, page=16):
    case = {"name": name, "op": op, "tokens": tokens, "heads": heads, "kv": kv, "dim": dim, "rotated": rotated,
            "layout": layout, "dtype": dtype, "reach": reach}
    case.update({"inverse": inverse} if op == "rotary" else {"page": page})
    return case


def _attention(name, requests, new, length, prefix, heads, kv, dim, page, ragged):
    return {"name": name, "op": "attention", "requests": requests, "new": new, "length": length, "prefix": prefix,
            "heads": heads, "kv": kv, "dim": dim, "page": page, "ragged": ragged, "mix": 1}


def listed():
    return [
        # the bookkeeping of one decode step of a small batch: latency only
        _slots("slots_b8_decode", 8, 1, 2000, 16, 256),
        # a large batch between decode steps and prompt chunks, tables for 32768 tokens each
        _slots("slots_b256_mixed", 256, 64, 16000, 16, 2048),
        # one decode step of a few sequences before a cache of another layout
        _rotary("rotary_t8_half", "rotary", 8, 32, 8, 128, 128, "half", "float16", 40960),
        # a long prompt's gradient direction, interleaved pairs over part of the head, fp32 values
        _rotary("rotary_t4093_interleaved_f32", "rotary", 4093, 32, 8, 128, 64, "interleaved", "float32", 131072, True),
        # one decode step of 64 sequences, keys and values stored
        _rotary("store_t64_half", "store", 64, 32, 8, 128, 128, "half", "float16", 40960),
        # a prompt of 8192 tokens, keys and values stored
        _rotary("store_t8192_half", "store", 8192, 32, 8, 128, 128, "half", "float16", 40960),
        # a chat turn of one user: one token, a thousand or so behind it, no prefix
        _attention("attention_b1_n1", 1, 1, 1021, 0, 32, 8, 128, 16, False),
        # decode of 64 requests that share a long system prompt, own parts short and ragged
        _attention("attention_b64_prefix16384", 64, 1, 600, 16384, 32, 8, 128, 16, True),
        # decode of a large batch of long requests behind a short shared prompt: the cache's bytes
        _attention("attention_b256_n1", 256, 1, 4096, 133, 32, 8, 128, 16, True),
        # drafted tokens verified, a smaller head size, every query head with keys of its own
        _attention("attention_b12_n5_d64", 12, 5, 3000, 1500, 16, 16, 64, 32, True),
        # one long document asked one question: a whole context of prefix for a single token
        _attention("attention_b1_prefix131072", 1, 1, 40, 131071, 32, 8, 128, 64, False),
        # prompt chunks of three requests behind the shared prompt: the most arithmetic of one call
        _attention("attention_b3_n1024_prefix8192", 3, 1024, 2500, 8192, 32, 8, 128, 16, True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("slots", "rotary", "store", "attention", "attention", "attention"))
    if op == "slots":
        page = rng.choice((8, 16, 32, 64))
        case = _slots("", _log_int(rng, 1, 256), _log_int(rng, 1, 64), _log_int(rng, 1, 16000), page, 0)
        case["columns"] = -(-(case["length"] + case["new"]) // page) + rng.randint(0, 200)
        if case["requests"] * case["columns"] > 256 * 2048:
            case["requests"] = max(1, 256 * 2048 // case["columns"])
    elif op in ("rotary", "store"):
        heads, kv = rng.choice(((32, 8), (16, 16), (28, 4), (12, 2), (8, 1), (5, 5)))
        dim = rng.choice((64, 96, 128, 128))
        rotated = rng.choice((dim, dim, dim // 2, dim // 2 - 2))
        case = _rotary("", op, _log_int(rng, 1, 4096), heads, kv, dim, rotated, rng.choice(("half", "interleaved")),
                       rng.choice(("float16", "float16", "float32")), _log_int(rng, 4096, 131072), rng.random() < 0.3,
                       rng.choice((8, 16, 64)))
    else:
        heads, kv = rng.choice(((32, 8), (32, 8), (16, 16), (28, 4), (16, 1), (24, 8)))
        kind = rng.choice(("decode", "decode", "verify", "prompt"))
        requests = _log_int(rng, 1, 256) if kind != "prompt" else rng.randint(1, 4)
        new = {"decode": 1, "verify": rng.randint(2, 8), "prompt": _log_int(rng, 9, 1024)}[kind]
        case = _attention("", requests, new, max(new, _log_int(rng, 1, 8192)),
                          rng.choice((0, _log_int(rng, 1, 32768))), heads, kv, rng.choice((64, 128, 128)),
                          rng.choice((8, 16, 32, 64, 128)), rng.random() < 0.8)
        top = [work(each) for each in listed()]
        while any(work(case)[key] > max(each[key] for each in top) for key in ("bytes", "flops")):
            case["length"] = max(new, case["length"] * 3 // 4)
            case["requests"] = max(1, case["requests"] * 3 // 4)
            case["prefix"] = case["prefix"] * 3 // 4
    if "mix" in case:
        case["mix"] = rng.randint(2, 1 << 20)
    del case["name"]
    return case


# ------------------------------------------------------- lengths and counts


def _requests(case):
    """(tokens a request has behind it, new tokens) for each request of a case."""
    rng = random.Random(case["mix"])
    result = []
    for _ in range(case["requests"]):
        if case["op"] == "slots":
            result.append((rng.randint(0, case["length"]), rng.choice((1, 1, 1, rng.randint(0, case["new"])))))
        elif case["ragged"]:
            length = rng.randint(1, case["length"])
            new = min(length, case["new"] if rng.random() < 0.5 else rng.randint(1, case["new"]))
            result.append((length - new, new))
        else:
            result.append((case["length"] - case["new"], case["new"]))
    if not any(new for _, new in result):
        result[0] = (result[0][0], 1)
    return result


def work(case):
    if case["op"] == "slots":
        tokens = sum(new for _, new in _requests(case))
        taken = sum(-(-(b + n) // case["page"]) - -(-b // case["page"]) for b, n in _requests(case))
        table = case["requests"] * case["columns"]
        return {"bytes": 4 * (2 * table + taken + 2 * tokens + 4 * case["requests"] + 4), "flops": table + 2 * tokens}
    if case["op"] in ("rotary", "store"):
        size = 2 if case["dtype"] == "float16" else 4
        rows = case["tokens"] * (case["heads"] + case["kv"] * (2 if case["op"] == "store" else 1))
        values = rows * case["dim"]
        out = size if case["op"] == "rotary" else 2
        places = 4 * case["tokens"] * (1 + (case["op"] == "store"))
        return {"bytes": values * (size + out) + places + 4 * min(case["tokens"], case["reach"]) * case["rotated"],
                "flops": 3 * case["tokens"] * (case["heads"] + case["kv"]) * case["rotated"]}
    requests = _requests(case)
    tokens = sum(new for _, new in requests)
    keys = case["prefix"] + sum(behind + new for behind, new in requests)
    pairs = tokens * case["prefix"] + sum(new * behind + new * (new + 1) // 2 for behind, new in requests)
    return {"bytes": 4 * keys * case["kv"] * case["dim"] + 4 * tokens * case["heads"] * case["dim"]
            + 4 * (keys // case["page"] + 2 * case["requests"]),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ------------------------------------------------------------------ inputs


def _generator(seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    return generator


def _normal(generator, shape, dtype, scale=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(0.0, scale, generator=generator)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@functools.lru_cache(maxsize=4)
def _angles(reach, rotated):
    """cos and sin of position times frequency, [reach, rotated]: cosines, then sines."""
    frequency = 1e6 ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device="cuda") / rotated)
    angle = torch.arange(reach, dtype=torch.float64, device="cuda")[:, None] * frequency
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1).float()


def _inputs(case, seed):
    g = _generator(seed)
    if case["op"] == "slots":
        requests = _requests(case)
        page, columns = case["page"], case["columns"]
        used = [-(-behind // page) for behind, _ in requests]
        taken = sum(-(-(behind + new) // page) for behind, new in requests) - sum(used)
        order = torch.randperm(sum(used) + taken + 37, device="cuda", generator=g).to(torch.int32)
        held = torch.arange(columns, device="cuda")[None, :] < _ints(used)[:, None]
        table = torch.full((case["requests"], columns), -1, dtype=torch.int32, device="cuda")
        table[held] = order[:sum(used)]
        return {"lengths": _ints([behind for behind, _ in requests]), "counts": _ints([new for _, new in requests]),
                "start": _ints([133]), "free": order[sum(used):].contiguous(), "free_count": _ints([taken + 37]),
                "table": table, "tokens": sum(new for _, new in requests)}
    if case["op"] in ("rotary", "store"):
        dtype, tokens, dim = getattr(torch, case["dtype"]), case["tokens"], case["dim"]
        state = {"q": _normal(g, (tokens, case["heads"], dim), dtype), "k": _normal(g, (tokens, case["kv"], dim), dtype),
                 "positions": torch.randint(0, case["reach"], (tokens,), dtype=torch.int32, device="cuda", generator=g),
                 "angles": _angles(case["reach"], case["rotated"])}
        if case["op"] == "store":
            pages = -(-tokens // case["page"]) + 3
            places = torch.randperm(pages * case["page"], device="cuda", generator=g)[:tokens]
            shape = (pages, case["kv"], case["page"], dim)
            state.update(v=_normal(g, (tokens, case["kv"], dim), dtype), slots=places.to(torch.int32),
                         q_out=torch.empty((tokens, case["heads"], dim), dtype=torch.float16, device="cuda"),
                         k_cache=_normal(g, shape, torch.float16), v_cache=_normal(g, shape, torch.float16))
        return state
    requests, page = _requests(case), case["page"]
    lengths = [behind + new for behind, new in requests]
    prefix_pages = max(1, -(-case["prefix"] // page))
    held = [-(-length // page) for length in lengths]
    pages = sum(held) + prefix_pages
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    inside = torch.arange(max(held), device="cuda")[None, :] < _ints(held)[:, None]
    table = torch.full((case["requests"], max(held)), -1, dtype=torch.int32, device="cuda")
    table[inside] = order[:sum(held)]
    offsets = [0]
    for _, new in requests:
        offsets.append(offsets[-1] + new)
    shape = (pages, case["kv"], page, case["dim"])
    return {"q": _normal(g, (offsets[-1], case["heads"], case["dim"]), torch.float16, 2.0),
            "k_cache": _normal(g, shape, torch.float16), "v_cache": _normal(g, shape, torch.float16),
            "offsets": _ints(offsets), "lengths": _ints(lengths), "table": table,
            "prefix_pages": order[sum(held):].contiguous(), "prefix_length": _ints([case["prefix"]])}


@functools.lru_cache(maxsize=None)
def _kernel(name, **options):
    import tensor_amd.torch as tt

    return tt.load(name, **options)


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if not own:
        return state
    if case["op"] == "slots":
        call = _kernel("paged_slots", page_size=case["page"]).prepare(
            *(state[key] for key in ("lengths", "counts", "start", "free", "free_count", "table", "tokens")))
    elif case["op"] == "rotary":
        call = _kernel("rotary", layout=case["layout"], dtype=case["dtype"], inverse=case["inverse"]).prepare(
            state["q"], state["k"], state["positions"], state["angles"])
    elif case["op"] == "store":
        call = _kernel("rotary_store", layout=case["layout"], dtype=case["dtype"]).prepare(
            *(state[key] for key in ("q", "k", "v", "positions", "slots", "angles", "q_out", "k_cache", "v_cache")))
    else:
        from tensor_amd.torch.session import session

        tokens, heads, dim = state["q"].shape
        need = session(0).attention_workspace(tokens, case["requests"], heads, case["kv"], dim)
        workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
        call = _kernel("paged_attention").prepare(
            *(state[key] for key in ("q", "k_cache", "v_cache", "offsets", "lengths", "table", "prefix_pages",
                                     "prefix_length")), workspace)
    state["call"] = call
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        state["call"]()
        return (state["q_out"], state["k_cache"], state["v_cache"]) if op == "store" else state["call"].outputs
    return {"slots": _plain_slots, "rotary": _plain_rotary, "store": _plain_store, "attention": _plain_attention}[op](state)


# ------------------------------------------------------------- plain forms


def _plain_slots(state):
    page, columns = state["case"]["page"], state["case"]["columns"]
    before, counts, tokens = state["lengths"], state["counts"], state["tokens"]
    after = before + counts
    held, wanted = (before + page - 1) // page, (after + page - 1) // page
    ends = torch.cumsum(wanted - held, 0)
    column = torch.arange(columns, device="cuda")[None, :]
    rank = (ends - (wanted - held))[:, None] + column - held[:, None]  # of a new page, in request order
    fresh = state["free"][(state["free_count"] - 1 - rank).clamp(0, state["free"].shape[0] - 1)]
    nothing = torch.full_like(state["table"], -1)
    table = torch.where(column < held[:, None], state["table"], torch.where(column < wanted[:, None], fresh, nothing))
    offsets = torch.cat([torch.zeros_like(counts[:1]), torch.cumsum(counts, 0).to(torch.int32)])
    token = torch.arange(tokens, dtype=torch.int32, device="cuda")
    request = torch.searchsorted(offsets[1:], token, right=True)
    place = before[request] + token - offsets[request]
    slots = table[request, place // page] * page + place % page
    return (offsets, after, place + state["start"], slots, table, state["free_count"] - ends[-1:].to(torch.int32))


def _rotate(x, cos, sin, layout):
    """x [tokens, heads, dim] with its leading dimensions rotated, as many as cos and sin have pairs for."""
    pairs = cos.shape[1]
    cos, sin = cos[:, None, :], sin[:, None, :]
    head, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if layout == "half":
        a, b = head[..., :pairs], head[..., pairs:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = head[..., 0::2], head[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _plain_rotated(state, x):
    case = state["case"]
    rows = state["angles"][state["positions"]]
    pairs = case["rotated"] // 2
    sin = rows[:, pairs:]
    return _rotate(x.float(), rows[:, :pairs], -sin if case.get("inverse") else sin, case["layout"])


def _plain_rotary(state):
    return tuple(_plain_rotated(state, state[key]).to(state[key].dtype) for key in ("q", "k"))


def _plain_store(state):
    page = state["case"]["page"]
    where, inside = state["slots"] // page, state["slots"] % page
    state["k_cache"][where, :, inside] = _plain_rotated(state, state["k"]).half()
    state["v_cache"][where, :, inside] = state["v"].half()
    return _plain_rotated(state, state["q"]).half(), state["k_cache"], state["v_cache"]


def _gather(cache, pages, length):
    """[kv, length, dim] in fp32: the first `length` tokens of a list of pages."""
    rows = cache[pages].permute(1, 0, 2, 3)
    return rows.reshape(cache.shape[1], -1, cache.shape[3])[:, :length].float()


def _plain_attention(state):
    case = state["case"]
    page, prefix, kv, dim = case["page"], case["prefix"], case["kv"], case["dim"]
    share = case["heads"] // kv
    first = -(-prefix // page)
    prefix_k = _gather(state["k_cache"], state["prefix_pages"][:first], prefix)
    prefix_v = _gather(state["v_cache"], state["prefix_pages"][:first], prefix)
    out = torch.empty_like(state["q"])
    begin = 0
    for request, (behind, new) in enumerate(_requests(case)):
        length = behind + new
        pages = state["table"][request, :-(-length // page)]
        k = torch.cat([prefix_k, _gather(state["k_cache"], pages, length)], 1)
        v = torch.cat([prefix_v, _gather(state["v_cache"], pages, length)], 1)
        q = state["q"][begin:begin + new].float().reshape(new, kv, share, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim)
        scores = torch.bmm(q, k.transpose(1, 2).contiguous()) * dim ** -0.5
        if new > 1:
            hidden = (torch.arange(prefix + length, device="cuda")[None, :]
                      > prefix + behind + torch.arange(new, device="cuda")[:, None]).repeat(share, 1)
            scores = scores.masked_fill(hidden, -math.inf)
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        weights = weights / weights.sum(-1, keepdim=True)
        result = torch.bmm(weights, v).reshape(kv, share, new, dim).permute(2, 0, 1, 3)
        out[begin:begin + new] = result.reshape(new, kv * share, dim).half()
        begin += new
    return (out,)


# ------------------------------------------------------- the same in 64 bits


def _turn(x, positions, case):
    """Rotary positions from their definition: pair p of a head is a point of the plane turned by
    position times base ** (-2 p / rotated), whose cosine and sine enter as the fp32 values given."""
    rotated, result = case["rotated"], x.double().clone()
    rows = _angles(case["reach"], rotated).double()[positions.long()]
    for p in range(rotated // 2):
        i, j = (p, p + rotated // 2) if case["layout"] == "half" else (2 * p, 2 * p + 1)
        point = torch.complex(x[..., i].double(), x[..., j].double())
        unit = torch.complex(rows[:, p], rows[:, rotated // 2 + p])[:, None]
        point = point * (unit.conj() if case.get("inverse") else unit)
        result[..., i], result[..., j] = point.real, point.imag
    return result


def exact(case, seed):
    inputs = _inputs(case, seed)
    if case["op"] == "slots":
        return None  # whole numbers
    if case["op"] == "rotary":
        return tuple(_turn(inputs[key], inputs["positions"], case) for key in ("q", "k"))
    if case["op"] == "store":
        k_cache, v_cache = inputs["k_cache"].double(), inputs["v_cache"].double()
        k = _turn(inputs["k"], inputs["positions"], case)
        place = inputs["slots"].long()
        flat = (place // case["page"]) * case["kv"] * case["page"] + place % case["page"]
        for head in range(case["kv"]):
            rows = flat + head * case["page"]
            k_cache.view(-1, case["dim"])[rows] = k[:, head]
            v_cache.view(-1, case["dim"])[rows] = inputs["v"][:, head].double()
        return _turn(inputs["q"], inputs["positions"], case), k_cache, v_cache
    share, page, prefix = case["heads"] // case["kv"], case["page"], case["prefix"]
    out = torch.zeros(inputs["q"].shape, dtype=torch.float64, device="cuda")
    for head in range(case["kv"]):
        keys, values = (inputs[name][:, head].reshape(-1, case["dim"]) for name in ("k_cache", "v_cache"))

        def rows(pages, length):
            at = torch.arange(length, device="cuda")
            return pages[at // page].long() * page + at % page

        shared = rows(inputs["prefix_pages"], prefix)
        begin = 0
        for request, (behind, new) in enumerate(_requests(case)):
            at = torch.cat([shared, rows(inputs["table"][request], behind + new)])
            k, v = keys[at].double(), values[at].double()
            limit = prefix + behind + torch.arange(new, device="cuda")
            seen = torch.arange(at.shape[0], device="cuda")[None, :] <= limit[:, None]
            q = inputs["q"][begin:begin + new, head * share:(head + 1) * share].double()
            for j in range(share):
                logits = (q[:, j] @ k.T) / math.sqrt(case["dim"])
                logits = torch.where(seen, logits, torch.full_like(logits, -math.inf))
                out[begin:begin + new, head * share + j] = torch.softmax(logits, -1) @ v
            begin += new
    return (out,)
