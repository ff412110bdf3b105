"""The paged key-value cache and the attention of a decode step, as a list of cases and a way to draw more of the same kind.

Three operators, each with its plain form in elementary torch operations and with its definition in 64 bits:

``attend``  attention of one new token per sequence over the cache, in bf16 or as the e4m3 codes that the output projection
            takes.
``write``   the keys and values of a step's tokens go to their slots of the cache: as they are (bf16), or as e4m3 codes with
            one scale per token and head.
``read``    the first tokens of some sequences come back out of the cache as bf16 rows, one sequence behind the other: what
            the attention of a prompt takes whose beginning is cached already.

Heads are those of the 7B-sized dense model (28 query heads on 4, of 128) and of the 60-expert block's model (16 on 16, of
128), and generic ones.  Keys have a constant part in each channel and a few loud channels, queries are large enough for a
softmax that prefers some tokens, as those of trained models are.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
OUT_SCALE = 0.01              # the static scale of the projection behind the attention


def _kernels():
    return importlib.import_module("nano-vllm-moe_b200.quantization.kernels")


def _attend(name, batch, shortest, longest, heads, kv_heads, dim, cache, block, codes=False, empty=0):
    """Sequences of ``shortest`` to ``longest`` cached tokens; the last ``empty`` rows of the batch are padding."""
    return {"name": name, "op": "attend", "batch": batch, "shortest": shortest, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "cache": cache, "block": block, "codes": codes, "empty": empty}


def _write(name, tokens, kv_heads, dim, cache, block, padding=0):
    """``tokens`` rows, the last ``padding`` of which have no slot."""
    return {"name": name, "op": "write", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "cache": cache, "block": block,
            "padding": padding}


def _read(name, batch, shortest, longest, kv_heads, dim, cache, block):
    return {"name": name, "op": "read", "batch": batch, "shortest": shortest, "longest": longest, "kv_heads": kv_heads,
            "dim": dim, "cache": cache, "block": block}


def listed():
    return [
        # the second step of a short chat, one user: launch and latency are everything
        _attend("attend_bf16_b1_c17", 1, 17, 17, 28, 4, 128, "bf16", 256),
        # one user with a book in the cache: one long axis for the whole chip
        _attend("attend_e4m3_b1_c131071", 1, 131071, 131071, 28, 4, 128, "e4m3", 256),
        # a few users at different places of their conversations
        _attend("attend_bf16_b8_ragged", 8, 1, 4096, 28, 4, 128, "bf16", 256),
        # a full decode batch over an 8-bit cache, its output quantised for the projection behind it
        _attend("attend_e4m3_b64_ragged_codes", 64, 1000, 8192, 28, 4, 128, "e4m3", 256, codes=True),
        # every query head has its own keys, small pages
        _attend("attend_bf16_b32_own_keys", 32, 100, 2048, 16, 16, 128, "bf16", 16),
        # many short answers of a small model, the batch padded to the size of a captured graph
        _attend("attend_e4m3_b256_short", 256, 1, 512, 14, 2, 64, "e4m3", 16, empty=13),
        # the tokens of a decode batch
        _write("write_e4m3_t64", 64, 4, 128, "e4m3", 256),
        # a mixed batch of decode tokens and prompt pieces, padded, 16 heads
        _write("write_bf16_t1031", 1031, 16, 128, "bf16", 16, padding=7),
        # the tokens of a full prefill batch
        _write("write_e4m3_t16384", 16384, 4, 128, "e4m3", 256),
        # the cached beginning of one prompt
        _read("read_e4m3_b1_c777", 1, 777, 777, 4, 128, "e4m3", 256),
        # cached beginnings of a batch of prompts, 16 heads, small pages
        _read("read_bf16_b8_own_keys", 8, 1, 2048, 16, 128, "bf16", 16),
        # cached beginnings of a batch of long prompts
        _read("read_e4m3_b16_ragged", 16, 100, 8192, 4, 128, "e4m3", 256),
    ]


def _spread(rng, low, high):
    """A whole number between ``low`` and ``high``, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


HEADS = [(28, 4, 128), (16, 16, 128), (14, 2, 64), (32, 8, 128), (16, 2, 128), (12, 12, 64), (10, 10, 80), (8, 1, 256), (24, 2, 96),
         (20, 1, 128)]
BLOCKS = [8, 16, 24, 32, 64, 128, 256]


def draw(rng):
    op = rng.choice(["attend", "attend", "write", "read"])
    heads, kv_heads, dim = rng.choice(HEADS)
    cache, block = rng.choice(["bf16", "e4m3"]), rng.choice(BLOCKS)
    cached = dim + 4 if cache == "e4m3" else 2 * dim
    if op == "write":
        tokens = _spread(rng, 1, 50_000_000 // (2 * kv_heads * (2 * dim + cached)))
        return {"op": op, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "cache": cache, "block": block,
                "padding": rng.randrange(0, tokens // 8 + 1)}
    # cached tokens in all: as many as the largest listed case moves bytes and multiplies for
    most = min(200_000_000 // (2 * kv_heads * (2 * dim + cached)), 4_000_000_000 // (4 * heads * dim))
    longest = _spread(rng, 1, min(131071, most))
    batch = _spread(rng, 1, max(1, min(256, most // longest)))
    shortest = rng.choice([1, max(1, longest // 2), longest])
    if op == "read":
        return {"op": op, "batch": batch, "shortest": shortest, "longest": longest, "kv_heads": kv_heads, "dim": dim, "cache": cache,
                "block": block}
    return {"op": op, "batch": batch, "shortest": shortest, "longest": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "cache": cache, "block": block, "codes": rng.random() < 0.3, "empty": rng.randrange(0, batch // 8 + 1)}


# ---- inputs ----------------------------------------------------------------------------------------------------------------


def _lengths(case):
    """Spread evenly between the shortest and the longest, in an order that no kernel can rely on; the same for every seed."""
    real = case["batch"] - case.get("empty", 0)
    span = case["longest"] - case["shortest"]
    lengths = [case["longest"] - span * i // max(1, real - 1) for i in range(real)]
    at = sorted(range(real), key=lambda i: (i * 7919 + 13) % max(1, real))
    return [lengths[i] for i in at] + [0] * (case["batch"] - real)


def _keys(rows, kv_heads, dim, gen):
    """Keys as trained models have them: a constant part in each channel, a few channels eight times as loud."""
    loud = torch.ones(kv_heads, dim, device="cuda")
    loud[:, torch.randperm(dim, generator=gen, device="cuda")[: max(1, dim // 32)]] = 8.0
    constant = torch.randn(kv_heads, dim, generator=gen, device="cuda")
    return ((torch.randn(rows, kv_heads, dim, generator=gen, device="cuda") + constant) * loud).to(torch.bfloat16)


def _quantised(x):
    """(codes, scales): one scale per row of the last dimension."""
    x = x.float()
    amax = x.abs().amax(-1).clamp(min=1e-8)
    scale = amax / torch.full_like(amax, FP8_MAX)         # (by a tensor: a true division, where one by a number multiplies by 1 / 448)
    return (x / scale[..., None]).clamp(-FP8_MAX, FP8_MAX).to(FP8), scale


def _empty_cache(case, blocks):
    """Pages of [block, head, token, channel] in memory, [block, token, head, channel] to the caller."""
    shape = (blocks, case["kv_heads"], case["block"], case["dim"])
    e4m3 = case["cache"] == "e4m3"
    made = {}
    for name in ("k", "v"):
        made[name + "_cache"] = torch.zeros(shape, device="cuda", dtype=torch.uint8 if e4m3 else torch.bfloat16).transpose(1, 2)
        if e4m3:
            made[name + "_cache"] = made[name + "_cache"].view(FP8)
        made[name + "_scale"] = torch.zeros(shape[:3], device="cuda").transpose(1, 2) if e4m3 else None
    return made


def _bytes_of(t):
    return t.view(torch.uint8) if t.dtype == FP8 else t


def _full_cache(case, lengths, gen):
    """A cache whose pages are dealt to the sequences in no order, every page filled; pages that belong to nobody lie between."""
    need = [-(-n // case["block"]) for n in lengths]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    host = torch.arange(max(1, max(need))).expand(len(need), -1)
    first = torch.tensor([sum(need[:i]) for i in range(len(need))])[:, None]
    inside = host < torch.tensor(need)[:, None]
    tables = torch.where(inside.cuda(), order[(first + host).clamp(max=blocks - 1).cuda()], -1).to(torch.int32)
    state = _empty_cache(case, blocks)
    for name in ("k", "v"):
        rows = blocks * case["block"]
        x = (_keys(rows, case["kv_heads"], case["dim"], gen) if name == "k" else
             torch.randn(rows, case["kv_heads"], case["dim"], generator=gen, device="cuda").to(torch.bfloat16))
        x = x.view(blocks, case["block"], case["kv_heads"], case["dim"])
        if case["cache"] == "e4m3":
            codes, scale = _quantised(x)
            _bytes_of(state[name + "_cache"]).copy_(_bytes_of(codes))
            state[name + "_scale"].copy_(scale)
        else:
            state[name + "_cache"].copy_(x)
    return state | {"block_tables": tables}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kv_heads, dim, block = case["kv_heads"], case["dim"], case["block"]
    if case["op"] == "write":
        tokens, kept = case["tokens"], case["tokens"] - case["padding"]
        blocks = -(-kept // block) + 2
        # keys and values are slices of one projection's output, as a layer hands them over
        qkv = torch.randn(tokens, (kv_heads + 2 * kv_heads) * dim, generator=gen, device="cuda").to(torch.bfloat16)
        qkv[:, kv_heads * dim:2 * kv_heads * dim] = _keys(tokens, kv_heads, dim, gen).view(tokens, -1)
        slots = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
        slots[:kept] = torch.randperm(blocks * block, generator=gen, device="cuda")[:kept].to(torch.int32)
        k, v = (qkv[:, i * kv_heads * dim:(i + 1) * kv_heads * dim].view(tokens, kv_heads, dim) for i in (1, 2))
        return _empty_cache(case, blocks) | {"case": dict(case), "k": k, "v": v, "slots": slots, "kept": kept}
    lengths = _lengths(case)
    state = _full_cache(case, lengths, gen) | {"case": dict(case)}
    if case["op"] == "read":
        ends = [0]
        for n in lengths:
            ends.append(ends[-1] + n)
        state["cu_seqlens"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        state["total"] = ends[-1]
        return state
    state["context_lens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    # the queries, like the keys, are a slice of the projection's output
    qkv = torch.randn(case["batch"], (case["heads"] + 2 * kv_heads) * dim, generator=gen, device="cuda") * 1.5
    state["q"] = qkv.to(torch.bfloat16)[:, :case["heads"] * dim].view(case["batch"], case["heads"], dim)
    state["out_scale"] = torch.tensor(OUT_SCALE, device="cuda") if case["codes"] else None
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return _own[op](state)
    return _plain[op](state)


def _rows(state, name, blocks, offsets):
    """Rows of the cache in 32 bits."""
    x = _bytes_of(state[name + "_cache"])[blocks, offsets]
    if state[name + "_scale"] is None:
        return x.float()
    return x.view(FP8).float() * state[name + "_scale"][blocks, offsets][..., None]


def _plain_attend(state):
    case, tables, lengths = state["case"], state["block_tables"], state["context_lens"]
    batch, kv_heads, dim = case["batch"], case["kv_heads"], case["dim"]
    longest = tables.shape[1] * case["block"]
    at = torch.arange(longest, device="cuda")
    blocks = tables.clamp(min=0).long()[:, at // case["block"]]
    k = _rows(state, "k", blocks, at % case["block"]).permute(0, 2, 3, 1)
    q = state["q"].float().view(batch, kv_heads, -1, dim)
    s = (q @ k) * dim ** -0.5
    del k
    inside = (at < lengths[:, None])[:, None, None, :]
    s = s.masked_fill(~inside, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    total = p.sum(-1, keepdim=True)
    v = _rows(state, "v", blocks, at % case["block"]).permute(0, 2, 1, 3)
    v = v.masked_fill(~inside.view(batch, 1, -1, 1), 0.0)
    o = (p @ v / total.masked_fill(total == 0, 1.0)).to(torch.bfloat16).view(batch, case["heads"], dim)
    if not case["codes"]:
        return o
    return (o.float() / state["out_scale"]).clamp(-FP8_MAX, FP8_MAX).to(FP8)


def _plain_write(state):
    kept, block = state["kept"], state["case"]["block"]
    slots = state["slots"][:kept].long()
    for name in ("k", "v"):
        cache = _bytes_of(state[name + "_cache"])
        if state[name + "_scale"] is None:
            cache[slots // block, slots % block] = state[name][:kept]
        else:
            codes, scale = _quantised(state[name][:kept])
            cache[slots // block, slots % block] = _bytes_of(codes)
            state[name + "_scale"][slots // block, slots % block] = scale
    return _cache_of(state)


def _plain_read(state):
    cu, block = state["cu_seqlens"].long(), state["case"]["block"]
    row = torch.arange(state["total"], device="cuda")
    b = torch.searchsorted(cu, row, right=True) - 1
    at = row - cu[b]
    blocks = state["block_tables"][b, at // block].long()
    return tuple(_rows(state, name, blocks, at % block).to(torch.bfloat16) for name in ("k", "v"))


def _cache_of(state):
    return {name: state[name] for name in ("k_cache", "v_cache", "k_scale", "v_scale") if state[name] is not None}


def _own_attend(state):
    out = _kernels().paged_attention(state["q"], state["k_cache"], state["v_cache"], state["block_tables"], state["context_lens"],
                                     k_scale=state["k_scale"], v_scale=state["v_scale"], out_scale=state["out_scale"])
    return out.view(FP8) if state["case"]["codes"] else out


def _own_write(state):
    _kernels().kv_cache_write(state["k"], state["v"], state["slots"], state["k_cache"], state["v_cache"], state["k_scale"],
                              state["v_scale"])
    return _cache_of(state)


def _own_read(state):
    return _kernels().kv_cache_read(state["k_cache"], state["v_cache"], state["block_tables"], state["cu_seqlens"], state["total"],
                                    k_scale=state["k_scale"], v_scale=state["v_scale"])


_plain = {"attend": _plain_attend, "write": _plain_write, "read": _plain_read}
_own = {"attend": _own_attend, "write": _own_write, "read": _own_read}


def work(case):
    kv_heads, dim = case["kv_heads"], case["dim"]
    cached = dim + 4 if case["cache"] == "e4m3" else 2 * dim             # bytes of one token's keys (or values) of one head
    if case["op"] == "write":
        kept = case["tokens"] - case["padding"]
        return {"bytes": 2 * kept * kv_heads * (2 * dim + cached) + 4 * case["tokens"], "flops": 0}
    lengths = _lengths(case)
    total = sum(lengths)
    pages = sum(-(-n // case["block"]) for n in lengths)
    read = 2 * total * kv_heads * cached + 4 * pages + 4 * len(lengths)
    if case["op"] == "read":
        return {"bytes": read + 2 * total * kv_heads * 2 * dim, "flops": 0}
    return {"bytes": read + case["batch"] * case["heads"] * dim * (3 if case["codes"] else 4), "flops": 4 * total * case["heads"] * dim}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"attend": _exact_attend, "write": _exact_write, "read": _exact_read}[case["op"]](case, state)


def _exact_rows(state, name, b, n):
    """The first n tokens of sequence b: [n, kv_heads, dim] in 64 bits."""
    block = state["case"]["block"]
    pages = state["block_tables"][b, :-(-n // block)].tolist()
    raw = _bytes_of(state[name + "_cache"])
    x = torch.cat([raw[p] for p in pages])[:n]
    if state[name + "_scale"] is None:
        return x.double()
    scale = torch.cat([state[name + "_scale"][p] for p in pages])[:n]
    return x.view(FP8).double() * scale.double()[..., None]


def _exact_attend(case, state):
    o = torch.zeros(case["batch"], case["heads"], case["dim"], dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for b, n in enumerate(_lengths(case)):
        if n:
            k, v = (_exact_rows(state, name, b, n) for name in ("k", "v"))
            for h in range(case["kv_heads"]):
                own_heads = slice(h * group, (h + 1) * group)
                weights = torch.softmax(state["q"][b, own_heads].double() @ k[:, h].T / math.sqrt(case["dim"]), -1)
                o[b, own_heads] = weights @ v[:, h]
    return (o / state["out_scale"].double()).clamp(-FP8_MAX, FP8_MAX) if case["codes"] else o


def _exact_write(case, state):
    out = {}
    slots = state["slots"][:state["kept"]].long()
    for name in ("k", "v"):
        cache = torch.zeros(state[name + "_cache"].shape, dtype=torch.float64, device="cuda")
        x = state[name][:state["kept"]].double()
        if state[name + "_scale"] is not None:
            scale = torch.clamp(x.abs().max(-1).values, min=1e-8) / FP8_MAX
            scales = torch.zeros(cache.shape[:3], dtype=torch.float64, device="cuda")
            scales[slots // case["block"], slots % case["block"]] = scale
            out[name + "_scale"] = scales
            x = x / scale[..., None]
        cache[slots // case["block"], slots % case["block"]] = x
        out[name + "_cache"] = cache
    return out


def _exact_read(case, state):
    rows = [(b, n) for b, n in enumerate(_lengths(case)) if n]
    return tuple(torch.cat([_exact_rows(state, name, b, n) for b, n in rows]) for name in ("k", "v"))
