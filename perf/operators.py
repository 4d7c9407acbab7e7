"""Workloads of attention over a paged cache, of writing that cache and of reading it back.

Every case is one call as a serving program makes it.  "attend": new tokens of a batch of sequences attend to what the
cache holds of them, themselves among it.  "write": keys and values of new tokens go to their places in the cache, as they
are or in 8 bits with a scale for each token and head.  "read": the cache's keys and values come back as dense tensors.

Import with the repository's root as the working folder.
"""
import functools
import math
import os
import random
import sys

import numpy as np
import torch

own = False  # whether run() calls the package's operators or computes their plain form

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
E4M3_MAX = 448.0
LARGEST_KEPT = {"f16": 61440.0, "bf16": 1.875 * 2.0 ** 127}  # a type's largest value of 4 significant bits


def _case(name, op, batch, new, length, heads, kv_heads, dim, dtype, cache, page, spread=0.0, chunks=0, causal=True):
    """new: new tokens of a sequence; length: most keys of a sequence; spread: sequences are up to that share shorter;
    chunks: so many sequences have `new` new tokens, the others one each, and all are packed (0: all have `new`, padded to
    the same length); cache: "same" as dtype or "e4m3"; page: positions of a page."""
    return {"name": name, "op": op, "batch": batch, "new": new, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "cache": cache, "page": page, "spread": spread, "chunks": chunks, "causal": causal}


def listed():
    return [
        # one user, next token of a small model's short text: launches are all there is
        _case("attend_b1_n1_l77_h8_d64_f16", "attend", 1, 1, 77, 8, 8, 64, "f16", "same", 16),
        # a few drafted tokens of four users looked at together, one key head for each query head
        _case("attend_b4_n6_l1500_h12_d64_bf16", "attend", 4, 6, 1500, 12, 12, 64, "bf16", "same", 32, 0.3),
        # next tokens of a few users at a medium context, grouped heads
        _case("attend_b8_n1_l4096_h32_kv8_d128_bf16", "attend", 8, 1, 4096, 32, 8, 128, "bf16", "same", 16, 0.5),
        # next tokens of many users of all lengths, cache in 8 bits
        _case("attend_b32_n1_l8192_h32_kv8_d128_bf16_e4m3", "attend", 32, 1, 8192, 32, 8, 128, "bf16", "e4m3", 64, 0.95),
        # next token of one user with a very long context
        _case("attend_b1_n1_l131072_h32_kv8_d128_f16", "attend", 1, 1, 131072, 32, 8, 128, "f16", "same", 128),
        # a chunk of one user's prompt, the rest of which is in the cache
        _case("attend_b1_n512_l8192_h32_kv8_d128_f16", "attend", 1, 512, 8192, 32, 8, 128, "f16", "same", 64),
        # a step of continuous batching: two chunks of prompts of no round length among single tokens, cache in 8 bits
        _case("attend_b16_n731_l4001_h20_kv4_d128_bf16_e4m3_packed", "attend", 16, 731, 4001, 20, 4, 128, "bf16", "e4m3", 16, 0.6, 2),
        # a large chunk deep in a long document: the largest call
        _case("attend_b1_n4096_l32768_h32_kv8_d128_f16", "attend", 1, 4096, 32768, 32, 8, 128, "f16", "same", 128),
        # the write of a step of next tokens
        _case("write_b64_n1_kv8_d128_bf16", "write", 64, 1, 2048, 32, 8, 128, "bf16", "same", 16, 0.9),
        # the write of a prompt, in 8 bits
        _case("write_b3_n8192_kv8_d128_bf16_e4m3_packed", "write", 3, 8192, 8192, 32, 8, 128, "bf16", "e4m3", 64, 0.2, 2),
        # one short sequence's cache as dense tensors
        _case("read_b1_l1500_kv12_d64_f16", "read", 1, 1, 1500, 12, 12, 64, "f16", "same", 16),
        # a batch of long ones out of 8 bits
        _case("read_b4_l8192_kv8_d128_bf16_e4m3", "read", 4, 1, 8192, 32, 8, 128, "bf16", "e4m3", 64, 0.5),
    ]


def _lengths(case):
    """(keys, new tokens) of each sequence."""
    rng = random.Random(case["length"] * 31 + case["batch"])
    keys = [case["length"]] + [max(1, round(case["length"] * (1 - case["spread"] * rng.random()))) for _ in range(case["batch"] - 1)]
    some = case["chunks"]
    new = [case["new"] if not some or i < some else 1 for i in range(case["batch"])]
    return keys, [min(n, m) for n, m in zip(new, keys)] if some else [min(case["new"], min(keys))] * case["batch"]


def _pairs(case):
    """(query, visible key) pairs of one head."""
    keys, new = _lengths(case)
    return sum(n * m - (n * (n - 1) // 2 if case["causal"] else 0) for m, n in zip(keys, new))


def work(case):
    keys, new = _lengths(case)
    row = case["kv_heads"] * case["dim"]
    held = 2 * row * (2 if case["cache"] == "same" else 1) + (0 if case["cache"] == "same" else 2 * case["kv_heads"])  # of a position
    if case["op"] == "attend":
        return {"bytes": 4 * sum(new) * case["heads"] * case["dim"] + sum(keys) * held,
                "flops": 4 * _pairs(case) * case["heads"] * case["dim"]}
    if case["op"] == "write":
        return {"bytes": sum(new) * (4 * row + held), "flops": 0}
    return {"bytes": sum(keys) * held + 4 * case["batch"] * max(keys) * row, "flops": 0}


_MOST_FLOPS = 4 * 32 * 128 * (4096 * 32768 - 4096 * 4095 // 2)  # of the largest listed case
_MOST_HELD = 1 << 29                                            # values of K in a cache
_MOST_SCORES = 32 * 4096 * 32768                                # that the plain form holds


def draw(rng):
    """Another call of the same ranges: 1 to 64 sequences, 1 to 131072 keys, 1 to 8192 new tokens, 1 to 64 heads, up to 16
    of them to a key head."""
    log_int = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))
    while True:
        op = rng.choice(["attend", "attend", "attend", "write", "read"])
        kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        case = {"op": op, "batch": log_int(1, 64), "new": 1 if rng.random() < 0.4 else log_int(1, 8192), "length": log_int(1, 131072),
                "heads": kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 8, 16]), "kv_heads": kv_heads, "dim": rng.choice([64, 128]),
                "dtype": rng.choice(["f16", "bf16"]), "cache": rng.choice(["same", "e4m3"]), "page": rng.choice([16, 32, 48, 64, 128, 256]),
                "spread": rng.choice([0.0, 0.3, 0.95]), "chunks": 0, "causal": rng.random() < 0.8}
        if op != "read" and case["batch"] > 1 and case["new"] > 1 and rng.random() < 0.5:
            case["chunks"] = rng.randint(1, case["batch"])
        if op == "read":
            case["new"] = 1
        case["new"] = min(case["new"], case["length"])
        keys, new = _lengths(case)
        held = case["batch"] * max(keys) * case["kv_heads"] * case["dim"]
        scores = case["batch"] * max(new) * max(keys) * case["heads"]
        if case["heads"] > 64 or held > _MOST_HELD or (op == "read" and held > _MOST_HELD // 8):
            continue
        if op == "attend" and (scores > _MOST_SCORES or work(case)["flops"] > _MOST_FLOPS or held * 2 > _MOST_HELD):
            continue
        if op == "write" and sum(new) * case["kv_heads"] * case["dim"] > 1 << 26:
            continue
        return case


def _to_e4m3(x, dtype):
    """Rows in 8 bits and their scales 2^e, e the least integer, -126 or more, for which no value of x 2^-e is over 448."""
    most = LARGEST_KEPT[dtype]
    x = x.float().clamp(-most, most)
    m, e = torch.frexp(torch.nan_to_num(x, nan=0.0).abs().amax(-1, keepdim=True))
    e = torch.clamp(torch.where(m <= 0.875, e - 9, e - 8), min=-126)  # 448 = 0.875 * 2^9
    down = torch.bitwise_left_shift(127 - e, 23).view(torch.float32)  # 2^-e
    return (x * down).to(torch.float8_e4m3fn), (e[..., 0] + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, device="cuda", dtype=TYPES[case["dtype"]], generator=gen)
    ints = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)
    keys, new = _lengths(case)
    batch, page, heads, kv_heads, dim = (case[k] for k in ("batch", "page", "heads", "kv_heads", "dim"))
    width = -(-max(keys) // page)
    used = [-(-m // page) for m in keys]
    pages = sum(used) + 3  # some that belong to nobody
    order = torch.randperm(pages, device="cuda", generator=gen).int()
    filled = torch.arange(width, device="cuda")[None] < ints(used)[:, None]
    table = torch.full((batch, width), -1, device="cuda", dtype=torch.int32)
    table[filled] = order[:sum(used)]
    state = {"op": case["op"], "dtype": case["dtype"], "causal": case["causal"], "page_table": table, "cache_seqlens": ints(keys),
             "cu_seqlens": None, "max_seqlen": max(new), "longest": max(keys), "k_scale": None, "v_scale": None}
    # which tokens of a padded (batch, new tokens) grid there are
    state["present"] = torch.arange(max(new), device="cuda")[None] < ints(new)[:, None]
    if case["chunks"]:
        state["cu_seqlens"] = ints([0] + np.cumsum(new).tolist())
    lead = (sum(new),) if case["chunks"] else (batch, max(new))
    state["q"] = normal(*lead, heads, dim) if case["op"] == "attend" else None
    # keys with some channels much larger than the others, as models have them
    channels = torch.where(torch.rand(kv_heads, dim, device="cuda", generator=gen) < 0.05, 4.0, 1.0).to(TYPES[case["dtype"]])
    if case["op"] == "write":
        state["k"], state["v"] = normal(*lead, kv_heads, dim) * channels, normal(*lead, kv_heads, dim)
    for name in "kv":
        rows = normal(pages, page, kv_heads, dim)
        if name == "k":
            rows = rows * channels
        if case["cache"] == "e4m3":
            cache, scale = torch.empty_like(rows, dtype=torch.float8_e4m3fn), torch.empty(rows.shape[:3], dtype=torch.float8_e8m0fnu, device="cuda")
            step = max(1, (1 << 26) // rows[0].numel())
            for i in range(0, pages, step):
                cache[i:i + step], scale[i:i + step] = _to_e4m3(rows[i:i + step], case["dtype"])
            state[name + "_cache"], state[name + "_scale"] = cache, scale
        else:
            state[name + "_cache"] = rows
    return state


@functools.cache
def _package():
    sys.path.insert(0, os.path.join(os.getcwd(), "flash-attention-v100_amd"))
    import flash_attn_v100
    return flash_attn_v100


def _run_own(s):
    package = _package()
    scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if s["op"] == "attend":
        return package.flash_attn_paged_func(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["cache_seqlens"], None, s["causal"],
                                             cu_seqlens=s["cu_seqlens"], max_seqlen=s["max_seqlen"], **scales)
    if s["op"] == "write":
        package.kv_cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["cache_seqlens"],
                               cu_seqlens=s["cu_seqlens"], **scales)
        return {k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale") if s[k] is not None}
    return package.kv_cache_read(s["k_cache"], s["v_cache"], s["page_table"], s["cache_seqlens"], s["longest"],
                                 dtype=TYPES[s["dtype"]], **scales)


def _rows(s, name):
    """Keys or values in 32 bits, (batch, longest, kv heads, dim), with 0 behind each sequence."""
    cache, scale, page = s[name + "_cache"], s[name + "_scale"], s[name + "_cache"].shape[1]
    at = torch.arange(s["longest"], device=cache.device)
    slot = s["page_table"].clamp(min=0).long()[:, at // page] * page + at % page
    rows = cache.flatten(0, 1)[slot].float()
    if scale is not None:
        rows = rows * scale.flatten(0, 1)[slot].float()[..., None]
    return rows.masked_fill_((at >= s["cache_seqlens"][:, None])[..., None, None], 0.0)


def _attend(s):
    packed = s["cu_seqlens"] is not None
    q = s["q"]
    if packed:  # to a padded grid
        grid = torch.zeros((*s["present"].shape, *q.shape[1:]), device=q.device, dtype=torch.float32)
        grid[s["present"]] = q.float()
    else:
        grid = q.float()
    k, v = _rows(s, "k"), _rows(s, "v")
    (batch, new, heads, dim), kv_heads, longest = grid.shape, k.shape[2], k.shape[1]
    # (batch, kv heads, heads of one kv head x new tokens, keys)
    rows = grid.view(batch, new, kv_heads, -1, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, dim)
    scores = torch.matmul(rows, k.permute(0, 2, 3, 1).contiguous()).mul_(dim ** -0.5)
    n = s["present"].sum(1)
    last = s["cache_seqlens"][:, None] - 1 - ((n[:, None] - 1 - torch.arange(new, device=q.device)).clamp(min=0) if s["causal"] else 0)
    last = last.expand(batch, new)[:, None, None, :, None]
    scores.view(batch, kv_heads, -1, new, longest).masked_fill_(torch.arange(longest, device=q.device) > last, -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores, v.permute(0, 2, 1, 3).contiguous()).div_(total)
    out = out.view(batch, kv_heads, -1, new, dim).permute(0, 3, 1, 2, 4).reshape(batch, new, heads, dim)
    return (out[s["present"]] if packed else out).to(q.dtype)


def _write(s):
    page, new = s["k_cache"].shape[1], s["present"].shape[1]
    n = s["present"].sum(1)
    at = (s["cache_seqlens"] - n)[:, None] + torch.arange(new, device=n.device)
    slot = (s["page_table"].gather(1, (at // page).clamp(max=s["page_table"].shape[1] - 1)).long() * page + at % page)[s["present"]]
    for name in "kv":
        x, cache, scale = s[name].flatten(0, -3), s[name + "_cache"], s[name + "_scale"]
        if scale is not None:
            x, y = _to_e4m3(x, s["dtype"])
            scale.view(torch.uint8).flatten(0, 1)[slot] = y.view(torch.uint8)
            cache.view(torch.uint8).flatten(0, 1)[slot] = x.view(torch.uint8)
        else:
            cache.flatten(0, 1)[slot] = x
    return {k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale") if s[k] is not None}


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "attend":
        return _attend(state)
    if state["op"] == "write":
        return _write(state)
    return tuple(_rows(state, name).to(TYPES[state["dtype"]]) for name in "kv")


def exact(case, seed):
    """The same in 64 bits, sequence by sequence."""
    s = prepare(case, seed)
    keys, new = _lengths(case)
    page, dim = case["page"], case["dim"]

    def places(b, first, count):
        p = torch.arange(first, first + count, device="cuda")
        ids = s["page_table"][b].long()[torch.div(p, page, rounding_mode="floor")]
        return ids, p % page

    def held(name, b):
        ids, slots = places(b, 0, keys[b])
        x = s[name + "_cache"][ids, slots].double()
        return x if s[name + "_scale"] is None else x * s[name + "_scale"][ids, slots].double().unsqueeze(-1)

    if case["op"] == "read":
        out = []
        for name in "kv":
            x = torch.zeros(case["batch"], max(keys), case["kv_heads"], dim, device="cuda", dtype=torch.float64)
            for b in range(case["batch"]):
                x[b, :keys[b]] = held(name, b)
            out.append(x)
        return tuple(out)
    starts = [0] + np.cumsum(new).tolist()
    if case["op"] == "write":
        out = {}
        for name in "kv":
            cache, scale = s[name + "_cache"].double(), s[name + "_scale"]
            scale = None if scale is None else scale.double()
            for b in range(case["batch"]):
                ids, slots = places(b, keys[b] - new[b], new[b])
                x = (s[name][starts[b]:starts[b + 1]] if case["chunks"] else s[name][b]).double()
                if scale is not None:
                    x = x.clamp(-LARGEST_KEPT[case["dtype"]], LARGEST_KEPT[case["dtype"]])
                    m, e = np.frexp(x.abs().amax(-1).cpu().numpy() / E4M3_MAX)
                    unit = torch.from_numpy(np.ldexp(1.0, np.maximum(np.where(m > 0.5, e, e - 1), -126))).cuda()
                    y = x / unit.unsqueeze(-1)
                    at = np.frexp(y.abs().clamp(min=2.0 ** -6).cpu().numpy())[1] - 1  # 2^at <= |y| < 2^(at + 1)
                    step = torch.from_numpy(np.ldexp(1.0, at - 3)).cuda()  # from one e4m3 value to the next
                    x = torch.round(y / step) * step
                    scale[ids, slots] = unit
                cache[ids, slots] = x
            out[name + "_cache"] = cache
            if scale is not None:
                out[name + "_scale"] = scale
        return {k: out[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale") if k in out}
    q = s["q"]
    out = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    group = case["heads"] // case["kv_heads"]
    for b in range(case["batch"]):
        k, v = held("k", b), held("v", b)
        queries, results = (x[starts[b]:starts[b + 1]] if case["chunks"] else x[b] for x in (q, out))
        position = torch.arange(keys[b] - new[b], keys[b], device="cuda") if case["causal"] else torch.full((new[b],), keys[b] - 1, device="cuda")
        hidden = torch.arange(keys[b], device="cuda")[None] > position[:, None]
        for h in range(case["heads"]):
            x = queries[:, h].double() @ k[:, h // group].t().contiguous() / math.sqrt(dim)
            x.masked_fill_(hidden, -math.inf)
            results[:, h] = torch.softmax(x, -1) @ v[:, h // group].contiguous()
    return out
