"""Serving operators whose time is tracked: a paged cache of keys and values, in 16 or 32 bits and in 4.

    rope_append, rope_append_mxfp4   1 to 16384 new tokens, rotated at their positions and written to their slots
    attn_paged, attn_paged_mxfp4     1 to 64 sequences of 1 to 2048 new tokens over 1 to 131072 cached ones

A case is one call: its sizes and its type. `listed()` holds fixed cases, `draw(rng)` gives more of the same ranges,
`prepare` makes what a serving program holds before the call, `run` is the call, in plain torch or (with `own`) by the
framework's operators, `work` the bytes and operations it cannot do without and `exact` its outputs in float64.

The cache is [pages, kv_heads, page, head_dim]. In 4 bits it is MXFP4: two e2m1 codes to a byte along head_dim, the even
channel low, and for every 32 channels the exponent of their scale, scales [pages, kv_heads, head_dim / 32, page].
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 500000.0
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed() -> list[dict]:
    return [
        # one decode step of 32 requests: what counts is the latency of the call
        {"name": "append_step", "op": "rope_append", "dtype": "bf16", "tokens": 32, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "half": 64, "interleaved": False, "page": 16, "positions": 32768, "padded": False},
        # a packed batch of prompts entering the cache
        {"name": "append_prompt", "op": "rope_append", "dtype": "bf16", "tokens": 16384, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "half": 64, "interleaved": False, "page": 64, "positions": 8192, "padded": False},
        # fp32, a partial rotation of neighbouring pairs, odd counts, a page that is no power of two, padding tokens
        {"name": "append_odd", "op": "rope_append", "dtype": "fp32", "tokens": 1003, "q_heads": 15, "kv_heads": 5,
         "head_dim": 80, "half": 20, "interleaved": True, "page": 48, "positions": 4096, "padded": True},
        # a decode step into the 4-bit cache
        {"name": "append4_step", "op": "rope_append_mxfp4", "dtype": "bf16", "tokens": 64, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "half": 64, "interleaved": False, "page": 16, "positions": 32768, "padded": False},
        # prompts into the 4-bit cache
        {"name": "append4_prompt", "op": "rope_append_mxfp4", "dtype": "bf16", "tokens": 8192, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "half": 64, "interleaved": False, "page": 64, "positions": 8192, "padded": False},
        # one request early in its answer: eight blocks' worth of work, all latency
        {"name": "decode_short", "op": "attn_paged", "dtype": "bf16", "seqs": 1, "new": 1, "shortest": 500,
         "longest": 500, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "causal": True},
        # a decode step of 64 requests of very different lengths
        {"name": "decode_batch", "op": "attn_paged", "dtype": "bf16", "seqs": 64, "new": 1, "shortest": 200,
         "longest": 8192, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "causal": True},
        # two long documents answered at once: few rows, a long axis
        {"name": "decode_long", "op": "attn_paged", "dtype": "fp16", "seqs": 2, "new": 1, "shortest": 120001,
         "longest": 131071, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "causal": True},
        # chunks of prompts over what is cached of them
        {"name": "chunk_prompt", "op": "attn_paged", "dtype": "bf16", "seqs": 4, "new": 2048, "shortest": 4096,
         "longest": 8192, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "causal": True},
        # a few drafted tokens a request checked at once, in fp32, without grouped heads
        {"name": "verify_fp32", "op": "attn_paged", "dtype": "fp32", "seqs": 12, "new": 5, "shortest": 100,
         "longest": 1531, "q_heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "causal": True},
        # a decode step of 48 requests over the 4-bit cache
        {"name": "decode4_batch", "op": "attn_paged_mxfp4", "dtype": "bf16", "seqs": 48, "new": 1, "shortest": 1000,
         "longest": 32768, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "causal": True},
        # chunks over the 4-bit cache, fp16, groups of 7, a width between the powers of two
        {"name": "chunk4_odd", "op": "attn_paged_mxfp4", "dtype": "fp16", "seqs": 3, "new": 300, "shortest": 5000,
         "longest": 20011, "q_heads": 28, "kv_heads": 4, "head_dim": 96, "page": 128, "causal": True},
    ]


def _log_int(rng: random.Random, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(("rope_append", "rope_append_mxfp4") + 2 * ("attn_paged", "attn_paged_mxfp4"))
    four = op.endswith("mxfp4")
    group = rng.choice((1, 2, 3, 4, 4, 5, 7, 8, 16))
    kv_heads = rng.choice([n for n in (1, 2, 3, 4, 5, 8, 8, 12) if n * group <= 64])
    head_dim = rng.choice((32, 64, 64, 96, 128, 128, 128, 192, 256) + (() if four else (40, 80)))
    case = {"op": op, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "q_heads": kv_heads * group,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": rng.choice((16, 16, 32, 48, 64, 128, 256))}
    e = 4 if case["dtype"] == "fp32" else 2
    if op.startswith("rope"):
        row = (case["q_heads"] + 2 * kv_heads) * head_dim * e
        most = (16384 if not four else 8192) * 48 * 128 * 2 // row  # the listed prompt's bytes
        case["tokens"] = _log_int(rng, 1, min(16384, max(1, most)))
        case["half"] = rng.choice((head_dim // 2, head_dim // 2, head_dim // 4))
        case["interleaved"] = rng.random() < 0.3
        case["positions"] = _log_int(rng, 64, 131072)
        case["padded"] = rng.random() < 0.3
        return case
    case["causal"] = rng.random() < 0.8
    new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 2048)
    case["seqs"] = _log_int(rng, 1, 64) if new == 1 else _log_int(rng, 1, 16)
    # at most about a third of the listed chunk's operations (a sixteenth of the rate in fp32), and twice the listed caches'
    # bytes
    ops = 1e11 if case["dtype"] != "fp32" else 6e9
    keys = min(131072, int(ops / (4 * head_dim * case["q_heads"] * new * case["seqs"])),
               int((2e9 if not four else 5e8) / (2 * kv_heads * head_dim * (0.55 if four else e) * case["seqs"])))
    if keys < new:  # as many tokens as can see each other
        keys = new = max(1, min(new, int(math.sqrt(ops / (4 * head_dim * case["q_heads"] * case["seqs"])))))
    case["longest"] = _log_int(rng, new, keys)
    case["shortest"] = max(1, case["longest"] // rng.choice((1, 2, 10, 50)))
    case["new"] = new
    return case


# ------------------------------------------------------------------ inputs


def _spread(case: dict) -> tuple[list[int], list[int]]:
    """Cached keys of every sequence, new ones among them, and its new tokens: the longest first, then over the range."""
    rng = random.Random(case["seqs"] * 1000003 + case["longest"])
    keys = [case["longest"]] + [_log_int(rng, case["shortest"], case["longest"]) for _ in range(case["seqs"] - 1)]
    new = [case["new"]] + [rng.randint(1, case["new"]) for _ in range(case["seqs"] - 1)]
    return keys, [min(n, k) for n, k in zip(new, keys)]


def _angles(count: int, half: int, dev: torch.device) -> torch.Tensor:
    freq = THETA ** (-torch.arange(half, device=dev, dtype=torch.float64) / max(half, 1))
    return torch.arange(count, device=dev, dtype=torch.float64)[:, None] * freq


def _rows_of(slots: torch.Tensor, page: int) -> tuple[torch.Tensor, torch.Tensor]:
    return torch.div(slots, page, rounding_mode="floor"), slots % page


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, op, page = DTYPES[case["dtype"]], case["op"], case["page"]
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)

    state = {"case": case}
    if op.startswith("rope"):
        tokens = case["tokens"]
        pages = 2 * -(-tokens // page) + 8
        qkv = randn(tokens, hq + 2 * hkv, d)  # one packed projection; q, k and v are views of it
        state["q"], state["k"], state["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        angles = _angles(case["positions"], case["half"], dev)
        state["cos"], state["sin"] = angles.cos().float(), angles.sin().float()
        if tokens <= 64:  # a decode step: each token in a sequence of its own, anywhere
            state["positions"] = torch.randint(0, case["positions"], (tokens,), generator=gen, device=dev)
            state["slots"] = torch.randperm(pages * page, generator=gen, device=dev)[:tokens]
        else:  # prompts: runs of tokens over pages in any order
            at = torch.arange(tokens, device=dev)
            order = torch.randperm(pages, generator=gen, device=dev)
            state["positions"] = at % case["positions"]
            state["slots"] = order[at // page] * page + at % page
        if case["padded"]:
            state["slots"] = torch.where(torch.rand(tokens, generator=gen, device=dev) < 0.1, -1, state["slots"])
        if op == "rope_append":
            state["k_cache"], state["v_cache"] = randn(pages, hkv, page, d), randn(pages, hkv, page, d)
        else:
            for name in ("k", "v"):
                state[name + "_codes"], state[name + "_scales"] = _quantised(randn(pages, hkv, page, d).float())
        return state
    keys, new = _spread(case)
    held = [-(-n // page) for n in keys]
    order = torch.randperm(sum(held) + 8, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(len(keys), max(held), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    state["block_table"] = table
    state["cache_lens"] = torch.tensor(keys, dtype=torch.int32, device=dev)
    state["q"] = randn(sum(new), hq, d)
    cuts = [0]
    for n in new:
        cuts.append(cuts[-1] + n)
    state["cu_seqlens"] = None if case["new"] == 1 else torch.tensor(cuts, dtype=torch.int32, device=dev)
    state["longest"], state["most_new"] = max(keys), max(new)
    if op == "attn_paged":
        state["k_cache"], state["v_cache"] = randn(len(order), hkv, page, d), randn(len(order), hkv, page, d)
    else:
        for name in ("k", "v"):
            state[name + "_codes"], state[name + "_scales"] = _quantised(randn(len(order), hkv, page, d).float())
    return state


# ------------------------------------------------------------------ the plain forms


def _quantised(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """y [pages, heads, page, d] as MXFP4: codes [pages, heads, page, d / 2] and scales [pages, heads, d / 32, page]."""
    blocks = y.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    exponent = torch.where(top > 0, torch.frexp(top).exponent - 3, -126).clamp(min=-126)
    fine = top.isfinite()
    scale = torch.where(fine, exponent + 127, 255).to(torch.uint8)
    m = torch.ldexp(blocks.abs(), -exponent[..., None])
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)
            + 8 * blocks.signbit())
    code = torch.where(fine[..., None], code, 0).to(torch.uint8).flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] | code[..., 1] << 4, scale.transpose(-1, -2).contiguous()


def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes [..., d / 2] with scales [..., d / 32] stand for, in float32."""
    grid = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=torch.float32, device=codes.device)
    pairs = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    scale = torch.ldexp(torch.ones((), device=codes.device), scales.to(torch.int32) - 127)
    scale = torch.where(scales == 255, float("nan"), scale)
    return (grid[pairs.int()].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _turned(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x [tokens, heads, d] rotated by cos, sin [tokens, half] of its own type."""
    half = cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        u, v = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack((u * c - v * s, v * c + u * s), dim=-1).flatten(-2)
    else:
        u, v = x[..., :half], x[..., half:2 * half]
        y = torch.cat((u * c - v * s, v * c + u * s), dim=-1)
    return torch.cat((y, x[..., 2 * half:]), dim=-1)


def _plain_append(state: dict):
    case, page = state["case"], state["case"]["page"]
    q, k, v, dtype = state["q"], state["k"], state["v"], state["q"].dtype
    cos, sin = state["cos"][state["positions"]], state["sin"][state["positions"]]
    yq = _turned(q.float(), cos, sin, case["interleaved"]).to(dtype)
    kept = state["slots"] >= 0 if case["padded"] else slice(None)
    at, off = _rows_of(state["slots"][kept], page)
    if case["op"] == "rope_append":
        yk = _turned(k.float(), cos, sin, case["interleaved"]).to(dtype)
        state["k_cache"][at, :, off] = yk[kept]
        state["v_cache"][at, :, off] = v[kept]
        return {"yq": yq, "yk": yk, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    # a rotated key may lie next to a border between two codes: 64 bits
    rows = {"k": _turned(k.double(), cos.double(), sin.double(), case["interleaved"]), "v": v.double()}
    out = {"yq": yq}
    for name, y in rows.items():
        codes, scales = _quantised(y[:, :, None])  # pages of one token
        out["y" + name] = _values(codes[:, :, 0], scales[..., 0]).to(dtype)
        state[name + "_codes"][at, :, off] = codes[kept, :, 0]
        state[name + "_scales"][at, :, :, off] = scales[kept, :, :, 0]
        out[name + "_codes"], out[name + "_scales"] = state[name + "_codes"], state[name + "_scales"]
    return out


def _plain_attention(state: dict):
    case, page = state["case"], state["case"]["page"]
    q, lens, table = state["q"], state["cache_lens"].long(), state["block_table"].long()
    total, hq, d = q.shape
    hkv, seqs, dev = case["kv_heads"], lens.numel(), q.device
    cuts = torch.arange(seqs + 1, device=dev) if state["cu_seqlens"] is None else state["cu_seqlens"].long()
    key = torch.arange(state["longest"], device=dev)
    at, off = table[:, key // page], (key % page).expand(seqs, -1)
    if case["op"] == "attn_paged":
        k, v = state["k_cache"][at, :, off].float(), state["v_cache"][at, :, off].float()
    else:
        k = _values(state["k_codes"][at, :, off], state["k_scales"][at, :, :, off])
        v = _values(state["v_codes"][at, :, off], state["v_scales"][at, :, :, off])
    k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()  # [seqs, hkv, keys, d]
    # every sequence's queries, padded to the longest run: [seqs, hkv, most_new * group, d]
    token = torch.arange(total, device=dev)
    seq = (token[:, None] >= cuts[None, 1:]).sum(1)
    turn = token - cuts[seq]
    padded = torch.zeros(seqs, state["most_new"], hq, d, device=dev)
    padded[seq, turn] = q.float()
    rows = padded.unflatten(2, (hkv, -1)).transpose(1, 2).flatten(2, 3)
    s = torch.matmul(rows, k.transpose(-1, -2).contiguous()) * d ** -0.5
    last = lens[:, None] - 1
    if case["causal"]:
        last = last - (cuts[1:] - cuts[:-1])[:, None] + 1 + torch.arange(state["most_new"], device=dev)
    else:
        last = last.expand(-1, state["most_new"])
    seen = (key <= last[..., None])[:, None, :, None].expand(-1, hkv, -1, hq // hkv, -1).flatten(2, 3)
    s = torch.where(seen, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - top), 0.0)
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = torch.where(seen.any(-1, keepdim=True), o, 0.0)
    o = o.unflatten(2, (state["most_new"], -1)).transpose(1, 2).flatten(2, 3)
    return {"o": o[seq, turn].to(q.dtype)}


def run(state: dict):
    op = state["case"]["op"]
    if not own:
        return _plain_append(state) if op.startswith("rope") else _plain_attention(state)
    from popcorn_amd import impls

    if op == "rope_append":
        yq, yk = impls.rope_append(state["q"], state["k"], state["v"], state["cos"], state["sin"], state["positions"],
                                   state["slots"], state["k_cache"], state["v_cache"], state["case"]["interleaved"])
        return {"yq": yq, "yk": yk, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    if op == "rope_append_mxfp4":
        yq, yk, yv = impls.rope_append_mxfp4(state["q"], state["k"], state["v"], state["cos"], state["sin"],
                                             state["positions"], state["slots"], state["k_codes"], state["k_scales"],
                                             state["v_codes"], state["v_scales"], state["case"]["interleaved"])
        return {"yq": yq, "yk": yk, "yv": yv, "k_codes": state["k_codes"], "k_scales": state["k_scales"],
                "v_codes": state["v_codes"], "v_scales": state["v_scales"]}
    if op == "attn_paged":
        return {"o": impls.attn_paged(state["q"], state["k_cache"], state["v_cache"], state["block_table"],
                                      state["cache_lens"], state["cu_seqlens"], state["case"]["causal"])}
    return {"o": impls.attn_paged_mxfp4(state["q"], state["k_codes"], state["k_scales"], state["v_codes"],
                                        state["v_scales"], state["block_table"], state["cache_lens"],
                                        state["cu_seqlens"], state["case"]["causal"])}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case: dict) -> dict:
    """Appending: q, k and v in, the rotated ones out, the cache's rows out, a row of each table and the two indices a
    token. Attention: the cached keys and values that exist, once; q in, o out; the products of every pair that is seen."""
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    e = 4 if case["dtype"] == "fp32" else 2
    held = 0.5 * d + d // 32 if case["op"].endswith("mxfp4") else d * e  # one cached row of one head
    if case["op"].startswith("rope"):
        values = 2 * hq + 2 * hkv + (2 if case["op"] == "rope_append_mxfp4" else 1) * hkv
        return {"bytes": case["tokens"] * (values * d * e + 2 * hkv * held + 8 * case["half"] + 16),
                "flops": case["tokens"] * (6 * (hq + hkv) * case["half"])}
    keys, new = _spread(case)
    pairs = sum(n * k - (n * (n - 1) // 2 if case["causal"] else 0) for k, n in zip(keys, new))
    table = 4 * sum(-(-k // case["page"]) for k in keys)
    return {"bytes": sum(keys) * 2 * hkv * held + 2 * sum(new) * hq * d * e + table,
            "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------ the same outputs in 64 bits


def _nearest(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """For float64 y [..., d]: the value each element is held as, and the exponent byte of every 32."""
    blocks = y.reshape(*y.shape[:-1], y.shape[-1] // 32, 32)
    top = blocks.abs().max(dim=-1, keepdim=True).values
    power = torch.floor(torch.log2(top.clamp(min=2.0 ** -200)))
    # log2 may round over a power of two
    power = power + (torch.exp2(power + 1) <= top).double() - (torch.exp2(power) > top).double()
    power = (power - 2).clamp(min=-126)
    grid = torch.tensor(E2M1, dtype=torch.float64, device=y.device)
    borders = (grid[1:] + grid[:-1]) / 2
    m = blocks.abs() * torch.exp2(-power)
    at = torch.bucketize(m, borders)  # borders below m: a tie stays under its border
    tie = (at < 7) & (m == borders[at.clamp(max=6)]) & (at % 2 == 1)
    held = torch.copysign(grid[at + tie.long()], blocks) * torch.exp2(power)
    return held.reshape(y.shape), power[..., 0] + 127


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    page, hkv = case["page"], case["kv_heads"]
    if case["op"].startswith("rope"):
        turn = torch.complex(state["cos"].double(), state["sin"].double())[state["positions"]][:, None]
        half = case["half"]

        def rotated(x):
            x = x.double()
            first = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
            second = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
            z = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        yq, yk, yv = rotated(state["q"]), rotated(state["k"]), state["v"].double()
        kept = torch.nonzero(state["slots"] >= 0)[:, 0]
        at, off = _rows_of(state["slots"][kept], page)
        if case["op"] == "rope_append":
            caches = state["k_cache"].double(), state["v_cache"].double()
            for cache, y in zip(caches, (yk, yv)):
                cache[at, :, off] = y[kept]
            return {"yq": yq, "yk": yk, "k_cache": caches[0], "v_cache": caches[1]}
        return {"yq": yq, "yk": _nearest(yk)[0], "yv": _nearest(yv)[0], "k_codes": None, "k_scales": None,
                "v_codes": None, "v_scales": None}
    keys, new = _spread(case)
    out, first = torch.empty(state["q"].shape, dtype=torch.float64, device=state["q"].device), 0
    group = case["q_heads"] // hkv
    for i, (length, count) in enumerate(zip(keys, new)):
        pages = state["block_table"][i, :-(-length // page)].long()
        last = length - count + torch.arange(count, device=out.device) if case["causal"] else torch.full(
            (count,), length - 1, device=out.device)
        hidden = torch.arange(length, device=out.device)[None] > last[:, None]
        for h in range(hkv):
            if case["op"] == "attn_paged":
                k, v = (state[n][pages, h].flatten(0, 1).double() for n in ("k_cache", "v_cache"))
            else:
                k, v = (_held(state[n + "_codes"][pages, h], state[n + "_scales"][pages, h]) for n in ("k", "v"))
            kt, v = k[:length].t().contiguous(), v[:length]
            for g in range(group):
                s = state["q"][first:first + count, h * group + g].double() @ kt / math.sqrt(case["head_dim"])
                out[first:first + count, h * group + g] = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1) @ v
        first += count
    return {"o": out}


def _held(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 rows [pages * page, d] of codes [pages, page, d / 2] with scales [pages, d / 32, page]."""
    two = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.int64, device=codes.device)
    two[..., 0::2], two[..., 1::2] = (codes % 16).long(), (codes // 16).long()
    size = torch.tensor(E2M1, dtype=torch.float64, device=codes.device)[two % 8]
    value = torch.where(two >= 8, -size, size)
    power = torch.exp2(scales.double() - 127.0).permute(0, 2, 1).repeat_interleave(32, dim=-1)
    return (value * power).flatten(0, 1)
