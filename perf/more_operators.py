"""A decode step's cache in 4 bits and its per-head norms, as cases to be measured.

* ``append4``: new keys and values into a paged 4-bit cache (a scale and an
  offset per 64 values), queries and keys normalised per head and rotated in
  the same pass; the pages written are read back.
* ``norms``: the same norms and rotation in front of the 8-bit cache.
* ``attend4``: attention of the new tokens over the 4-bit cache.

With ``own`` false, ``run`` computes them in elementary torch operations in
fp32 (the norms' sums in 64 bits: they decide values next to a rounding
border), rounded once at the end; with ``own`` true it makes the calls a user
of ``se12_b200`` makes. Head counts and dimensions are those of the decoder
configurations in ``se12_b200/shapes.py``, and a small one with heads of 64.

The 4-bit layout (``PagedKvCache(kind="int4")``): a value is (u - 8) * scale +
offset, u a code of 4 bits, scale and offset FP16 per token, head and group of
64 dimensions; the values' tensor has a power of two 2^E per token and head
besides, which scale and offset are relative to. Codes of a row: words of 8
codes (the first in the lowest bits), word 8 g + r of the row at place r *
groups + g. ``k_scales`` [pages, heads, page, groups, 2]; ``v_scales`` [pages,
heads, page / 16, 32 * groups + 16]: of 16 tokens, for each two neighbours the
groups' scales and then offsets (the two tokens' side by side), and then E.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
QMAX = {"int8": 127.0, "e4m3": 448.0}
MIN_EXPONENT = -100
GROUP = 64
EPS = 1e-6
# (query heads, KV heads, head dimension) of the decoder configurations
HEADS = {"gemma2-2b": (8, 4, 256), "gemma2-9b": (16, 8, 256), "gemma2-27b": (32, 16, 128), "llama3.1-70b": (64, 8, 128),
         "small": (8, 2, 64)}
ROTARY_BASE = {"gemma2-2b": 1e4, "gemma2-9b": 1e4, "gemma2-27b": 1e4, "llama3.1-70b": 5e5, "small": 1e4}


# ------------------------------------------------------------------ cases


def listed() -> list:
    return [
        # the smallest call: one sequence's next token, straight from the fp32 output of the grouped q/k/v GEMV
        dict(name="append4-1", op="append4", model="gemma2-2b", page=16, kind="int4", dtype="fp32", norms=True, rotary="whole", seqs=1,
             shortest=40, longest=40, new_low=1, new_high=1, window=0, softcap=0.0),
        # a serving batch's next tokens, without norms
        dict(name="append4-64", op="append4", model="llama3.1-70b", page=64, kind="int4", dtype="fp32", norms=False, rotary="whole",
             seqs=64, shortest=5, longest=16000, new_low=1, new_high=1, window=0, softcap=0.0),
        # a batch of prompt chunks behind cached prefixes, ragged, BF16 projections (the exact mode's F.linear)
        dict(name="append4-prompts", op="append4", model="gemma2-9b", page=32, kind="int4", dtype="bf16", norms=True, rotary="whole",
             seqs=13, shortest=0, longest=3001, new_low=301, new_high=2043, window=0, softcap=0.0),
        # a serving batch's next tokens into the 8-bit cache, neighbouring pairs rotated
        dict(name="norms-64", op="norms", model="gemma2-27b", page=64, kind="int8", dtype="fp32", norms=True, rotary="neighbours",
             seqs=64, shortest=5, longest=16000, new_low=1, new_high=1, window=0, softcap=0.0),
        # prompt chunks into the 8-bit cache
        dict(name="norms-prompts", op="norms", model="llama3.1-70b", page=32, kind="e4m3", dtype="bf16", norms=True, rotary="whole",
             seqs=7, shortest=0, longest=3001, new_low=77, new_high=1021, window=0, softcap=0.0),
        # the smallest attention: a new conversation's second page
        dict(name="attend4-1-short", op="attend4", model="gemma2-2b", page=16, kind="int4", seqs=1, shortest=17, longest=17, new_low=1,
             new_high=1, window=0, softcap=50.0),
        # a local (sliding-window, capped) layer of a serving batch
        dict(name="attend4-16-window", op="attend4", model="gemma2-9b", page=32, kind="int4", seqs=16, shortest=301, longest=8191,
             new_low=1, new_high=1, window=4096, softcap=50.0),
        # a large serving batch, ragged lengths
        dict(name="attend4-64", op="attend4", model="llama3.1-70b", page=64, kind="int4", seqs=64, shortest=1000, longest=16384,
             new_low=1, new_high=1, window=0, softcap=0.0),
        # one very long conversation
        dict(name="attend4-1-long", op="attend4", model="gemma2-27b", page=128, kind="int4", seqs=1, shortest=131071, longest=131071,
             new_low=1, new_high=1, window=0, softcap=50.0),
        # drafted tokens to verify: a few queries per sequence
        dict(name="attend4-verify", op="attend4", model="llama3.1-70b", page=16, kind="int4", seqs=24, shortest=77, longest=4093,
             new_low=2, new_high=6, window=0, softcap=0.0),
        # prompt chunks behind a cached prefix
        dict(name="attend4-chunk", op="attend4", model="gemma2-9b", page=64, kind="int4", seqs=2, shortest=5000, longest=8191,
             new_low=509, new_high=509, window=0, softcap=50.0),
    ]


def log_uniform(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(("append4", "norms", "attend4", "attend4"))
    model = rng.choice(sorted(HEADS))
    page, seqs = rng.choice((16, 32, 64, 128)), log_uniform(rng, 1, 64)
    if op != "attend4":
        if rng.random() < 0.5:
            new_low = new_high = 1
        else:
            new_high = log_uniform(rng, 2, max(2, 16000 // seqs))
            new_low = rng.randint(1, new_high)
        longest = log_uniform(rng, 1, 16000)
        return dict(op=op, model=model, page=page, kind="int4" if op == "append4" else rng.choice(("int8", "e4m3")),
                    dtype=rng.choice(("fp32", "bf16")), norms=op == "norms" or rng.random() < 0.6,
                    rotary=rng.choice(("whole", "whole", "neighbours", "part")), seqs=seqs, shortest=rng.randint(0, longest),
                    longest=longest, new_low=new_low, new_high=new_high, window=0, softcap=0.0)
    how = rng.random()
    if how < 0.6:  # next tokens
        new_low = new_high = 1
    elif how < 0.8:  # drafted tokens
        new_low, new_high = 1, rng.randint(2, 8)
    else:  # prompt chunks
        seqs = min(seqs, 3)
        new_high = log_uniform(rng, 16, 340)
        new_low = rng.randint(1, new_high)
    longest = log_uniform(rng, max(16, new_high), 16384)
    case = dict(op=op, model=model, page=page, kind="int4", seqs=seqs, shortest=rng.randint(new_high, longest), longest=longest,
                new_low=new_low, new_high=new_high, window=rng.choice((0, 0, 512, 4096)), softcap=rng.choice((0.0, 50.0)))
    while work(case)["bytes"] > 4.5e8 or work(case)["flops"] > 1e11:
        case["seqs"] = max(1, case["seqs"] // 2)
        case["longest"] = max(new_high, case["longest"] * 3 // 4)
        case["shortest"] = min(case["shortest"], case["longest"])
    return case


def spread(low: int, high: int, count: int, step: float) -> list:
    """``count`` whole numbers over low..high in a fixed uneven order, the last one ``high``."""
    return [low + int((high - low) * ((i * step) % 1.0)) for i in range(count - 1)] + [high]


def new_tokens(case: dict) -> list:
    return spread(case["new_low"], case["new_high"], case["seqs"], 0.754877)


def lengths(case: dict) -> list:
    """Tokens in the cache once the new ones are in (appends: longest/shortest are the prefix before them)."""
    base = spread(case["shortest"], case["longest"], case["seqs"], 0.618034)
    return base if case["op"] == "attend4" else [b + n for b, n in zip(base, new_tokens(case))]


def rotary_dim(case: dict) -> int:
    d = HEADS[case["model"]][2]
    return d // 2 if case["rotary"] == "part" else d


def work(case: dict) -> dict:
    hq, hkv, d = HEADS[case["model"]]
    new, lens = new_tokens(case), lengths(case)
    t = sum(new)
    # codes, scales and offsets of one token of one KV head, keys and values
    token = d + 8 * (d // GROUP) + 2 if case["kind"] == "int4" else 2 * d
    if case["op"] != "attend4":
        pages = sum((ln - 1) // case["page"] - (ln - n) // case["page"] + 1 for n, ln in zip(new, lens))
        scales = 0 if case["kind"] == "int4" else 2 * pages * hkv * 4
        return {"bytes": t * (hq + 2 * hkv) * d * (4 if case["dtype"] == "fp32" else 2)  # queries, keys, values in
                + t * rotary_dim(case) * 4 + t * hq * d * 2  # cosines and sines in, rotated queries out
                + t * hkv * token + scales  # codes and scales out
                + pages * case["page"] * hkv * (token + 2 * d * 2) + scales,  # the pages read back: codes in, BF16 values out
                "flops": (6 if case["norms"] else 3) * t * (hq + 2 * hkv) * d}
    pairs = visible = 0
    for n, ln in zip(new, lens):
        first = max(0, ln - n + 1 - case["window"]) if case["window"] else 0
        visible += ln - first
        for p in range(ln - n, ln):
            pairs += min(p + 1, case["window"]) if case["window"] else p + 1
    return {"bytes": visible * hkv * token + 4 * t * hq * d, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ the caches in elementary operations


def power_of_two(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32, e whole numbers."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def fit_scale(amax: torch.Tensor, kind: str) -> torch.Tensor:
    """The power of two 2^e, e >= MIN_EXPONENT least, with amax <= QMAX 2^e."""
    half, e = torch.frexp(amax)  # amax = half 2^e, 0.5 <= half < 1
    q_half, q_e = math.frexp(QMAX[kind])
    e = torch.where(half <= q_half, e - q_e, e - q_e + 1)
    return power_of_two(torch.where(amax > 0, e, torch.full_like(e, MIN_EXPONENT)).clamp(min=MIN_EXPONENT))


def to_codes(x: torch.Tensor, kind: str) -> torch.Tensor:
    """Scaled values as codes: whole numbers of int8, or e4m3 bit patterns (both as int8 tensors)."""
    return torch.round(x).to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn).view(torch.int8)


def from_codes(c: torch.Tensor, kind: str) -> torch.Tensor:
    return c.to(torch.float32) if kind == "int8" else c.view(torch.float8_e4m3fn).to(torch.float32)


def quantise(x: torch.Tensor, values: bool) -> tuple:
    """x [..., d] as (codes 0..15 uint8 [..., d], scale and offset FP16 [..., groups], E int32 [...])."""
    exponent = torch.zeros(x.shape[:-1], dtype=torch.int32, device=x.device)
    if values:
        amax = x.abs().amax(-1)
        exponent = torch.where(amax > 0, torch.frexp(amax).exponent - 4, exponent - 30).clamp(min=-30)
        x = x * power_of_two(-exponent)[..., None]
    x = x.unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    scale = ((high - low) * (1.0 / 15.0)).to(torch.float16)
    offset = (low + 8.0 * scale.float()).to(torch.float16)
    inverse = torch.where(scale > 0, 1.0 / scale.float(), torch.zeros_like(low))
    u = (torch.round((x - offset.float()[..., None]) * inverse[..., None]) + 8.0).clamp(0.0, 15.0)
    return u.to(torch.uint8).flatten(-2), scale, offset, exponent


def pack(u: torch.Tensor) -> torch.Tensor:
    """Codes 0..15 [..., d] as bytes [..., d / 2] in the cache's order."""
    words = u.unflatten(-1, (-1, 8, 8)).transpose(-3, -2)  # [..., 8, groups, codes of a word]
    return (words[..., 0::2] | (words[..., 1::2] << 4)).flatten(-3)


def unpack(codes: torch.Tensor) -> torch.Tensor:
    """(u - 8) in fp32 [..., d] of bytes [..., d / 2]."""
    groups = codes.shape[-1] * 2 // GROUP
    words = codes.unflatten(-1, (8, groups, 4)).transpose(-3, -2)
    return torch.stack((words & 15, words >> 4), dim=-1).flatten(-4).to(torch.float32) - 8.0


def key_pages(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Keys in fp32 [..., page, d] of 4-bit pages."""
    x = unpack(codes).unflatten(-1, (-1, GROUP))
    return (x * scales[..., 0].float()[..., None] + scales[..., 1].float()[..., None]).flatten(-2)


def value_pages(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Values in fp32 [..., page, d] of 4-bit pages."""
    groups = codes.shape[-1] * 2 // GROUP
    pairs = scales[..., : 32 * groups].unflatten(-1, (8, 2 * groups, 2)).transpose(-1, -2)  # [..., pages / 16, 8, 2, 2 groups]
    per_token = pairs.flatten(-4, -2).float()  # [..., page, 2 groups]
    power = power_of_two(scales[..., 32 * groups :].flatten(-2).to(torch.int32))
    x = unpack(codes).unflatten(-1, (-1, GROUP))
    return ((x * per_token[..., :groups, None] + per_token[..., groups:, None]) * power[..., None, None]).flatten(-2)


# ------------------------------------------------------------------ inputs


def key_values(g: torch.Generator, shape: tuple) -> torch.Tensor:
    """Keys or values as models have them: normal, some channels several times the others, some shifted."""
    gain = 1.0 + 5.0 * (torch.rand(shape[-1], generator=g, device=DEVICE) < 0.04).float()
    shift = torch.randn(shape[-1], generator=g, device=DEVICE) * 0.3
    return torch.randn(shape, generator=g, device=DEVICE) * gain + shift


def filled_pages(g: torch.Generator, pages: int, case: dict, values: bool) -> tuple:
    """Codes and scales of ``pages`` pages filled with quantised values."""
    _, hkv, d = HEADS[case["model"]]
    page, groups = case["page"], d // GROUP
    four = case["kind"] == "int4"
    codes = torch.empty(pages, hkv, page, d // 2 if four else d, dtype=torch.uint8 if four else torch.int8, device=DEVICE)
    if not four:
        scales = torch.empty(pages, hkv, dtype=torch.float32, device=DEVICE)
    elif values:
        scales = torch.empty(pages, hkv, page // 16, 32 * groups + 16, dtype=torch.float16, device=DEVICE)
    else:
        scales = torch.empty(pages, hkv, page, groups, 2, dtype=torch.float16, device=DEVICE)
    step = max(1, (1 << 26) // (hkv * page * d))
    for i in range(0, pages, step):
        x = key_values(g, (min(step, pages - i), hkv, page, d))
        if not four:
            s = fit_scale(x.abs().amax(dim=(2, 3)), case["kind"])
            codes[i : i + step] = to_codes(x / s[:, :, None, None], case["kind"])
            scales[i : i + step] = s
            continue
        u, scale, offset, exponent = quantise(x, values)
        codes[i : i + step] = pack(u)
        if values:
            both = torch.cat((scale, offset), -1).unflatten(2, (-1, 8, 2)).transpose(-1, -2)  # [..., 8, 2 groups, 2]
            scales[i : i + step, ..., : 32 * groups] = both.flatten(-3)
            scales[i : i + step, ..., 32 * groups :] = exponent.to(torch.float16).unflatten(2, (-1, 16))
        else:
            scales[i : i + step] = torch.stack((scale, offset), -1)
    return codes, scales


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    hq, hkv, d = HEADS[case["model"]]
    page, new, lens = case["page"], new_tokens(case), lengths(case)
    t = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state = {"case": case, "max_query": max(new),
             "lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE),
             "query_start": None if max(new) == 1 else torch.tensor(starts, dtype=torch.int32, device=DEVICE)}
    # the plain form's view of the same: sequence and position of every new token
    state["seq"] = torch.tensor([b for b, n in enumerate(new) for _ in range(n)], device=DEVICE)
    state["pos"] = torch.tensor([ln - n + i for n, ln in zip(new, lens) for i in range(n)], device=DEVICE)
    # pages in the order a busy allocator hands them out; the appends' pool holds the pages they write to
    first = [0 if case["op"] == "attend4" else (ln - n) // page for n, ln in zip(new, lens)]
    last = [(ln - 1) // page for ln in lens]
    pool = sum(b - a + 1 for a, b in zip(first, last))
    order = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((case["seqs"], max(last) + 1), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, (lo, hi) in enumerate(zip(first, last)):
        table[b, lo : hi + 1] = order[at : at + hi - lo + 1]
        at += hi - lo + 1
    state["table"] = table
    state["k_codes"], state["k_scales"] = filled_pages(g, pool, case, False)
    state["v_codes"], state["v_scales"] = filled_pages(g, pool, case, True)
    if case["op"] == "attend4":
        state["q"] = (torch.randn(t, hq, d, generator=g, device=DEVICE) * 1.5).to(torch.bfloat16)
    else:
        # q, k and v side by side, as the grouped projection's output has them
        qkv = key_values(g, (t, hq + 2 * hkv, d)).reshape(t, -1)
        state["qkv"] = qkv if case["dtype"] == "fp32" else qkv.to(torch.bfloat16)
        if case["norms"]:  # the weights in the projections' type, as a checkpoint has them
            for name in ("q_norm", "k_norm"):
                state[name] = (1.0 + 0.3 * torch.randn(d, generator=g, device=DEVICE)).to(state["qkv"].dtype)
        r = rotary_dim(case)
        angle = torch.arange(max(lens), device=DEVICE, dtype=torch.float64)[:, None] * torch.pow(
            torch.tensor(ROTARY_BASE[case["model"]], dtype=torch.float64, device=DEVICE),
            -torch.arange(0, r, 2, device=DEVICE, dtype=torch.float64) / r)[None, :]
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    if own:
        from se12_b200.kv_cache import PagedKvCache

        state["cache"] = PagedKvCache.from_tensors(state["k_codes"], state["v_codes"], state["k_scales"], state["v_scales"],
                                                   kind=case["kind"])
    return state


# ------------------------------------------------------------------ one pass


def run(state: dict):
    return run_attend(state) if state["case"]["op"] == "attend4" else run_append(state)


def run_append(state: dict) -> dict:
    case = state["case"]
    hq, hkv, d = HEADS[case["model"]]
    qkv = state["qkv"].view(-1, hq + 2 * hkv, d)
    q, k, v = qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
    four = case["kind"] == "int4"
    if own:
        cache = state["cache"]
        q_out = cache.append(k, v, state["table"], state["lens"], q=q, cos=state["cos"], sin=state["sin"],
                             query_start=state["query_start"], interleaved=case["rotary"] == "neighbours",
                             q_norm=state.get("q_norm"), k_norm=state.get("k_norm"), norm_eps=EPS)
        keys, values = cache.decode()
        out = {"q": q_out, "keys": keys, "values": values}
        return out if four else {**out, "k_scales": cache.k_scales, "v_scales": cache.v_scales}
    pos, page = state["pos"], case["page"]
    cos, sin = state["cos"][pos][:, None, :], state["sin"][pos][:, None, :]
    pages = state["table"][state["seq"], pos // page].long()  # [T]
    slot = pos % page
    q, k, v = q.float(), k.float(), v.float()
    if case["norms"]:
        q, k = plain_norm(q, state["q_norm"]), plain_norm(k, state["k_norm"])
    q, k = (plain_rotate(x, cos, sin, case["rotary"] == "neighbours") for x in (q, k))
    out = {"q": q.to(torch.bfloat16)}
    if four:
        u, scale, offset, _ = quantise(k, False)
        state["k_codes"][pages, :, slot] = pack(u)
        state["k_scales"][pages, :, slot] = torch.stack((scale, offset), -1)
        u, scale, offset, exponent = quantise(v, True)
        state["v_codes"][pages, :, slot] = pack(u)
        groups = d // GROUP
        pairs = state["v_scales"][..., : 32 * groups].unflatten(-1, (8, 2 * groups, 2))
        pairs[pages, :, slot // 16, slot % 16 // 2, :, slot % 2] = torch.cat((scale, offset), -1)
        state["v_scales"][..., 32 * groups :][pages, :, slot // 16, slot % 16] = exponent.to(torch.float16)
        return {**out, "keys": key_pages(state["k_codes"], state["k_scales"]).to(torch.bfloat16),
                "values": value_pages(state["v_codes"], state["v_scales"]).to(torch.bfloat16)}
    keys = plain_store(state["k_codes"], state["k_scales"], k, pages, slot, case["kind"])
    values = plain_store(state["v_codes"], state["v_scales"], v, pages, slot, case["kind"])
    return {**out, "keys": keys, "values": values, "k_scales": state["k_scales"], "v_scales": state["v_scales"]}


def plain_norm(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    factor = 1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)
    return (x * factor.float()) * weight.float()


def plain_rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, neighbours: bool) -> torch.Tensor:
    n = cos.shape[-1]
    turned, rest = x[..., : 2 * n], x[..., 2 * n :]
    x1, x2 = (turned[..., 0::2], turned[..., 1::2]) if neighbours else (turned[..., :n], turned[..., n:])
    both = (x1 * cos - x2 * sin, x2 * cos + x1 * sin)
    turned = torch.stack(both, dim=-1).flatten(-2) if neighbours else torch.cat(both, dim=-1)
    return torch.cat((turned, rest), dim=-1)


def plain_store(codes: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, pages: torch.Tensor, slot: torch.Tensor,
                kind: str) -> torch.Tensor:
    """Stores x [T, heads, d] at (pages, slot) of an 8-bit cache and returns the pages' values."""
    n_pages, heads, page, d = codes.shape
    index = pages[:, None].expand(-1, heads)
    need = torch.zeros_like(scales).scatter_reduce_(0, index, x.abs().amax(-1), "amax")
    earlier = torch.full((n_pages,), page, device=codes.device).scatter_reduce_(0, pages, slot, "amin")  # tokens already there
    touched = earlier < page
    before = torch.where((touched & (earlier > 0))[:, None], scales, torch.zeros_like(scales))
    after = torch.maximum(before, fit_scale(need, kind))
    after = torch.where(touched[:, None], after, scales)
    ratio = torch.where(touched[:, None], before / after, torch.ones_like(scales))
    again = to_codes(from_codes(codes, kind) * ratio[:, :, None, None], kind)
    old = torch.arange(page, device=codes.device)[None, :] < torch.where(touched, earlier, torch.zeros_like(earlier))[:, None]
    codes.copy_(torch.where(old[:, None, :, None], again, codes))
    codes[pages, :, slot] = to_codes(x / after[pages][:, :, None], kind)
    scales.copy_(after)
    return (from_codes(codes, kind) * scales[:, :, None, None]).to(torch.bfloat16)


def run_attend(state: dict) -> torch.Tensor:
    case = state["case"]
    hq, hkv, d = HEADS[case["model"]]
    if own:
        return state["cache"].attend(state["q"], state["table"], state["lens"], query_start=state["query_start"],
                                     max_query=state["max_query"], softcap=case["softcap"], window=case["window"])
    lens, page = state["lens"].long(), case["page"]
    ids = state["table"].clamp(min=0).long()  # pages a sequence does not have read page 0 (masked later)
    seqs, n, length = case["seqs"], state["max_query"], ids.shape[1] * page

    def by_sequence(x):  # [seqs, columns, heads, page, d] -> [seqs, heads, length, d]
        return x.permute(0, 2, 1, 3, 4).reshape(seqs, hkv, length, d)

    # queries of each sequence side by side: [seqs, n, ...], the missing ones zero
    place = state["pos"] - (lens - count_tokens(state))[state["seq"]]
    q = torch.zeros(seqs, n, hq, d, device=lens.device)
    q[state["seq"], place] = state["q"].float()
    where = torch.zeros(seqs, n, dtype=torch.long, device=lens.device)
    where[state["seq"], place] = state["pos"]
    q = q.view(seqs, n, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, -1, d)
    s = torch.matmul(q, by_sequence(key_pages(state["k_codes"][ids], state["k_scales"][ids])).transpose(-1, -2))
    s = s * (1.0 / math.sqrt(d))  # [seqs, hkv, n * group, length]
    if case["softcap"]:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    s = s.view(seqs, hkv, n, hq // hkv, length)
    j = torch.arange(length, device=lens.device)
    seen = j[None, None, :] <= where[:, :, None]
    if case["window"]:
        seen = seen & (where[:, :, None] - j[None, None, :] < case["window"])
    s = s.masked_fill(~seen[:, None, :, None, :], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(seqs, hkv, -1, length)
    o = torch.matmul(p, by_sequence(value_pages(state["v_codes"][ids], state["v_scales"][ids])))
    o = o.view(seqs, hkv, n, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(seqs, n, hq, d)
    return o[state["seq"], place].to(torch.bfloat16)


def count_tokens(state: dict) -> torch.Tensor:
    start = state["query_start"]
    return torch.ones_like(state["lens"]).long() if start is None else (start[1:] - start[:-1]).long()


# ------------------------------------------------------------------ in 64 bits


def exact(case: dict, seed: int):
    global own
    asked, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = asked
    return exact_attend(case, state) if case["op"] == "attend4" else exact_append(case, state)


def stored_values(case: dict, state: dict, which: str, ids: torch.Tensor) -> torch.Tensor:
    """What the pages ``ids`` hold, in 64 bits [pages, heads, page, d]."""
    codes, scales = state[which + "_codes"][ids].to(torch.int64), state[which + "_scales"][ids].double()
    if case["kind"] == "int8":
        return codes.double() * scales[:, :, None, None]
    if case["kind"] == "e4m3":
        c = codes & 255
        e, m = (c >> 3) & 15, (c & 7).double()
        size = torch.where(e > 0, (1 + m / 8) * torch.exp2(e.double() - 7), m * 2.0**-9)
        return torch.where(c >= 128, -size, size) * scales[:, :, None, None]
    d = HEADS[case["model"]][2]
    groups = d // GROUP
    at = torch.arange(d, device=DEVICE)
    g, r, e = at // GROUP, at % GROUP // 8, at % 8  # a dimension's group, word and place in the word
    u = (codes[..., (r * groups + g) * 4 + e // 2] >> (4 * (e % 2))) & 15
    if which == "k":
        return (u - 8).double() * scales[..., g, 0] + scales[..., g, 1]
    token = torch.arange(case["page"], device=DEVICE)
    cell, pair, side = (token // 16)[:, None], (token % 16 // 2)[:, None], (token % 2)[:, None]
    scale = scales[:, :, cell, (pair * 2 * groups + g) * 2 + side]
    offset = scales[:, :, cell, (pair * 2 * groups + groups + g) * 2 + side]
    return ((u - 8).double() * scale + offset) * torch.exp2(scales[:, :, cell, 32 * groups + (token % 16)[:, None]])


def nearest(x: torch.Tensor, kind: str) -> torch.Tensor:
    """x rounded to the nearest value of the 8-bit grid, ties to even."""
    if kind == "int8":
        return torch.round(x)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0**-6)))
    e = torch.where(torch.exp2(e + 1) <= x.abs(), e + 1, torch.where(torch.exp2(e) > x.abs().clamp(min=2.0**-6), e - 1, e))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def least_scale(amax: float, kind: str) -> float:
    e = MIN_EXPONENT
    if amax > 0:
        e = max(e, math.ceil(math.log2(amax / QMAX[kind])) - 1)
    while amax > QMAX[kind] * 2.0**e:
        e += 1
    return 2.0**e


def four_bit_values(x: torch.Tensor, values: bool) -> torch.Tensor:
    """What x [..., d] (64 bits) becomes in 4 bits: each group of 64 on a line of 16 points."""
    power = torch.ones_like(x[..., :1])
    if values:
        size = x.abs().amax(-1, keepdim=True)
        power = torch.exp2((torch.floor(torch.log2(size.clamp(min=1e-300))) - 3).clamp(min=-30.0))
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], GROUP):
        y = x[..., at : at + GROUP] / power
        low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
        step = ((high - low) / 15).half().double()
        middle = (low + 8 * step).half().double()
        point = torch.round((y - middle) / step.clamp(min=1e-300)).clamp(-8, 7)
        out[..., at : at + GROUP] = torch.where(step > 0, point * step + middle, middle.expand_as(y)) * power
    return out


def exact_append(case: dict, state: dict) -> dict:
    hq, hkv, d = HEADS[case["model"]]
    kind, page, four = case["kind"], case["page"], case["kind"] == "int4"
    qkv = state["qkv"].double().view(-1, hq + 2 * hkv, d)
    c, s = state["cos"].double(), state["sin"].double()
    r = rotary_dim(case)
    at = torch.arange(r // 2, device=DEVICE)
    first, second = (2 * at, 2 * at + 1) if case["rotary"] == "neighbours" else (at, at + r // 2)

    def turned(x, name, p):
        if case["norms"]:
            x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / d + EPS) * state[name].double()
        a, b, cp, sp = x[..., first], x[..., second], c[p][:, None], s[p][:, None]
        y = x.clone()
        y[..., first], y[..., second] = a * cp - b * sp, b * cp + a * sp
        return y

    everything = torch.arange(state["k_codes"].shape[0], device=DEVICE)
    out_q = []
    pools = {w: stored_values(case, state, w, everything) for w in "kv"}
    scales = {w: state[w + "_scales"].double() for w in "kv"}
    t = 0
    for b, (n, ln) in enumerate(zip(new_tokens(case), lengths(case))):
        p = torch.arange(ln - n, ln, device=DEVICE)
        rows = qkv[t : t + n]
        out_q.append(turned(rows[:, :hq], "q_norm", p))
        parts = {"k": turned(rows[:, hq : hq + hkv], "k_norm", p), "v": rows[:, hq + hkv :]}
        if four:
            parts = {w: four_bit_values(x, w == "v") for w, x in parts.items()}
        for begin in sorted({max(i * page, ln - n) for i in range((ln - n) // page, (ln - 1) // page + 1)}):
            column, there = begin // page, begin % page
            end = min(ln, (column + 1) * page)
            pid = int(state["table"][b, column])
            for w, values in pools.items():
                x = parts[w][begin - (ln - n) : end - (ln - n)].transpose(0, 1)
                if not four:
                    need = torch.tensor([least_scale(a, kind) for a in x.abs().amax(dim=(1, 2)).tolist()], dtype=torch.float64,
                                        device=DEVICE)
                    now = (torch.maximum(scales[w][pid], need) if there else need)[:, None, None]
                    if there:
                        values[pid, :, :there] = nearest(values[pid, :, :there] / now, kind) * now
                    x = nearest(x / now, kind) * now
                    scales[w][pid] = now[:, 0, 0]
                values[pid, :, there : there + end - begin] = x
                if not four:  # slots past the new tokens keep their codes, which the new scale gives another value
                    old = stored_values(case, state, w, everything[pid : pid + 1])[0, :, there + end - begin :]
                    values[pid, :, there + end - begin :] = old / state[w + "_scales"][pid].double()[:, None, None] * now
        t += n
    out = {"q": torch.cat(out_q), "keys": pools["k"], "values": pools["v"]}
    return out if four else {**out, "k_scales": scales["k"], "v_scales": scales["v"]}


def exact_attend(case: dict, state: dict) -> torch.Tensor:
    hq, hkv, d = HEADS[case["model"]]
    group, page = hq // hkv, case["page"]
    out, t = [], 0
    for b, (n, ln) in enumerate(zip(new_tokens(case), lengths(case))):
        ids = state["table"][b, : (ln + page - 1) // page].long()
        rows = torch.empty(n, hq, d, dtype=torch.float64, device=DEVICE)
        j, i = torch.arange(ln, device=DEVICE), torch.arange(ln - n, ln, device=DEVICE)
        hidden = j[None, :] > i[:, None]
        if case["window"]:
            hidden |= i[:, None] - j[None, :] >= case["window"]
        keys, values = (stored_values(case, state, w, ids).transpose(0, 1).reshape(hkv, -1, d)[:, :ln] for w in "kv")
        for h in range(hkv):
            for r in range(h * group, (h + 1) * group):
                s = state["q"][t : t + n, r].double() @ keys[h].T / math.sqrt(d)
                if case["softcap"]:
                    s = case["softcap"] * torch.tanh(s / case["softcap"])
                rows[:, r] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ values[h]
        out.append(rows)
        t += n
    return torch.cat(out)
