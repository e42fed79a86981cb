"""The operators of a decode step around the SE12 GEMVs, as cases to be measured.

* ``append``: new keys and values, rotated to their positions, into a paged
  8-bit cache with one power-of-two scale per page and KV head; the queries
  rotated in the same pass.
* ``attend``: attention of the new tokens over that cache.
* ``logprobs``: log probabilities of given tokens, the entropy and the top
  alternatives of each row of LM-head logits.

With ``own`` false, ``run`` computes them in elementary torch operations in
fp32, rounded once at the end; with ``own`` true it makes the calls a user of
``se12_b200`` makes. Head counts and dimensions are those of the decoder
configurations in ``se12_b200/shapes.py``.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
QMAX = {"int8": 127.0, "e4m3": 448.0}
MIN_EXPONENT = -100
# (query heads, KV heads, head dimension) of the decoder configurations
HEADS = {"gemma2-2b": (8, 4, 256), "gemma2-9b": (16, 8, 256), "gemma2-27b": (32, 16, 128), "llama3.1-70b": (64, 8, 128)}
ROTARY_BASE = {"gemma2-2b": 1e4, "gemma2-9b": 1e4, "gemma2-27b": 1e4, "llama3.1-70b": 5e5}


# ------------------------------------------------------------------ cases


def listed() -> list:
    return [
        # the smallest call: one sequence's next token, straight from the fp32 output of the grouped q/k/v GEMV
        dict(name="append-1", op="append", model="gemma2-2b", page=16, kind="int8", dtype="fp32", seqs=1, shortest=40, longest=40,
             new_low=1, new_high=1, window=0, softcap=0.0),
        # a serving batch's next tokens
        dict(name="append-64", op="append", model="llama3.1-70b", page=64, kind="e4m3", dtype="fp32", seqs=64, shortest=5,
             longest=16000, new_low=1, new_high=1, window=0, softcap=0.0),
        # a batch of prompt chunks behind cached prefixes, ragged, BF16 projections (the exact mode's F.linear)
        dict(name="append-prompts", op="append", model="gemma2-9b", page=32, kind="int8", dtype="bf16", seqs=13, shortest=0,
             longest=3001, new_low=301, new_high=2043, window=0, softcap=0.0),
        # the smallest attention: a new conversation's second page
        dict(name="attend-1-short", op="attend", model="gemma2-2b", page=16, kind="int8", seqs=1, shortest=17, longest=17, new_low=1,
             new_high=1, window=0, softcap=50.0),
        # a local (sliding-window, capped) layer of a serving batch
        dict(name="attend-16-window", op="attend", model="gemma2-9b", page=32, kind="int8", seqs=16, shortest=301, longest=8191,
             new_low=1, new_high=1, window=4096, softcap=50.0),
        # a large serving batch, ragged lengths
        dict(name="attend-64", op="attend", model="llama3.1-70b", page=64, kind="e4m3", seqs=64, shortest=1000, longest=16384,
             new_low=1, new_high=1, window=0, softcap=0.0),
        # one very long conversation
        dict(name="attend-1-long", op="attend", model="gemma2-27b", page=128, kind="int8", seqs=1, shortest=131071, longest=131071,
             new_low=1, new_high=1, window=0, softcap=50.0),
        # drafted tokens to verify: a few queries per sequence
        dict(name="attend-verify", op="attend", model="llama3.1-70b", page=16, kind="e4m3", seqs=24, shortest=77, longest=4093,
             new_low=2, new_high=6, window=0, softcap=0.0),
        # prompt chunks behind a cached prefix
        dict(name="attend-chunk", op="attend", model="gemma2-9b", page=64, kind="int8", seqs=2, shortest=5000, longest=8191,
             new_low=509, new_high=509, window=0, softcap=50.0),
        # the token a decode step just chose
        dict(name="logprobs-1", op="logprobs", vocab=256000, rows=1, dtype="fp32", top=5, softcap=30.0, banned=0.0),
        # a serving batch with constrained rows (banned tokens at -inf)
        dict(name="logprobs-16", op="logprobs", vocab=256000, rows=16, dtype="fp32", top=20, softcap=30.0, banned=0.3),
        # scoring a prompt: BF16 logits of the exact mode, many equal values
        dict(name="logprobs-prompt", op="logprobs", vocab=128256, rows=1023, dtype="bf16", top=20, softcap=0.0, banned=0.0),
    ]


def log_uniform(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(("append", "attend", "attend", "logprobs"))
    if op == "logprobs":
        vocab = rng.choice((256000, 128256, log_uniform(rng, 1000, 260000)))
        rows = log_uniform(rng, 1, min(1023, 1023 * 128256 // vocab))
        return dict(op=op, vocab=vocab, rows=rows, dtype=rng.choice(("fp32", "bf16")) if rows * vocab < 60_000_000 else "bf16",
                    top=rng.randint(0, 20), softcap=rng.choice((0.0, 30.0)), banned=rng.choice((0.0, 0.3)))
    model = rng.choice(sorted(HEADS))
    page, kind = rng.choice((16, 32, 64, 128)), rng.choice(("int8", "e4m3"))
    seqs = log_uniform(rng, 1, 64)
    if op == "append":
        if rng.random() < 0.5:
            new_low = new_high = 1
        else:
            new_high = log_uniform(rng, 2, max(2, 16000 // seqs))
            new_low = rng.randint(1, new_high)
        longest = log_uniform(rng, 1, 16000)
        return dict(op=op, model=model, page=page, kind=kind, dtype=rng.choice(("fp32", "bf16")), seqs=seqs,
                    shortest=rng.randint(0, longest), longest=longest, new_low=new_low, new_high=new_high, window=0, softcap=0.0)
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
    case = dict(op=op, model=model, page=page, kind=kind, seqs=seqs, shortest=rng.randint(new_high, longest), longest=longest,
                new_low=new_low, new_high=new_high, window=rng.choice((0, 0, 512, 4096)), softcap=rng.choice((0.0, 50.0)))
    while work(case)["bytes"] > 9e8 or work(case)["flops"] > 1e11:
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
    """Tokens in the cache once the new ones are in (append: longest/shortest are the prefix before them)."""
    base = spread(case["shortest"], case["longest"], case["seqs"], 0.618034)
    return [b + n for b, n in zip(base, new_tokens(case))] if case["op"] == "append" else base


def element_bytes(case: dict) -> int:
    return 4 if case["dtype"] == "fp32" else 2


def work(case: dict) -> dict:
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": n * v * element_bytes(case) + n * (8 + 4 + 4 + 12 * k), "flops": 4 * n * v}
    hq, hkv, d = HEADS[case["model"]]
    new, lens = new_tokens(case), lengths(case)
    t = sum(new)
    if case["op"] == "append":
        pages = sum((ln - 1) // case["page"] - (ln - n) // case["page"] + 1 for n, ln in zip(new, lens))
        block = case["page"] * hkv * d
        return {"bytes": t * (hq + 2 * hkv) * d * element_bytes(case)  # queries, keys, values in
                + t * d * 4 + t * hq * d * 2  # cosines and sines in, rotated queries out
                + 2 * t * hkv * d + 2 * pages * hkv * 4  # codes and scales out
                + 2 * pages * block * (1 + 2),  # the pages read back: codes in, BF16 values out
                "flops": 3 * t * (hq + 2 * hkv) * d}
    pairs = visible = 0
    for n, ln in zip(new, lens):
        first = max(0, ln - n + 1 - case["window"]) if case["window"] else 0
        visible += ln - first
        for p in range(ln - n, ln):
            pairs += min(p + 1, case["window"]) if case["window"] else p + 1
    return {"bytes": 2 * visible * hkv * d + 4 * t * hq * d + 8 * hkv * (visible // case["page"]), "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ inputs


def fit_scale(amax: torch.Tensor, kind: str) -> torch.Tensor:
    """The power of two 2^e, e >= MIN_EXPONENT least, with amax <= QMAX 2^e."""
    half, e = torch.frexp(amax)  # amax = half 2^e, 0.5 <= half < 1
    q_half, q_e = math.frexp(QMAX[kind])
    e = torch.where(half <= q_half, e - q_e, e - q_e + 1)
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXPONENT)).clamp(min=MIN_EXPONENT)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def to_codes(x: torch.Tensor, kind: str) -> torch.Tensor:
    """Scaled values as codes: whole numbers of int8, or e4m3 bit patterns (both as int8 tensors)."""
    return torch.round(x).to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn).view(torch.int8)


def from_codes(c: torch.Tensor, kind: str) -> torch.Tensor:
    return c.to(torch.float32) if kind == "int8" else c.view(torch.float8_e4m3fn).to(torch.float32)


def key_values(g: torch.Generator, shape: tuple) -> torch.Tensor:
    """Keys or values as models have them: normal, some channels several times the others."""
    gain = 1.0 + 5.0 * (torch.rand(shape[-1], generator=g, device=DEVICE) < 0.04).float()
    return torch.randn(shape, generator=g, device=DEVICE) * gain


def filled_pages(g: torch.Generator, pages: int, case: dict) -> tuple:
    """Codes and scales of ``pages`` pages filled with quantised values."""
    _, hkv, d = HEADS[case["model"]]
    codes = torch.empty(pages, hkv, case["page"], d, dtype=torch.int8, device=DEVICE)
    scales = torch.empty(pages, hkv, dtype=torch.float32, device=DEVICE)
    step = max(1, (1 << 26) // (hkv * case["page"] * d))
    for i in range(0, pages, step):
        x = key_values(g, tuple(codes[i : i + step].shape))
        s = fit_scale(x.abs().amax(dim=(2, 3)), case["kind"])
        codes[i : i + step] = to_codes(x / s[:, :, None, None], case["kind"])
        scales[i : i + step] = s
    return codes, scales


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["op"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        x = torch.randn(n, v, generator=g, device=DEVICE) * 2.5
        likely = torch.randint(0, v, (n, 8), generator=g, device=DEVICE)  # a few likely tokens stand out
        x.scatter_add_(1, likely, 6.0 + 6.0 * torch.rand(n, 8, generator=g, device=DEVICE))
        tokens = torch.where(torch.rand(n, generator=g, device=DEVICE) < 0.7, likely[:, 0],
                             torch.randint(0, v, (n,), generator=g, device=DEVICE))
        if case["banned"]:
            ban = torch.rand(n, v, generator=g, device=DEVICE) < case["banned"]
            ban.scatter_(1, tokens[:, None], False)
            x.masked_fill_(ban, float("-inf"))
        return {"case": case, "logits": x if case["dtype"] == "fp32" else x.to(torch.bfloat16), "tokens": tokens}

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
    # pages in the order a busy allocator hands them out; append's pool holds the pages it writes to
    first = [(ln - n) // page if case["op"] == "append" else 0 for n, ln in zip(new, lens)]
    last = [(ln - 1) // page for ln in lens]
    pool = sum(b - a + 1 for a, b in zip(first, last))
    order = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((case["seqs"], max(last) + 1), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, (lo, hi) in enumerate(zip(first, last)):
        table[b, lo : hi + 1] = order[at : at + hi - lo + 1]
        at += hi - lo + 1
    state["table"] = table
    state["k_codes"], state["k_scales"] = filled_pages(g, pool, case)
    state["v_codes"], state["v_scales"] = filled_pages(g, pool, case)
    if case["op"] == "append":
        # q, k and v side by side, as the grouped projection's output has them
        qkv = key_values(g, (t, hq + 2 * hkv, d)).reshape(t, -1)
        state["qkv"] = qkv if case["dtype"] == "fp32" else qkv.to(torch.bfloat16)
        angle = torch.arange(max(lens), device=DEVICE, dtype=torch.float64)[:, None] * torch.pow(
            torch.tensor(ROTARY_BASE[case["model"]], dtype=torch.float64, device=DEVICE),
            -torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d)[None, :]
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    else:
        state["q"] = (torch.randn(t, hq, d, generator=g, device=DEVICE) * 1.5).to(torch.bfloat16)
    if own:
        from se12_b200.kv_cache import PagedKvCache

        state["cache"] = PagedKvCache.from_tensors(state["k_codes"], state["v_codes"], state["k_scales"], state["v_scales"],
                                                   kind=case["kind"])
    return state


# ------------------------------------------------------------------ one pass


def run(state: dict):
    return {"append": run_append, "attend": run_attend, "logprobs": run_logprobs}[state["case"]["op"]](state)


def run_append(state: dict) -> dict:
    case = state["case"]
    hq, hkv, d = HEADS[case["model"]]
    qkv = state["qkv"].view(-1, hq + 2 * hkv, d)
    q, k, v = qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
    if own:
        cache = state["cache"]
        q_out = cache.append(k, v, state["table"], state["lens"], q=q, cos=state["cos"], sin=state["sin"],
                             query_start=state["query_start"])
        keys, values = cache.decode()
        return {"q": q_out, "keys": keys, "values": values, "k_scales": cache.k_scales, "v_scales": cache.v_scales}
    pos, page = state["pos"], case["page"]
    cos, sin = state["cos"][pos][:, None, :], state["sin"][pos][:, None, :]
    pages = state["table"][state["seq"], pos // page].long()  # [T]
    slot = pos % page
    keys = plain_store(state["k_codes"], state["k_scales"], plain_rotate(k.float(), cos, sin), pages, slot, case["kind"])
    values = plain_store(state["v_codes"], state["v_scales"], v.float(), pages, slot, case["kind"])
    return {"q": plain_rotate(q.float(), cos, sin).to(torch.bfloat16), "keys": keys, "values": values,
            "k_scales": state["k_scales"], "v_scales": state["v_scales"]}


def plain_rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    x1, x2 = x[..., : cos.shape[-1]], x[..., cos.shape[-1] :]
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1)


def plain_store(codes: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, pages: torch.Tensor, slot: torch.Tensor,
                kind: str) -> torch.Tensor:
    """Stores x [T, heads, d] at (pages, slot) and returns the pages' values."""
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
    lens, table, page = state["lens"].long(), state["table"], case["page"]
    seqs, n, length = case["seqs"], state["max_query"], table.shape[1] * page
    keys = plain_pages(state["k_codes"], state["k_scales"], table, case["kind"])
    values = plain_pages(state["v_codes"], state["v_scales"], table, case["kind"])
    # queries of each sequence side by side: [seqs, n, ...], the missing ones zero
    place = state["pos"] - (lens - count_tokens(state))[state["seq"]]
    q = torch.zeros(seqs, n, hq, d, device=lens.device)
    q[state["seq"], place] = state["q"].float()
    where = torch.zeros(seqs, n, dtype=torch.long, device=lens.device)
    where[state["seq"], place] = state["pos"]
    q = q.view(seqs, n, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, -1, d)
    s = torch.matmul(q, keys.transpose(-1, -2)) * (1.0 / math.sqrt(d))  # [seqs, hkv, n * group, length]
    del keys
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
    o = torch.matmul(p, values).view(seqs, hkv, n, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(seqs, n, hq, d)
    return o[state["seq"], place].to(torch.bfloat16)


def count_tokens(state: dict) -> torch.Tensor:
    start = state["query_start"]
    return torch.ones_like(state["lens"]).long() if start is None else (start[1:] - start[:-1]).long()


def plain_pages(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, kind: str) -> torch.Tensor:
    """The sequences' values [seqs, heads, pages * page, d]; pages a sequence does not have read page 0 (masked later)."""
    ids = table.clamp(min=0).long()
    x = from_codes(codes[ids], kind) * scales[ids][:, :, :, None, None]
    return x.permute(0, 2, 1, 3, 4).reshape(ids.shape[0], codes.shape[1], -1, codes.shape[3])


def run_logprobs(state: dict) -> dict:
    case = state["case"]
    if own:
        from se12_b200.logprobs import token_logprobs

        r = token_logprobs(state["logits"], state["tokens"], top=case["top"], softcap=case["softcap"])
        return {"logprob": r.logprob, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
    x = state["logits"].float()
    z = torch.tanh(x / case["softcap"]) * case["softcap"] if case["softcap"] else x
    z = z.masked_fill(x == float("-inf"), float("-inf"))  # a banned token stays banned behind the cap
    above = z - z.amax(-1, keepdim=True)
    e = torch.exp(above)
    total = e.sum(-1, keepdim=True)
    mean = torch.where(e > 0, e * above, torch.zeros_like(e)).sum(-1) / total[:, 0]
    logp = above - torch.log(total)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, : case["top"]]
    return {"logprob": logp.gather(1, state["tokens"][:, None])[:, 0], "entropy": torch.log(total[:, 0]) - mean,
            "top_ids": ids, "top_logprobs": logp.gather(1, ids)}


# ------------------------------------------------------------------ in 64 bits


def exact(case: dict, seed: int):
    global own
    asked, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = asked
    return {"append": exact_append, "attend": exact_attend, "logprobs": exact_logprobs}[case["op"]](case, state)


def grid_value(c: torch.Tensor, kind: str) -> torch.Tensor:
    """What a code stands for, from its bits."""
    c = c.to(torch.int64)
    if kind == "int8":
        return c.double()
    c = c & 255
    e, m = (c >> 3) & 15, (c & 7).double()
    size = torch.where(e > 0, (1 + m / 8) * torch.exp2(e.double() - 7), m * 2.0**-9)
    return torch.where(c >= 128, -size, size)


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


def exact_append(case: dict, state: dict) -> dict:
    hq, hkv, d = HEADS[case["model"]]
    kind, page = case["kind"], case["page"]
    qkv = state["qkv"].double().view(-1, hq + 2 * hkv, d)
    c, s = state["cos"].double(), state["sin"].double()
    half = d // 2

    def turn(x, p):
        a, b = x[..., :half], x[..., half:]
        cp, sp = c[p][:, None], s[p][:, None]
        return torch.cat((a * cp - b * sp, b * cp + a * sp), -1)

    out_q = []
    pools = {"k": (grid_value(state["k_codes"], kind), state["k_scales"].double()),
             "v": (grid_value(state["v_codes"], kind), state["v_scales"].double())}
    t = 0
    for b, (n, ln) in enumerate(zip(new_tokens(case), lengths(case))):
        p = torch.arange(ln - n, ln, device=DEVICE)
        rows = qkv[t : t + n]
        out_q.append(turn(rows[:, :hq], p))
        parts = {"k": turn(rows[:, hq : hq + hkv], p), "v": rows[:, hq + hkv :]}
        for first in sorted({max(i * page, ln - n) for i in range((ln - n) // page, (ln - 1) // page + 1)}):
            at, there = first // page, first % page
            end = min(ln, (at + 1) * page)
            pid = int(state["table"][b, at])
            for which, (codes, scales) in pools.items():
                x = parts[which][first - (ln - n) : end - (ln - n)]
                need = torch.tensor([least_scale(a, kind) for a in x.abs().amax(dim=(0, 2)).tolist()], dtype=torch.float64,
                                    device=DEVICE)
                now = torch.maximum(scales[pid], need) if there else need
                if there:
                    codes[pid, :, :there] = nearest(codes[pid, :, :there] * (scales[pid] / now)[:, None, None], kind)
                codes[pid, :, there : there + end - first] = nearest(x / now[None, :, None], kind).transpose(0, 1)
                scales[pid] = now
        t += n
    return {"q": torch.cat(out_q), "keys": pools["k"][0] * pools["k"][1][:, :, None, None],
            "values": pools["v"][0] * pools["v"][1][:, :, None, None], "k_scales": pools["k"][1], "v_scales": pools["v"][1]}


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
        for h in range(hkv):
            k, v = ((grid_value(c[ids, h], case["kind"]) * sc[ids, h].double()[:, None, None]).reshape(-1, d)[:ln]
                    for c, sc in ((state["k_codes"], state["k_scales"]), (state["v_codes"], state["v_scales"])))
            for r in range(h * group, (h + 1) * group):
                s = state["q"][t : t + n, r].double() @ k.T / math.sqrt(d)
                if case["softcap"]:
                    s = case["softcap"] * torch.tanh(s / case["softcap"])
                rows[:, r] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
        out.append(rows)
        t += n
    return torch.cat(out)


def exact_logprobs(case: dict, state: dict) -> dict:
    lp, ent, top = [], [], []
    for r in range(case["rows"]):
        x = state["logits"][r].double()
        z = x if not case["softcap"] else torch.where(torch.isinf(x), x, case["softcap"] * torch.tanh(x / case["softcap"]))
        logp = z - torch.logsumexp(z, 0)
        p = torch.exp(logp)
        lp.append(logp[state["tokens"][r]])
        ent.append(-(p[p > 0] * logp[p > 0]).sum())
        top.append(torch.sort(logp, descending=True).values[: case["top"]])
    return {"logprob": torch.stack(lp), "entropy": torch.stack(ent), "top_ids": None, "top_logprobs": torch.stack(top)}
