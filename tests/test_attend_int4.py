"""Attention over the paged 4-bit cache, against 64-bit sums over the values
that the pages stand for.

Tolerance, elementwise. The output is rounded to BF16 (half a unit in its last
place). Few rows: a value is scale (u - 8) + offset; its weight is rounded to
FP16 (2^-11), and for the first part once more times the scale (2^-11), so
2^-10 of sum_j p_j |scale (u - 8)| and 2^-11 of sum_j p_j |offset|; the fp32
errors of logits, exponential and sum are below 2^-12 of sum_j p_j |v_j|.
Weights below FP16's normal range: off by 2^-25 of the largest, times codes and
scales of up to 40 where the largest values are 8 or more: 2^-22 of the length
times the largest |v|. Many rows: keys and values are rounded to FP16 (2^-11)
themselves; a key's rounding moves a logit by 2^-11 of scale sum_d |q k|, which
changes weights and their sum by that much each."""

from __future__ import annotations

import math

import pytest
import torch
from test_kv_cache import random_tables, rope, starts_of
from test_kv_int4 import GROUP, Plain4, make_pair


def power_of_two(e):
    return torch.exp2(e.double())


class Filled:
    """A cache of random lines, and on the GPU in 64 bits what it holds."""

    def __init__(self, g, pool, page, heads, dim, spread=1.0, shift=0.3):
        from se12_b200.kv_cache import PagedKvCache

        plain = Plain4(pool, page, heads, dim)
        for w in "kv":
            plain.u[w] = torch.randint(0, 16, plain.u[w].shape, generator=g, dtype=torch.uint8)
            shape = plain.scale[w].shape
            size = 2.0 ** ((torch.rand(shape, generator=g) * 2 - 1) * min(spread, 6.0))
            plain.scale[w] = (size * (0.1 + 0.1 * torch.rand(shape, generator=g))).half()
            plain.offset[w] = (torch.randn(shape, generator=g) * shift * size).half()
        plain.e = torch.randint(-int(spread), int(spread) + 1, plain.e.shape, generator=g).float()
        self.plain, self.page, self.heads, self.dim = plain, page, heads, dim
        self.cache = PagedKvCache.from_tensors(*(t.cuda() for t in plain.tensors()), "int4")
        self.keys = plain.values("k").cuda()
        steps = (plain.u["v"].double().unflatten(-1, (-1, GROUP)) - 8) * plain.scale["v"].double()[..., None]
        power = power_of_two(plain.e)[..., None]
        self.steps = steps.flatten(-2).cuda() * power.cuda()
        self.offsets = plain.offset["v"].double().repeat_interleave(GROUP, -1).cuda() * power.cuda()

    def check(self, q, table, lens, counts, got, softcap=0.0, window=0, scale=None, many=False):
        dim, group = self.dim, q.shape[1] // self.heads
        scale = dim**-0.5 if scale is None else scale
        starts, worst = starts_of(counts), 0.0
        q, table, got = q.cuda(), table.cuda(), got.double()
        for b, ln in enumerate(lens):
            if counts[b] == 0:
                continue
            i, j = torch.arange(ln - counts[b], ln, device="cuda"), torch.arange(ln, device="cuda")
            seen = j[None, :] <= i[:, None]
            if window:
                seen &= i[:, None] - j[None, :] < window
            ids = table[b, : (ln + self.page - 1) // self.page].long()
            for h in range(self.heads):
                k, s, o = (t[ids, h].reshape(-1, dim)[:ln] for t in (self.keys, self.steps, self.offsets))
                for r in range(h * group, (h + 1) * group):
                    x = q[starts[b] : starts[b + 1], r].double()
                    logits = x @ k.T * scale
                    if softcap:
                        logits = softcap * torch.tanh(logits / softcap)
                    p = torch.softmax(logits.masked_fill(~seen, -math.inf), -1).nan_to_num(0)  # (rows that see nothing: zeros)
                    want, size = p @ (s + o), p @ (s + o).abs()
                    tol = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=1e-300))) - 8)
                    tol = tol + 2.0**-10 * (p @ s.abs()) + 2.0**-11 * (p @ o.abs()) + 2.0**-12 * size
                    if ln:
                        tol = tol + 2.0**-22 * ln * (s + o).abs().max()
                        if many:
                            moved = 2.0**-11 * abs(scale) * (x.abs() @ k.abs().T).masked_fill(~seen, 0).amax(-1, keepdim=True)
                            tol = tol + (2.0**-11 + 2 * moved) * size
                    err = (got[starts[b] : starts[b + 1], r] - want).abs()
                    assert bool((err <= tol).all()), (b, r, float((err / tol.clamp(min=1e-300)).max()))
                    worst = max(worst, float((err / tol.clamp(min=1e-300)).max()))
        return worst


def attend_case(seed, page, heads, q_heads, dim, lens, counts, softcap=0.0, window=0, spread=1.0, q_scale=1.0, max_query=None,
                scale=None, shift=0.3):
    g = torch.Generator().manual_seed(seed)
    table, pool = random_tables(g, lens, page)
    f = Filled(g, pool, page, heads, dim, spread, shift)
    starts = starts_of(counts)
    q = (torch.randn(starts[-1], q_heads, dim, generator=g) * q_scale).to(torch.bfloat16)
    start = None if all(n == 1 for n in counts) and max_query is None else torch.tensor(starts, dtype=torch.int32).cuda()
    args = (table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    call = dict(query_start=start, softcap=softcap, window=window, scale=scale, max_query=max_query)
    got = f.cache.attend(q.cuda(), *args, **call)
    most = 1 if start is None else max(counts) if max_query is None else max_query
    f.check(q, table, lens, counts, got, softcap, window, scale, many=most * q_heads // heads > 16)
    assert torch.equal(got.view(torch.int16), f.cache.attend(q.cuda(), *args, **call).view(torch.int16))
    return f, q, args, got


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_lengths_around_pages_and_chunks(page, dim):
    attend_case(page + dim, page, 2, 4, dim, [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 255, 256, 257, 700], [1] * 18)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,q_heads", [(1, 1), (1, 8), (2, 6), (4, 20), (1, 16), (2, 34), (3, 3), (1, 64)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_head_layouts(heads, q_heads, dim):
    attend_case(heads * 100 + q_heads, 16, heads, q_heads, dim, [77, 3], [1, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 7, 16, 100])
@pytest.mark.parametrize("softcap", [0.0, 5.0, 300.0])
def test_windows_and_several_queries(dim, window, softcap):
    """Drafted tokens and prompt chunks, idle sequences, and more rows than the
    sequence is long (the first ones see nothing)."""
    counts = [1, 4, 0, 19, 33, 3, 0]
    f, q, args, got = attend_case(window + dim, 16, 2, 6, dim, [40, 4, 9, 200, 33, 2, 0], counts, softcap=softcap, window=window,
                                  q_scale=3.0)
    assert bool((got[starts_of(counts)[5]] == 0).all())  # position -1


@pytest.mark.gpu
@pytest.mark.parametrize("dim,q_heads,heads", [(64, 8, 2), (128, 8, 1), (256, 4, 2), (128, 12, 1), (256, 12, 1)])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 17, 70])
def test_query_counts(dim, q_heads, heads, n):
    attend_case(n, 64, heads, q_heads, dim, [300, n], [n, n], max_query=n)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [5000, 20011])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_one_long_sequence_is_split(length, dim):
    attend_case(length, 128, 1, 4, dim, [length], [1], softcap=30.0)
    attend_case(length, 16, 2, 2, dim, [length, 1, 3, length // 2], [1, 1, 1, 1], window=length // 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 5])
def test_values_of_very_different_sizes(dim, n):
    """E from -30 to 30, and groups of a token 2^12 apart: a weight's precision
    does not depend on what other tokens hold."""
    attend_case(9, 16, 2, 4, dim, [200, 45], [n, n], spread=30.0, q_scale=2.0**-7)
    attend_case(10, 16, 1, 8, dim, [200, 45], [n, n], spread=6.0, scale=-(2.0**-9))


@pytest.mark.gpu
@pytest.mark.parametrize("q_size", [0.0, 2.0**-60, 2.0**60])
def test_queries_of_any_size(q_size):
    """Rows of zeros weigh all tokens alike, so that large offsets cancel or not
    exactly as their weights do; tiny and huge rows take their size."""
    scale = None if not q_size else 0.1 / q_size
    attend_case(3, 32, 2, 4, 128, [3000, 17], [1, 1], q_scale=q_size, scale=scale, shift=0.0)
    attend_case(3, 32, 2, 4, 128, [3000, 17], [1, 1], q_scale=q_size, scale=scale, shift=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_equal_weights_of_equal_scales_cancel_as_codes_do(dim):
    """A zero query over 16384 tokens whose scales and offsets are one number each:
    the mean of the codes, to which the rounding of weight and scale adds no more
    than its relative size (the zero points take the same rounded product)."""
    from se12_b200.kv_cache import PagedKvCache

    g = torch.Generator().manual_seed(dim)
    n, page = 16384, 256
    plain = Plain4(n // page, page, 1, dim)
    plain.u["v"] = torch.randint(0, 16, plain.u["v"].shape, generator=g, dtype=torch.uint8)
    plain.scale["v"].fill_(0.337)
    cache = PagedKvCache.from_tensors(*(t.cuda() for t in plain.tensors()), "int4")
    table = torch.arange(n // page, dtype=torch.int32)[None].cuda()
    out = cache.attend(torch.zeros(1, 2, dim, dtype=torch.bfloat16, device="cuda"), table, torch.tensor([n], dtype=torch.int32).cuda())
    want = plain.values("v").reshape(n, dim).mean(0)
    # weight, product and BF16's rounding, and fp32 sums of 16384 products below 16 codes
    tol = (2.0**-10 + 2.0**-8) * want.abs() + 2.0**-24 * 128 * 16 * 0.337
    assert bool(((out[0].double().cpu() - want).abs() <= tol).all())


@pytest.mark.gpu
def test_weights_of_zero_values_count():
    cache, _ = make_pair(2, 16, 1, 128)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    k = torch.zeros(32, 1, 128, device="cuda")
    v = torch.zeros(32, 1, 128, device="cuda")
    v[16:] = 8.0
    lens = torch.tensor([32], dtype=torch.int32, device="cuda")
    cache.append(k, v, table, lens, query_start=torch.tensor([0, 32], dtype=torch.int32, device="cuda"))
    out = cache.attend(torch.ones(1, 2, 128, dtype=torch.bfloat16, device="cuda"), table, lens)
    assert bool((out == 4.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group,n", [(1, 1), (8, 1), (8, 2), (8, 3), (8, 4), (11, 3), (8, 6)])
@pytest.mark.parametrize("long", [0, 3000])
def test_many_short_pairs(dim, group, n, long):
    """Sequences of no token to a few tiles, alone and around a long one: runs
    that begin and end anywhere in a pair, or hold no token of it."""
    g = torch.Generator().manual_seed(dim + group * n)
    lens = [(i * 37) % 90 for i in range(150)] + [0, n, 700]
    if long:
        lens[70] = long
    counts = [min(1 + i % n, ln) if ln else 1 for i, ln in enumerate(lens)]
    table, pool = random_tables(g, lens, 16)
    f = Filled(g, pool, 16, 2, dim, 2.0)
    q = (torch.randn(sum(counts), 2 * group, dim, generator=g) * 2).to(torch.bfloat16)
    start = torch.tensor(starts_of(counts), dtype=torch.int32).cuda()
    for _ in range(2):
        got = f.cache.attend(q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), query_start=start, max_query=n)
        f.check(q, table, lens, counts, got, many=group * n > 16)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,q_heads,dim,page", [(4, 32, 128, 16), (8, 16, 256, 64), (2, 24, 64, 32)])
@pytest.mark.parametrize("softcap,window", [(0.0, 0), (30.0, 700)])
def test_many_tiles_per_cta(heads, q_heads, dim, page, softcap, window):
    """Runs of many tiles of many pairs: drafted tokens and prompt chunks, also
    sequences whose chunk is all they have."""
    g = torch.Generator().manual_seed(heads)
    counts = [2 + i % 5 for i in range(20)] + [300, 0, 70, 513]
    lens = [n + (i * 397) % 2500 for i, n in enumerate(counts)]
    lens[-2] = 70
    table, pool = random_tables(g, lens, page)
    f = Filled(g, pool, page, heads, dim, 2.0)
    q = (torch.randn(sum(counts), q_heads, dim, generator=g) * 2).to(torch.bfloat16)
    start = torch.tensor(starts_of(counts), dtype=torch.int32).cuda()
    for _ in range(2):
        got = f.cache.attend(q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), query_start=start,
                             max_query=max(counts), softcap=softcap, window=window)
        f.check(q, table, lens, counts, got, softcap, window, many=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_ragged_batch(dim):
    g = torch.Generator().manual_seed(dim)
    lens = [1 + (i * 2999) % 9001 for i in range(30)] + [0, 30000]
    table, pool = random_tables(g, lens, 64)
    f = Filled(g, pool, 64, 2, dim, 2.0)
    q = torch.randn(32, 16, dim, generator=g).to(torch.bfloat16)
    got = f.cache.attend(q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), softcap=40.0)
    f.check(q, table, lens, [1] * 32, got, 40.0)
    assert bool((got[30] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 2, 40])
def test_what_lies_past_the_length_or_the_rows_does_not_count(dim, n):
    """NaN and infinite lines of other pages and slots, and of pages below the
    window, which the table may have no page for."""
    g = torch.Generator().manual_seed(4)
    page, ln = 32, 73 + n
    f = Filled(g, 7, page, 1, dim)
    table = torch.tensor([[1, 3, 2, 5]], dtype=torch.int32).cuda()
    lens = torch.tensor([ln], dtype=torch.int32).cuda()
    start = torch.tensor([0, n], dtype=torch.int32).cuda()
    q = torch.randn(n, 4, dim, generator=g).to(torch.bfloat16).cuda()
    call = dict(query_start=start, max_query=n)
    want = f.cache.attend(q, table, lens, **call)
    low = f.cache.attend(q, table, lens, window=20, **call)
    last, at = int(table[0, (ln - 1) // page]), (ln - 1) % page + 1
    cell = f.cache.v_scales.view(7, 1, page // 16, -1)
    for bad in (math.nan, math.inf):
        for other in (0, 4, 6):
            f.cache.k_scales[other] = bad
            f.cache.v_scales[other] = bad
        f.cache.k_scales[last, :, at:] = bad
        groups = dim // GROUP
        for slot in range(at, page):
            cell[last, 0, slot // 16, 32 * groups + slot % 16] = bad
            for line in range(2 * groups):
                cell[last, 0, slot // 16, (slot % 16 // 2 * 2 * groups + line) * 2 + slot % 2] = bad
        assert torch.equal(f.cache.attend(q, table, lens, **call).view(torch.int16), want.view(torch.int16))
        gone = table.clone()
        first = max(0, ln - n - 19) // page
        gone[0, :first] = -1
        for p in table[0, :first].tolist():
            f.cache.k_scales[p], f.cache.v_scales[p] = bad, bad
        assert torch.equal(f.cache.attend(q, gone, lens, window=20, **call).view(torch.int16), low.view(torch.int16))
        for p in table[0, :first].tolist():  # put back
            k, v = (t.cuda() for t in f.plain.tensors()[2:])
            f.cache.k_scales[p], f.cache.v_scales[p] = k[p], v[p]


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [3, 40])
def test_tokens_that_are_nan_reach_the_rows_that_see_them(dim, n):
    g = torch.Generator().manual_seed(12)
    page, before = 16, 21
    cache, _ = make_pair(8, page, 1, dim)
    table = torch.arange(8, dtype=torch.int32)[None].cuda()
    x = torch.randn(before + n, 1, dim, generator=g).cuda()

    def run(k, v):
        cache.append(k, v, table, torch.tensor([before + n], dtype=torch.int32).cuda(),
                     query_start=torch.tensor([0, before + n], dtype=torch.int32).cuda())
        q = x[-n:].expand(n, 4, dim).to(torch.bfloat16)
        return cache.attend(q, table, torch.tensor([before + n], dtype=torch.int32).cuda(),
                            query_start=torch.tensor([0, n], dtype=torch.int32).cuda(), max_query=n, window=9)

    good = run(x, x)
    for which in "kv":
        for at in (0, before - 9, before, before + n - 1):
            bad = x.clone()
            bad[at, 0, dim - 1] = math.inf if which == "k" else math.nan
            out = run(bad if which == "k" else x, x if which == "k" else bad)
            for i in range(n):
                seen = before + i - 9 < at <= before + i
                assert bool(out[i].isnan().all()) if seen else torch.equal(out[i].view(torch.int16), good[i].view(torch.int16)), (which, at, i)


@pytest.mark.gpu
def test_queries_that_are_not_finite_stay_in_their_rows():
    f, q, args, got = attend_case(6, 16, 1, 4, 128, [50, 9], [1, 1])
    q[0, 1, 3] = math.nan
    q[0, 2, 7] = math.inf
    out = f.cache.attend(q.cuda(), *args)
    assert bool(out[0, 1].isnan().all()) and bool(out[0, 2].isnan().all())
    for t, h in ((0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (1, 3)):
        assert torch.equal(out[t, h].view(torch.int16), got[t, h].view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attend_takes_any_strides(dim):
    f, q, args, got = attend_case(7, 16, 2, 4, dim, [50, 9, 130], [1, 1, 1])
    wide = torch.zeros(3, 4, dim + 3, dtype=torch.bfloat16)
    wide[:, :, 1 : dim + 1] = q
    out = torch.full((3, 4, dim + 2), 5.0, dtype=torch.bfloat16, device="cuda")
    res = f.cache.attend(wide.cuda()[:, :, 1 : dim + 1], *args, out=out[:, :, 1 : dim + 1])
    assert torch.equal(res.contiguous().view(torch.int16), got.view(torch.int16))
    assert bool((out[:, :, 0] == 5).all()) and bool((out[:, :, -1] == 5).all())
    table = torch.cat([args[0], args[0]], dim=1)[:, : args[0].shape[1]]  # a column of a wider table
    assert torch.equal(f.cache.attend(q.cuda(), table, args[1]).view(torch.int16), got.view(torch.int16))


@pytest.mark.gpu
def test_many_sequences():
    lens = [(i * 37) % 70 for i in range(2048)]
    attend_case(8, 16, 1, 2, 128, lens, [1] * 2048)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_pages_that_are_not_there(n):
    """Page ids out of range and lengths past the table set the status; what is
    there is attended to."""
    from se12_b200.device import device_status

    g = torch.Generator().manual_seed(2)
    f = Filled(g, 4, 16, 1, 128)
    q = torch.randn(n, 2, 128, generator=g).to(torch.bfloat16).cuda()
    start = torch.tensor([0, n], dtype=torch.int32).cuda()
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    for table, ln in (([[0, 4, 1, 2]], 60), ([[0, -1, 1, 2]], 60), ([[0, 1, 2, 3]], 65)):
        out = f.cache.attend(q, ints(table), ints([ln]), query_start=start)
        assert device_status(clear=True) == 2 and bool(torch.isfinite(out).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens_each", [1, 20])
def test_a_run_of_all_as_a_captured_step(dim, tokens_each):
    """Norms, rotation, append and attention in one graph, replayed as the
    sequences grow, on a stream of its own: the bits of eager calls."""
    from se12_b200.kv_cache import PagedKvCache

    g = torch.Generator().manual_seed(11)
    heads, q_heads, page, seqs = 2, 4, 16, 3
    pool, t = 3 * 40, seqs * tokens_each
    caches = [PagedKvCache(pool, page, heads, dim, "int4") for _ in range(2)]
    table = torch.randperm(pool, generator=g).to(torch.int32).view(seqs, 40).cuda()
    cos, sin = (x.cuda() for x in rope(g, 700, dim // 2))
    q_norm, k_norm = (torch.randn(dim, generator=g).cuda() for _ in "qk")
    lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    start = None if tokens_each == 1 else torch.arange(0, t + 1, tokens_each, dtype=torch.int32, device="cuda")
    y = torch.randn(t, q_heads + 2 * heads, dim, device="cuda")

    def step(cache):
        q = cache.append(y[:, q_heads : q_heads + heads], y[:, q_heads + heads :], table, lens, q=y[:, :q_heads], cos=cos, sin=sin,
                         query_start=start, q_norm=q_norm, k_norm=k_norm)
        return cache.attend(q, table, lens, query_start=start, max_query=tokens_each, softcap=50.0, window=100)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0])  # lens 0: nothing is stored
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(caches[0])
    torch.cuda.current_stream().wait_stream(side)
    for i in range(9):
        lens += tokens_each
        y.copy_(torch.randn(y.shape, generator=g))
        graph.replay()
        assert torch.equal(out.view(torch.int16), step(caches[1]).view(torch.int16))
    for a, b in zip(caches[0].decode(), caches[1].decode()):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes of codes: the last pages are the last pages."""
    from se12_b200.kv_cache import PagedKvCache

    page, heads, dim = 256, 8, 256
    pages = 2 * (1 << 32) // (page * heads * dim) + 40
    cache = PagedKvCache(pages, page, heads, dim, "int4")
    g = torch.Generator().manual_seed(1)
    n = 300
    x, y = torch.randn(n, heads, dim, generator=g).cuda(), torch.randn(n, heads, dim, generator=g).cuda()
    ids = [pages - 1, pages - 7]
    table, lens = torch.tensor([ids], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    small, near = PagedKvCache(2, page, heads, dim, "int4"), torch.tensor([[0, 1]], dtype=torch.int32).cuda()
    start = torch.tensor([0, n], dtype=torch.int32).cuda()
    for c, where in ((cache, table), (small, near)):
        c.append(x, y, where, lens, query_start=start)
    assert torch.equal(cache.k_codes[ids], small.k_codes) and torch.equal(cache.v_scales[ids], small.v_scales)
    assert bool((cache.k_codes[:2] == 0).all())
    for rows in (1, 30):
        q = torch.randn(rows, heads, dim, generator=g).to(torch.bfloat16).cuda()
        at = torch.tensor([0, rows], dtype=torch.int32).cuda()
        a, b = (c.attend(q, where, lens, query_start=at) for c, where in ((cache, table), (small, near)))
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    assert torch.equal(cache.decode(table[0])[1], small.decode()[1])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 60])
def test_calls_at_once_on_two_streams(n):
    """Long and short batches side by side, again and again, each on a stream of
    its own and one of them as a graph besides: the bits of calls one by one."""
    cases = []
    for seed, lens in ((1, [9000, 3, 700]), (2, [40, 5000, 5000])):
        g = torch.Generator().manual_seed(seed)
        lens = [max(ln, n) for ln in lens]
        table, pool = random_tables(g, lens, 32)
        f = Filled(g, pool, 32, 2, 128)
        q = torch.randn(3 * n, 8, 128, generator=g).to(torch.bfloat16).cuda()
        start = torch.arange(0, 3 * n + 1, n, dtype=torch.int32).cuda()
        table, lens = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()

        def call(f=f, q=q, table=table, lens=lens, start=start):
            return f.cache.attend(q, table, lens, query_start=start, max_query=n, window=4000)

        cases.append((call, call(), torch.cuda.Stream()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = cases[0][0]()
    torch.cuda.synchronize()
    for _ in range(20):
        graph.replay()
        outs = []
        for call, want, stream in cases:
            with torch.cuda.stream(stream):
                outs.append((call(), want))
        torch.cuda.synchronize()
        assert torch.equal(held.view(torch.int16), cases[0][1].view(torch.int16))
        for got, want in outs:
            assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 3, 70])
def test_rows_of_no_sequence_stay_as_they_are(dim, n):
    g = torch.Generator().manual_seed(dim + n)
    lens = [100, n + 7]
    table, pool = random_tables(g, lens, 16)
    f = Filled(g, pool, 16, 1, dim)
    q = torch.randn(2 * n + 9, 4, dim, generator=g).to(torch.bfloat16)
    start = torch.tensor([4, 4 + n, 4 + 2 * n], dtype=torch.int32).cuda()
    out = torch.full(q.shape, 3.0, dtype=torch.bfloat16, device="cuda")
    f.cache.attend(q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), query_start=start, max_query=n, out=out)
    assert bool((out[:4] == 3).all()) and bool((out[4 + 2 * n :] == 3).all())
    f.check(q[4 : 4 + 2 * n], table, lens, [n, n], out[4 : 4 + 2 * n], many=n * 4 > 16)
