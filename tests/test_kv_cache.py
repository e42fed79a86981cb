"""The paged 8-bit key/value cache and attention over it, against plain
implementations: the stored codes and scales bit for bit (the store's
arithmetic is elementary fp32 operations), attention against 64-bit sums
over the stored values.

Attention's tolerance, elementwise: the output is rounded to BF16 (half a
unit in the last place of o); a weight carries an FP16 rounding (2^-11) and the fp32 errors of the
logits, the exponential and the sum (together below 2^-12 for the logits
here, |s| < 100), so 2^-10 of sum_j p_j |v_j|; a weight below FP16's normal
range is off by 2^-25 of the largest, so 2^-24 of the length times the
largest |v|.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

QMAX = {"int8": 127.0, "e4m3": 448.0}


# ------------------------------------------------------------------ plain implementation (CPU)


def value_of(codes: torch.Tensor, kind: str) -> torch.Tensor:
    return codes.float() if kind == "int8" else codes.view(torch.float8_e4m3fn).float()


def code_of(x: torch.Tensor, kind: str) -> torch.Tensor:
    return torch.round(x).to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn).view(torch.int8)


def least_scale(amax: float, kind: str) -> float:
    if not math.isfinite(amax):
        return math.nan
    e = -100
    while amax > QMAX[kind] * 2.0**e:
        e += 1
    return 2.0**e


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x [..., dim] fp32 turned by cos, sin [rotary / 2]."""
    n = cos.shape[-1]
    out = x.clone()
    a, b = (x[..., 0 : 2 * n : 2], x[..., 1 : 2 * n : 2]) if interleaved else (x[..., :n], x[..., n : 2 * n])
    first, second = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        out[..., 0 : 2 * n : 2], out[..., 1 : 2 * n : 2] = first, second
    else:
        out[..., :n], out[..., n : 2 * n] = first, second
    return out


class PlainCache:
    """The same cache in elementary CPU operations, one block at a time."""

    def __init__(self, pages, page_size, heads, dim, kind):
        self.page_size, self.kind, self.heads, self.dim = page_size, kind, heads, dim
        self.codes = {w: torch.zeros(pages, heads, page_size, dim, dtype=torch.int8) for w in "kv"}
        self.scales = {w: torch.ones(pages, heads) for w in "kv"}

    def append(self, k, v, table, lens, starts, cos=None, sin=None, interleaved=False, q=None):
        out = None if q is None else torch.zeros(q.shape, dtype=torch.bfloat16)
        for b, ln in enumerate(lens):
            n = starts[b + 1] - starts[b]
            blocks: dict = {}
            for i in range(n):
                pos, t = ln - n + i, starts[b] + i
                if pos < 0:
                    continue
                turn = (lambda x: x) if cos is None else (lambda x, p=pos: rotate(x, cos[p], sin[p], interleaved))
                if q is not None:
                    out[t] = turn(q[t].float()).to(torch.bfloat16)
                blocks.setdefault(pos // self.page_size, []).append((pos % self.page_size, turn(k[t].float()), v[t].float()))
            for column, rows in blocks.items():
                page, first = int(table[b, column]), rows[0][0]
                for w, which in (("k", 1), ("v", 2)):
                    for h in range(self.heads):
                        new = torch.stack([r[which][h] for r in rows])
                        need = least_scale(float(new.abs().max()) if bool(torch.isfinite(new).all()) else math.inf, self.kind)
                        before = float(self.scales[w][page, h])
                        now = need if first == 0 else math.nan if math.isnan(need) or math.isnan(before) else max(need, before)
                        block = self.codes[w][page, h]
                        if first and now > before:
                            block[:first] = code_of(value_of(block[:first], self.kind) * (before / now), self.kind)
                        self.scales[w][page, h] = now
                        for r, x in zip(rows, new):
                            block[r[0]] = 0 if math.isnan(now) else code_of(x / now, self.kind)
        return out

    def values(self, w):
        return value_of(self.codes[w], self.kind).double() * self.scales[w].double()[:, :, None, None]


def plain_attend(q, keys, values, table, lens, starts, scale, softcap, window):
    """(output, sum of p |v|, largest |v|) in 64 bits; keys, values [pages, heads, page, dim]."""
    tokens, q_heads, dim = q.shape
    heads, page = keys.shape[1], keys.shape[2]
    out, size = torch.zeros(tokens, q_heads, dim, dtype=torch.float64), torch.zeros(tokens, q_heads, dim, dtype=torch.float64)
    biggest = torch.zeros(tokens, q_heads, 1, dtype=torch.float64)
    for b, ln in enumerate(lens):
        n = starts[b + 1] - starts[b]
        if ln == 0 or n == 0:
            continue
        ids = [int(p) for p in table[b, : (ln + page - 1) // page]]
        for h in range(heads):
            k = torch.cat([keys[p, h] for p in ids])[:ln]
            v = torch.cat([values[p, h] for p in ids])[:ln]
            for i in range(n):
                pos, t = ln - n + i, starts[b] + i
                low = max(0, pos - window + 1) if window else 0
                if pos < 0:
                    continue
                for g in range(h * q_heads // heads, (h + 1) * q_heads // heads):
                    s = k[low : pos + 1] @ q[t, g].double() * scale
                    if softcap:
                        s = softcap * torch.tanh(s / softcap)
                    p = torch.softmax(s, 0)
                    out[t, g] = p @ v[low : pos + 1]
                    size[t, g] = p @ v[low : pos + 1].abs()
                    biggest[t, g] = v[low : pos + 1].abs().max()
    return out, size, biggest


def check_attend(got, want, size, biggest, length):
    half_unit = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=1e-300))) - 8)
    tol = half_unit + 2.0**-10 * size + 2.0**-24 * length * biggest
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol.clamp(min=1e-300)).max()):.2f} of the tolerance"


# ------------------------------------------------------------------ CPU: refusals


@pytest.mark.parametrize("args", [
    dict(pages=0), dict(kv_heads=0), dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(head_dim=8),
    dict(head_dim=264), dict(head_dim=100), dict(kind="fp8"),
])
def test_cache_refuses_bad_shapes(args):
    from se12_b200.kv_cache import PagedKvCache

    full = dict(pages=4, page_size=16, kv_heads=2, head_dim=64, kind="int8")
    full.update(args)
    with pytest.raises(ValueError):
        PagedKvCache(**full)


def test_abi_refuses_bad_arguments_without_a_device():
    from se12_b200 import _build, _lib

    _build.build()
    lib = _lib.load()
    handle = ctypes.c_void_p()
    good = dict(pages=4, page_size=16, kv_heads=2, head_dim=64, kind=0, k_codes=256, v_codes=256, k_scales=256, v_scales=256)

    def create(**changed):
        return lib.se12_kv_cache_create(ctypes.byref(_lib.Se12KvPagesStruct(**{**good, **changed})), ctypes.byref(handle))

    assert lib.se12_kv_cache_create(None, ctypes.byref(handle)) == 1
    assert create(pages=0) == 1 and create(page_size=24) == 1 and create(head_dim=24) == 1 and create(k_codes=None) == 1
    assert create(kind=2) == 2  # SE12_ERR_UNSUPPORTED_FORMAT
    assert create(v_codes=257) == 3  # SE12_ERR_MISALIGNED
    assert create(pages=1 << 27) == 1 and b"31 bits" in lib.se12_last_error()
    assert lib.se12_kv_append(None, None, None, None) == 1
    assert lib.se12_kv_attend(None, None, None, None, 0, None) == 1
    assert lib.se12_kv_decode(None, None, 1, None, None, None) == 1
    assert lib.se12_kv_attend_workspace_bytes(None) == 0
    lib.se12_kv_cache_destroy(None)


def test_least_scale_holds_the_largest_magnitude():
    for kind in QMAX:
        for x in (0.0, 1e-40, 1e-30, 0.7, 127.0, 127.00001, 448.0, 449.0, 3e38):
            s = least_scale(x, kind)
            assert x <= QMAX[kind] * s and (s == 2.0**-100 or x > QMAX[kind] * s / 2)


# ------------------------------------------------------------------ GPU helpers


def random_tables(g, lens, page, spare=3):
    """A page table with the sequences' pages in random order, and the pool's size."""
    need = [(ln + page - 1) // page for ln in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g)
    table = torch.full((len(lens), max(max(need), 1) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    table[:, -1] = 1 << 30  # entries past a sequence's pages may hold anything
    return table, pool


def starts_of(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


def make_pair(pages, page, heads, dim, kind):
    from se12_b200.kv_cache import PagedKvCache

    return PagedKvCache(pages, page, heads, dim, kind), PlainCache(pages, page, heads, dim, kind)


def same_cache(cache, plain):
    for w, codes, scales in (("k", cache.k_codes, cache.k_scales), ("v", cache.v_codes, cache.v_scales)):
        assert torch.equal(scales.cpu().view(torch.int32), plain.scales[w].view(torch.int32)) or (
            torch.equal(scales.cpu().isnan(), plain.scales[w].isnan())
            and torch.equal(scales.cpu().nan_to_num(), plain.scales[w].nan_to_num()))
        assert torch.equal(codes.cpu(), plain.codes[w]), f"{w} codes"


def rope(g, rows, half):
    angle = torch.rand(rows, half, generator=g) * 6.3
    return torch.cos(angle), torch.sin(angle)


# ------------------------------------------------------------------ append


APPEND = [
    # kind, dtype, page, heads, q_heads, dim, rotary (0: none), interleaved
    ("int8", torch.float32, 16, 2, 4, 256, 256, False),
    ("e4m3", torch.float32, 32, 2, 6, 128, 128, False),
    ("int8", torch.bfloat16, 64, 3, 3, 128, 128, False),
    ("e4m3", torch.bfloat16, 16, 1, 8, 256, 256, False),
    ("int8", torch.float32, 16, 2, 2, 64, 64, False),
    ("int8", torch.float32, 16, 2, 2, 96, 32, False),    # partial rotation
    ("e4m3", torch.bfloat16, 16, 2, 2, 80, 80, True),    # neighbouring pairs
    ("int8", torch.bfloat16, 128, 1, 2, 192, 64, True),
    ("e4m3", torch.float32, 16, 1, 1, 16, 2, False),
    ("int8", torch.float32, 256, 2, 2, 128, 0, False),   # no rotation
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype,page,heads,q_heads,dim,rotary,interleaved", APPEND)
@pytest.mark.parametrize("steps", [
    [[1, 1, 1, 1, 1]] * 3,                                    # next tokens
    [[40, 1, 0, 17, 3], [1, 16, 33, 0, 2], [5, 5, 5, 5, 5]],  # prompts, continued
    [[300, 0, 0, 0, 1], [1, 1, 1, 1, 1]],
])
def test_append_stores_the_same_codes(kind, dtype, page, heads, q_heads, dim, rotary, interleaved, steps):
    g = torch.Generator().manual_seed(dim + page)
    counts = [sum(s[b] for s in steps) for b in range(5)]
    table, pool = random_tables(g, counts, page)
    cache, plain = make_pair(pool, page, heads, dim, kind)
    cos, sin = rope(g, max(counts), rotary // 2) if rotary else (None, None)
    dev_table = table.cuda()
    lens = [0] * 5
    for step, new in enumerate(steps):
        lens = [a + b for a, b in zip(lens, new)]
        starts = starts_of(new)
        # q, k and v side by side; magnitudes grow, so that blocks' scales do
        y = torch.randn(starts[-1], q_heads + 2 * heads, dim, generator=g) * 3.0**step * (1 + 9 * torch.rand(dim, generator=g))
        y = y.to(dtype)
        q, k, v = y[:, :q_heads], y[:, q_heads : q_heads + heads], y[:, q_heads + heads :]
        want = plain.append(k, v, table, lens, starts, cos, sin, interleaved, q)
        d = y.cuda()
        start = None if all(n == 1 for n in new) else torch.tensor(starts, dtype=torch.int32).cuda()
        got = cache.append(d[:, q_heads : q_heads + heads], d[:, q_heads + heads :], dev_table,
                           torch.tensor(lens, dtype=torch.int32).cuda(), q=d[:, :q_heads], query_start=start,
                           cos=None if cos is None else cos.cuda(), sin=None if sin is None else sin.cuda(),
                           interleaved=interleaved)
        assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
        same_cache(cache, plain)
    keys, values = cache.decode()
    assert torch.equal(keys.double().cpu(), plain.values("k")) and torch.equal(values.double().cpu(), plain.values("v"))
    some = torch.tensor([int(table[0, 0]), 0, int(table[0, 0])], dtype=torch.int32)
    keys, values = cache.decode(some.cuda())
    assert torch.equal(keys.double().cpu(), plain.values("k")[some.long()])
    assert torch.equal(values.double().cpu(), plain.values("v")[some.long()])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens_each", [1, 3])
@pytest.mark.parametrize("dim", [128, 256])
def test_append_takes_any_strides(tokens_each, dim):
    """Rows at odd offsets, heads far apart, an output with its own strides,
    a rotation table cut from a wider one: the scalar path, the same codes."""
    g = torch.Generator().manual_seed(5)
    heads, q_heads, seqs, page = 2, 4, 3, 16
    lens = [20, 7, 33]
    table, pool = random_tables(g, lens, page)
    cache, plain = make_pair(pool, page, heads, dim, "int8")
    cos, sin = rope(g, 40, dim // 2)
    starts = starts_of([tokens_each] * seqs)
    t = starts[-1]
    start = None if tokens_each == 1 else torch.tensor(starts, dtype=torch.int32).cuda()

    def odd(x):  # the same values, one element past an aligned address, head stride dim + 3
        wide = torch.zeros(t, x.shape[1], dim + 3)
        wide[:, :, 1 : dim + 1] = x
        return wide.cuda()[:, :, 1 : dim + 1]

    q, k, v = torch.randn(t, q_heads, dim, generator=g), torch.randn(t, heads, dim, generator=g), torch.randn(t, heads, dim, generator=g)
    want = plain.append(k, v, table, lens, starts, cos, sin, False, q)
    out = torch.full((t, q_heads, dim + 5), 7.0, dtype=torch.bfloat16, device="cuda")
    wide = torch.zeros(2, 40, dim // 2 + 1)
    wide[0, :, 1:], wide[1, :, 1:] = cos, sin
    wide = wide.cuda()
    got = cache.append(odd(k), odd(v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), q=odd(q), query_start=start,
                       cos=wide[0][:, 1:], sin=wide[1][:, 1:], q_out=out[:, :, 2 : dim + 2])
    assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
    assert bool((out[:, :, :2] == 7).all()) and bool((out[:, :, dim + 2 :] == 7).all())
    same_cache(cache, plain)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_repeated_growth_stays_below_a_step(kind):
    """Tokens whose magnitudes double again and again, appended one by one:
    the older values stay within the sum of the roundings. int8: each growth
    by 2^g rounds to half of the new step, and the steps at least double, so
    below one step of the last scale. e4m3: a relative 2^-4 at most once
    (exponent shifts are exact) plus half of the subnormal step 2^-9 each time."""
    g = torch.Generator().manual_seed(2)
    page, dim = 64, 128
    x = torch.randn(page, 1, dim, generator=g) * 2.0 ** (torch.arange(page) / 5.0)[:, None, None]
    cache, plain = make_pair(2, page, 1, dim, kind)
    table = torch.tensor([[1]], dtype=torch.int32)
    for i in range(page):
        lens = torch.tensor([i + 1], dtype=torch.int32).cuda()
        cache.append(x[i : i + 1].cuda(), x[i : i + 1].cuda(), table.cuda(), lens)
        plain.append(x[i : i + 1], x[i : i + 1], table, [i + 1], [0, 1])
    same_cache(cache, plain)
    keys, _ = cache.decode()
    step = float(cache.k_scales[1, 0])
    err = (keys[1, 0].double().cpu() - x[:, 0].double()).abs()
    assert float(err.max()) <= step if kind == "int8" else bool((err <= 2.0**-4 * x[:, 0].abs() + 2.0**-9 * step).all())


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_value_that_is_not_finite_poisons_its_block(prompt, bad):
    page, dim = 16, 128
    cache, plain = make_pair(3, page, 2, dim, "int8")
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(17, 2, dim, generator=g)
    x[9, 1, 5] = bad

    def feed(a, b):
        cache.append(x[a:b].cuda(), x[a:b].cuda(), table.cuda(), torch.tensor([b], dtype=torch.int32).cuda(),
                     query_start=torch.tensor([0, b - a], dtype=torch.int32).cuda() if prompt else None)
        plain.append(x[a:b], x[a:b], table, [b], [0, b - a])

    for a, b in [(0, 5), (5, 12), (12, 17)] if prompt else [(i, i + 1) for i in range(17)]:
        feed(a, b)
    same_cache(cache, plain)
    assert bool(cache.k_scales[2, 1].isnan()) and not bool(cache.k_scales[2, 0].isnan()) and not bool(cache.k_scales[0].isnan().any())
    q = torch.randn(1, 4, dim, generator=g).to(torch.bfloat16)
    out = cache.attend(q.cuda(), table.cuda(), torch.tensor([17], dtype=torch.int32).cuda()).cpu()
    assert bool(out[0, 2:].isnan().all()) and not bool(out[0, :2].isnan().any())
    # outside the window the poisoned block does not count
    out = cache.attend(q.cuda(), table.cuda(), torch.tensor([17], dtype=torch.int32).cuda(), window=1).cpu()
    assert not bool(out.isnan().any())
    # a page that starts anew is clean again
    cache.append(x[:1].cuda(), x[:1].cuda(), table.cuda(), torch.tensor([1], dtype=torch.int32).cuda())
    assert not bool(cache.k_scales.isnan().any())


@pytest.mark.gpu
def test_padding_rows_store_nothing():
    cache, _ = make_pair(3, 16, 2, 128, "int8")
    before = cache.k_codes.clone()
    table = torch.full((2, 1), -1, dtype=torch.int32, device="cuda")
    x = torch.randn(2, 2, 128, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    cos = torch.ones(1, 64, device="cuda")
    for start in (None, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")):
        q = cache.append(x, x, table, lens, q=x, cos=cos, sin=cos, query_start=start)
        assert bool((q == 0).all()) and torch.equal(cache.k_codes, before)
        assert bool((cache.attend(q, table, lens, query_start=start) == 0).all())
    # more new rows than the sequence is long: the first ones are padding
    q = cache.append(x, x, torch.tensor([[1]], dtype=torch.int32, device="cuda"), lens[:1] + 1, q=x,
                     query_start=torch.tensor([0, 2], dtype=torch.int32, device="cuda"))
    assert bool((q[0] == 0).all()) and bool((q[1] == x[1].to(torch.bfloat16)).all())
    assert bool((cache.k_codes[1, :, 0] != 0).any()) and bool((cache.k_codes[1, :, 1:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", [False, True])
def test_indexes_out_of_range_set_the_status(prompt):
    from se12_b200.device import device_status

    cache, _ = make_pair(3, 16, 2, 128, "int8")
    x = torch.randn(1, 2, 128, device="cuda")
    start = torch.tensor([0, 1], dtype=torch.int32, device="cuda") if prompt else None
    cos = torch.ones(4, 64, device="cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for table, lens, table_cos in ((ints([[3]]), ints([1]), None), (ints([[-1]]), ints([1]), None), (ints([[0]]), ints([17]), None),
                                   (ints([[0]]), ints([5]), cos)):
        q = cache.append(x, x, table, lens, q=x, cos=table_cos, sin=table_cos, query_start=start)
        assert device_status() == 2
        assert bool((cache.k_codes == 0).all()) and (table_cos is None or bool((q == 0).all()))
        if table_cos is None:
            out = cache.attend(x.to(torch.bfloat16), table, lens, query_start=start)
            assert device_status() == 2 and bool(torch.isfinite(out).all())
    keys, _ = cache.decode(ints([0, 7]))
    assert device_status() == 2 and bool((keys[1] == 0).all())


# ------------------------------------------------------------------ attention


def filled(g, pool, page, heads, dim, kind, spread=1.0):
    """A cache whose blocks hold random codes, with scales 2^(+-spread)."""
    from se12_b200.kv_cache import PagedKvCache

    tensors = []
    for _ in range(2):
        x = torch.randn(pool, heads, page, dim, generator=g)
        x *= 2.0 ** ((torch.rand(pool, heads, 1, 1, generator=g) * 2 - 1) * spread)
        s = torch.tensor([[least_scale(m, kind) for m in page] for page in x.abs().amax(dim=(2, 3)).tolist()])
        tensors.append((code_of(x / s[:, :, None, None], kind), s))
    (k, ks), (v, vs) = tensors
    cache = PagedKvCache.from_tensors(k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), kind)
    return cache, value_of(k, kind).double() * ks.double()[:, :, None, None], value_of(v, kind).double() * vs.double()[:, :, None, None]


def attend_case(seed, kind, page, heads, q_heads, dim, lens, counts, softcap=0.0, window=0, spread=1.0, q_scale=1.0,
                max_query=None, scale=None):
    g = torch.Generator().manual_seed(seed)
    table, pool = random_tables(g, lens, page)
    cache, keys, values = filled(g, pool, page, heads, dim, kind, spread)
    starts = starts_of(counts)
    q = (torch.randn(starts[-1], q_heads, dim, generator=g) * q_scale).to(torch.bfloat16)
    start = None if all(n == 1 for n in counts) and max_query is None else torch.tensor(starts, dtype=torch.int32).cuda()
    args = (table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    got = cache.attend(q.cuda(), *args, query_start=start, softcap=softcap, window=window, scale=scale, max_query=max_query)
    want = plain_attend(q, keys, values, table, lens, starts, dim**-0.5 if scale is None else scale, softcap, window)
    check_attend(got, *want, max(lens))
    again = cache.attend(q.cuda(), *args, query_start=start, softcap=softcap, window=window, scale=scale, max_query=max_query)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    return cache, q, args, got


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [128, 256])
def test_attend_lengths_around_pages_and_tiles(kind, page, dim):
    attend_case(page + dim, kind, page, 2, 4, dim, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 255, 256, 257, 700], [1] * 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 96, 112, 144, 192, 240])
def test_attend_head_dimensions(dim):
    attend_case(dim, "int8" if dim % 32 else "e4m3", 32, 2, 2, dim, [5, 100], [1, 1], softcap=20.0)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,q_heads", [(1, 1), (1, 8), (2, 6), (4, 20), (1, 16), (2, 34), (3, 3), (1, 64)])
@pytest.mark.parametrize("dim", [128, 256])
def test_attend_head_layouts(heads, q_heads, dim):
    attend_case(heads * 100 + q_heads, "int8", 16, heads, q_heads, dim, [77, 3], [1, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("window", [0, 1, 7, 16, 100])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
def test_attend_windows_and_several_queries(kind, dim, window, softcap):
    """Drafted tokens and prompt chunks, idle sequences, and more rows than
    the sequence is long (the first ones see nothing)."""
    counts = [1, 4, 0, 19, 33, 3, 0]
    cache, q, args, got = attend_case(window + dim, kind, 16, 2, 6, dim, [40, 4, 9, 200, 33, 2, 0], counts, softcap=softcap,
                                      window=window)
    start = torch.tensor(starts_of(counts), dtype=torch.int32).cuda()
    bound = cache.attend(q.cuda(), *args, query_start=start, softcap=softcap, window=window, max_query=33)
    assert torch.allclose(bound.float(), got.float(), rtol=2.0**-6, atol=2.0**-7)
    assert bool((got[starts_of(counts)[5]] == 0).all())  # position -1


@pytest.mark.gpu
@pytest.mark.parametrize("dim,q_heads,heads", [(128, 8, 1), (256, 4, 2), (128, 12, 1), (256, 12, 1)])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 17, 70])
def test_attend_query_counts(dim, q_heads, heads, n):
    attend_case(n, "e4m3", 64, heads, q_heads, dim, [300, n], [n, n], max_query=n)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [5000, 20011])
@pytest.mark.parametrize("dim", [128, 256])
def test_attend_one_long_sequence_is_split(length, dim):
    attend_case(length, "int8", 128, 1, 4, dim, [length], [1], softcap=30.0)
    attend_case(length, "e4m3", 16, 2, 2, dim, [length, 1, 3, length // 2], [1, 1, 1, 1], window=length // 3)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_attend_blocks_of_very_different_scales(kind):
    """Scales from 2^-40 to 2^40: a weight's precision does not depend on
    what other blocks hold."""
    attend_case(9, kind, 16, 2, 4, 128, [200, 45], [1, 1], spread=40.0, q_scale=2.0**-41)
    attend_case(10, kind, 16, 2, 4, 256, [200, 45], [2, 2], spread=18.0, scale=2.0**-20)


@pytest.mark.gpu
def test_attend_weights_of_zero_values_count():
    """Tokens whose values are all zero still take their share."""
    from se12_b200.kv_cache import PagedKvCache

    cache = PagedKvCache(2, 16, 1, 128)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    k = torch.zeros(32, 1, 128, device="cuda")
    v = torch.zeros(32, 1, 128, device="cuda")
    v[16:] = 8.0
    lens = torch.tensor([32], dtype=torch.int32, device="cuda")
    cache.append(k, v, table, lens, query_start=torch.tensor([0, 32], dtype=torch.int32, device="cuda"))
    out = cache.attend(torch.ones(1, 2, 128, dtype=torch.bfloat16, device="cuda"), table, lens)
    assert bool((out == 4.0).all())


def check_on_gpu(cache, q, table, lens, counts, got, softcap, window):
    """Against 64-bit sums on the GPU over the cache's values (BF16 holds them
    exactly), with the tolerance above; for batches too large for the CPU."""
    keys, values = cache.decode()
    page, dim, group = cache.page_size, cache.head_dim, q.shape[1] // cache.kv_heads
    starts = starts_of(counts)
    for b, ln in enumerate(lens):
        if counts[b] == 0 or ln == 0:
            continue
        ids = table[b, : (ln + page - 1) // page].long()
        rows = slice(starts[b], starts[b + 1])
        i, j = torch.arange(ln - counts[b], ln, device="cuda"), torch.arange(ln, device="cuda")
        hidden = j[None, :] > i[:, None]
        if window:
            hidden |= i[:, None] - j[None, :] >= window
        for h in range(cache.kv_heads):
            k, v = (t[ids, h].reshape(-1, dim)[:ln].double() for t in (keys, values))
            for g in range(h * group, (h + 1) * group):
                s = q[rows, g].double() @ k.T * dim**-0.5
                s = softcap * torch.tanh(s / softcap) if softcap else s
                p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
                want, size = p @ v, p @ v.abs()
                half_unit = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=1e-300))) - 8)
                tol = half_unit + 2.0**-10 * size + 2.0**-24 * ln * v.abs().max()
                assert bool(((got[rows, g].double() - want).abs() <= tol).all()), (b, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group,n", [(1, 1), (8, 1), (8, 2), (8, 3), (8, 4), (11, 3), (8, 6)])
@pytest.mark.parametrize("long", [0, 3000])
def test_attend_many_short_pairs(dim, group, n, long):
    """Sequences of no token to a few tiles, alone and around a long one: runs
    that begin and end anywhere in a pair, or hold no token of it."""
    g = torch.Generator().manual_seed(dim + group * n)
    lens = [(i * 37) % 90 for i in range(150)] + [0, n, 700]
    if long:
        lens[70] = long
    counts = [min(1 + i % n, ln) if ln else 1 for i, ln in enumerate(lens)]
    table, pool = random_tables(g, lens, 16)
    cache, _, _ = filled(g, pool, 16, 2, dim, "int8", 2.0)
    q = (torch.randn(sum(counts), 2 * group, dim, generator=g) * 2).to(torch.bfloat16).cuda()
    start = torch.tensor(starts_of(counts), dtype=torch.int32).cuda()
    for _ in range(2):
        got = cache.attend(q, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), query_start=start, max_query=n)
        check_on_gpu(cache, q, table.cuda(), lens, counts, got, 0.0, 0)
        for b, ln in enumerate(lens):
            if ln == 0:
                assert not got[starts_of(counts)[b] : starts_of(counts)[b + 1]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,q_heads,dim,page", [("int8", 4, 32, 128, 16), ("e4m3", 8, 16, 256, 64), ("int8", 2, 24, 192, 32)])
@pytest.mark.parametrize("softcap,window", [(0.0, 0), (30.0, 700)])
def test_attend_many_tiles_per_cta(kind, heads, q_heads, dim, page, softcap, window):
    """Runs of many tiles of many pairs: drafted tokens and prompt chunks, also
    sequences whose chunk is all they have."""
    g = torch.Generator().manual_seed(heads)
    counts = [2 + i % 5 for i in range(20)] + [300, 0, 70, 513]
    lens = [n + (i * 397) % 2500 for i, n in enumerate(counts)]
    lens[-2] = 70
    table, pool = random_tables(g, lens, page)
    cache, _, _ = filled(g, pool, page, heads, dim, kind, 2.0)
    q = (torch.randn(sum(counts), q_heads, dim, generator=g) * 2).to(torch.bfloat16).cuda()
    start = torch.tensor(starts_of(counts), dtype=torch.int32).cuda()
    for _ in range(2):
        got = cache.attend(q, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), query_start=start,
                           max_query=max(counts), softcap=softcap, window=window)
        check_on_gpu(cache, q, table.cuda(), lens, counts, got, softcap, window)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kind", [(128, "e4m3"), (256, "int8")])
def test_attend_long_ragged_batch(dim, kind):
    """Next tokens of a ragged batch over long sequences: runs of many pairs,
    pairs of many runs."""
    g = torch.Generator().manual_seed(dim)
    lens = [1 + (i * 2999) % 9001 for i in range(30)] + [0, 30000]
    table, pool = random_tables(g, lens, 64)
    cache, _, _ = filled(g, pool, 64, 2, dim, kind, 2.0)
    q = torch.randn(32, 16, dim, generator=g).to(torch.bfloat16).cuda()
    got = cache.attend(q, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), softcap=40.0)
    check_on_gpu(cache, q, table.cuda(), lens, [1] * 32, got, 40.0, 0)
    assert bool((got[30] == 0).all())


@pytest.mark.gpu
def test_attend_ignores_what_lies_past_the_length():
    """NaN codes and scales of other pages and slots do not reach the output."""
    g = torch.Generator().manual_seed(4)
    cache, keys, values = filled(g, 4, 32, 1, 128, "e4m3")
    table = torch.tensor([[1, 3, 2]], dtype=torch.int32).cuda()
    lens = torch.tensor([41], dtype=torch.int32).cuda()
    q = torch.randn(1, 4, 128, generator=g).to(torch.bfloat16).cuda()
    want = cache.attend(q, table, lens)
    for codes in (cache.k_codes, cache.v_codes):
        codes[3, :, 9:] = 0x7F  # NaN
        codes[2] = -1
    for scales in (cache.k_scales, cache.v_scales):
        scales[2] = math.nan
        scales[0] = math.inf
    assert torch.equal(cache.attend(q, table, lens).view(torch.int16), want.view(torch.int16))


@pytest.mark.gpu
def test_attend_queries_that_are_not_finite_stay_in_their_rows():
    cache, q, args, got = attend_case(6, "int8", 16, 1, 4, 128, [50, 9], [1, 1])
    q[0, 1, 3] = math.nan
    q[0, 2, 7] = math.inf
    out = cache.attend(q.cuda(), *args)
    assert bool(out[0, 1].isnan().all()) and bool(out[0, 2].isnan().all())
    for t, h in ((0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (1, 3)):
        assert torch.equal(out[t, h].view(torch.int16), got[t, h].view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [128, 256])
def test_attend_takes_any_strides(dim):
    cache, q, args, got = attend_case(7, "int8", 16, 2, 4, dim, [50, 9, 130], [1, 1, 1])
    wide = torch.zeros(3, 4, dim + 3, dtype=torch.bfloat16)
    wide[:, :, 1 : dim + 1] = q
    out = torch.full((3, 4, dim + 2), 5.0, dtype=torch.bfloat16, device="cuda")
    res = cache.attend(wide.cuda()[:, :, 1 : dim + 1], *args, out=out[:, :, 1 : dim + 1])
    assert torch.equal(res.contiguous().view(torch.int16), got.view(torch.int16))
    assert bool((out[:, :, 0] == 5).all()) and bool((out[:, :, -1] == 5).all())
    # a column of a wider table
    table = torch.cat([args[0], args[0]], dim=1)[:, : args[0].shape[1]]
    assert torch.equal(cache.attend(q.cuda(), table, args[1]).view(torch.int16), got.view(torch.int16))


@pytest.mark.gpu
def test_attend_many_sequences():
    lens = [(i * 37) % 70 for i in range(600)]
    attend_case(8, "int8", 16, 1, 2, 128, lens, [1] * 600)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 codes: the last pages are the last pages."""
    from se12_b200.kv_cache import PagedKvCache

    page, heads, dim = 256, 8, 256
    pages = (1 << 32) // (page * heads * dim) + 40
    cache = PagedKvCache(pages, page, heads, dim)
    g = torch.Generator().manual_seed(1)
    n = 300
    x, y = torch.randn(n, heads, dim, generator=g), torch.randn(n, heads, dim, generator=g)
    ids = [pages - 1, pages - 7]
    table = torch.tensor([ids], dtype=torch.int32)
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    cache.append(x.cuda(), y.cuda(), table.cuda(), lens, query_start=torch.tensor([0, n], dtype=torch.int32).cuda())
    small = PlainCache(2, page, heads, dim, "int8")
    small.append(x, y, torch.tensor([[0, 1]]), [n], [0, n])
    assert torch.equal(cache.k_codes[ids].cpu(), small.codes["k"]) and torch.equal(cache.v_codes[ids].cpu(), small.codes["v"])
    assert bool((cache.k_codes[:2] == 0).all())
    q = torch.randn(1, heads, dim, generator=g).to(torch.bfloat16)
    got = cache.attend(q.cuda(), table.cuda(), lens)
    want = plain_attend(q, small.values("k"), small.values("v"), torch.tensor([[0, 1]]), [n], [0, 1], dim**-0.5, 0.0, 0)
    check_attend(got, *want, n)
    keys, _ = cache.decode(torch.tensor(ids, dtype=torch.int32).cuda())
    assert torch.equal(keys.double().cpu(), small.values("k"))


@pytest.mark.gpu
def test_a_captured_step_follows_lengths_and_tables():
    """append + attend in one graph, replayed with other lengths and pages:
    the bits of the eager calls; also on a stream of its own."""
    from se12_b200.kv_cache import PagedKvCache

    g = torch.Generator().manual_seed(11)
    heads, q_heads, dim, page, seqs = 2, 4, 128, 16, 3
    pool = 3 * 40
    caches = [PagedKvCache(pool, page, heads, dim, "int8") for _ in range(2)]
    table = torch.randperm(pool, generator=g).to(torch.int32).view(seqs, 40).cuda()
    cos, sin = (t.cuda() for t in rope(g, 700, dim // 2))
    lens = torch.ones(seqs, dtype=torch.int32, device="cuda")
    y = torch.randn(seqs, q_heads + 2 * heads, dim, generator=g).cuda()

    def step(cache):
        q = cache.append(y[:, q_heads : q_heads + heads], y[:, q_heads + heads :], table, lens, q=y[:, :q_heads], cos=cos, sin=sin)
        return cache.attend(q, table, lens)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(caches[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(caches[1])
    torch.cuda.synchronize()
    for i in range(60):
        fresh = torch.randn(seqs, q_heads + 2 * heads, dim, generator=g)
        y.copy_(fresh.cuda())
        lens.copy_(torch.tensor([i + 1, 10 * i + 1, 0 if i < 30 else i - 29], dtype=torch.int32))
        want = step(caches[0])
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.default_stream())
            graph.replay()
        torch.cuda.default_stream().wait_stream(stream)
        assert torch.equal(out.view(torch.int16), want.view(torch.int16)), i
    assert torch.equal(caches[0].k_codes, caches[1].k_codes) and torch.equal(caches[0].v_scales, caches[1].v_scales)


@pytest.mark.gpu
def test_refusals_on_the_device():
    from se12_b200.kv_cache import PagedKvCache

    cache = PagedKvCache(4, 16, 2, 64)
    x = torch.randn(2, 2, 64, device="cuda")
    q = x.to(torch.bfloat16)
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    cos = torch.ones(4, 32, device="cuda")
    for call in (
        lambda: cache.append(x[:, :1], x, table, lens),
        lambda: cache.append(x, x[:1], table, lens),
        lambda: cache.append(x[:, :, :32], x, table, lens),
        lambda: cache.append(x, x, table, lens[:1]),
        lambda: cache.append(x, x, table.long(), lens),
        lambda: cache.append(x, x, table, lens.long()),
        lambda: cache.append(x, x, table, lens, cos=cos),
        lambda: cache.append(x, x, table, lens, cos=cos, sin=cos[:3]),
        lambda: cache.append(x, x, table, lens, cos=cos.repeat(1, 2), sin=cos.repeat(1, 2)),
        lambda: cache.append(x, x, table, lens, query_start=start[:2]),
        lambda: cache.append(x, x, table, lens, q_out=q),
        lambda: cache.append(x.cpu(), x, table, lens),
        lambda: cache.append(x.transpose(1, 2).contiguous().transpose(1, 2), x, table, lens),
        lambda: cache.attend(q[:, :1], table, lens),
        lambda: cache.attend(q, table, lens, query_start=start.long()),
        lambda: cache.attend(q, table.cpu(), lens),
        lambda: cache.attend(q, table, lens, out=torch.empty(2, 2, 32, dtype=torch.bfloat16, device="cuda")),
        lambda: cache.decode(lens.long()),
        lambda: PagedKvCache.from_tensors(cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales[:2]),
        lambda: PagedKvCache.from_tensors(cache.k_codes.float(), cache.v_codes.float(), cache.k_scales, cache.v_scales),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: cache.append(x.half(), x.half(), table, lens), lambda: cache.append(x, x.to(torch.bfloat16), table, lens),
                 lambda: cache.attend(x, table, lens)):
        with pytest.raises(TypeError):
            call()
    for args in (dict(window=-1), dict(softcap=-1.0), dict(softcap=math.inf), dict(scale=math.nan), dict(max_query=0),
                 dict(max_query=2)):
        with pytest.raises(RuntimeError):
            cache.attend(q, table, lens, **args)
    assert cache.append(x[:0], x[:0], table, lens, q=x[:0]).shape == (0, 2, 64)
    assert cache.attend(q[:0], table, lens).shape == (0, 2, 64)


# ------------------------------------------------------------------ expanded and overlapping views


@pytest.mark.parametrize("rows,columns,stride", [(3, 5, 0), (3, 5, 2), (1, 5, 0), (3, 1, 0), (4, 2, 7)])
def test_page_table_strides_reach_the_call(rows, columns, stride):
    """What a call is told of the table's rows is where they lie."""
    from se12_b200 import _lib
    from se12_b200.kv_cache import PagedKvCache

    cache = PagedKvCache.__new__(PagedKvCache)
    cache.device = torch.device("cpu")
    table = torch.zeros(64, dtype=torch.int32).as_strided((rows, columns), (stride, 1))
    packed = _lib.KV_BATCH.unpack(cache._batch(rows, table, torch.ones(rows, dtype=torch.int32), None))
    assert packed[4:] == (table.data_ptr(), stride, columns)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("step", [0, 1])
def test_expanded_and_overlapping_tables(n, step):
    """One table row for several sequences (candidates behind one prefix),
    rows that overlap, a rotation by the same angle everywhere: as copies."""
    g = torch.Generator().manual_seed(n)
    page, heads, q_heads, dim, seqs = 16, 2, 8, 128, 3
    length = 90
    order = torch.randperm(12, generator=g).to(torch.int32)
    view = order.cuda().as_strided((seqs, 6), (step, 1))
    table = order.as_strided((seqs, 6), (step, 1)).contiguous()
    cache, keys, values = filled(g, 12, page, heads, dim, "int8")
    lens = torch.tensor([length, length - 5, length - 9], dtype=torch.int32)
    starts = starts_of([n] * seqs)
    q = torch.randn(n * seqs, q_heads, dim, generator=g).to(torch.bfloat16)
    start = torch.tensor(starts, dtype=torch.int32).cuda()
    got = cache.attend(q.cuda(), view, lens.cuda(), query_start=start, max_query=n)
    check_attend(got, *plain_attend(q, keys, values, table, lens.tolist(), starts, dim**-0.5, 0.0, 0), length)
    # append: one sequence, a rotation table whose rows are the same
    one, plain = make_pair(12, page, heads, dim, "int8")
    cos, sin = rope(g, 1, dim // 2)
    y = torch.randn(20, q_heads + 2 * heads, dim, generator=g)
    k, v, q = y[:, :heads], y[:, heads : 2 * heads], y[:, 2 * heads :]
    want = plain.append(k, v, table[:1], [20], [0, 20], cos.expand(20, -1), sin.expand(20, -1), False, q)
    out = one.append(k.cuda(), v.cuda(), view[:1], torch.tensor([20], dtype=torch.int32).cuda(), q=q.cuda(),
                     query_start=torch.tensor([0, 20], dtype=torch.int32).cuda(), cos=cos.cuda().expand(20, -1),
                     sin=sin.cuda().expand(20, -1))
    assert torch.equal(out.cpu().view(torch.int16), want.view(torch.int16))
    same_cache(one, plain)


# ------------------------------------------------------------------ devices


class OtherDevice:
    """Stands in for torch.cuda.device while another GPU is the current one."""

    inside = False

    def __init__(self, index):
        pass

    def __enter__(self):
        OtherDevice.inside = True

    def __exit__(self, *_):
        OtherDevice.inside = False


def test_workspace_is_prepared_on_the_cache_device(monkeypatch):
    """With another GPU current, everything a call does there (asking whether
    a graph is captured, clearing the workspace, the launch) is done with the
    cache's GPU current."""
    from se12_b200 import kv_cache

    seen = []

    class Library:
        def se12_kv_attend_call_bytes(self, *_):
            return 8192

        def se12_kv_attend(self, *_):
            seen.append(("launch", OtherDevice.inside))
            return 0

    class Pool:
        def get(self, device, stream, nbytes):
            seen.append(("workspace", OtherDevice.inside))
            return torch.zeros(nbytes, dtype=torch.uint8)

    def capturing():
        seen.append(("capturing", OtherDevice.inside))
        return False

    cache = kv_cache.PagedKvCache.__new__(kv_cache.PagedKvCache)
    cache.device, cache._handle, cache._lib = torch.device("cpu"), None, Library()
    cache.pages, cache.kv_heads, cache.page_size, cache.head_dim = 2, 1, 16, 64
    monkeypatch.setattr(kv_cache, "_WORKSPACES", Pool())
    monkeypatch.setattr(torch.cuda, "device", OtherDevice)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", capturing)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: None if OtherDevice.inside else 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0)
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    cache.attend(torch.zeros(1, 2, 64, dtype=torch.bfloat16), ints([[0]]), ints([3]))
    assert sorted(seen) == [("capturing", True), ("launch", True), ("workspace", True)]


# ------------------------------------------------------------------ lengths and row starts that may be anything


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("n", [1, 3, 70])
@pytest.mark.parametrize("length", [321, 1 << 30, 2**31 - 1, -5, -(2**31)])
@pytest.mark.parametrize("window", [0, 50])
def test_attend_lengths_past_the_page_table(dim, n, length, window):
    """Rows past the page table see what it has (nothing, behind a window) and
    set the status; negative lengths are empty; the others' rows are right."""
    from se12_b200.device import device_status

    g = torch.Generator().manual_seed(n)
    page, heads, q_heads, capacity = 16, 2, 8, 320
    cache, keys, values = filled(g, 60, page, heads, dim, "int8")
    table = torch.randperm(60, generator=g).to(torch.int32).view(3, 20)
    q = torch.randn(3 * n, q_heads, dim, generator=g).to(torch.bfloat16)
    starts = starts_of([n] * 3)
    lens = [300, length, 91]
    got = cache.attend(q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                       query_start=torch.tensor(starts, dtype=torch.int32).cuda(), max_query=n, window=window)
    assert device_status() == (2 if length > capacity else 0)
    for b in (0, 2):
        rows = slice(starts[b], starts[b + 1])
        check_attend(got[rows], *plain_attend(q[rows], keys, values, table[b : b + 1], lens[b : b + 1], [0, n], dim**-0.5, 0.0, window), 300)
    for i in range(n, 2 * n):
        pos = max(length, 0) - n + (i - n)
        if pos < 0 or (window and pos - window + 1 >= capacity):
            assert not bool(got[i].any())
            continue
        seen, back = min(pos + 1, capacity), max(pos + 1 - capacity, 0)  # the window's tokens past the table are missing
        check_attend(got[i : i + 1], *plain_attend(q[i : i + 1], keys, values, table[1:2], [seen], [0, 1], dim**-0.5, 0.0,
                                                   window - back if window else 0), seen)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 70])
@pytest.mark.parametrize("starts", [[-9, 1, 2, 3], [0, 1, 2, 2**31 - 1], [-(2**31), 1, 2, 30], [0, 1, 0, 1], [3, 2, 1, 0], [9, 10, 11, 12],
                                    [2**31 - 1, -(2**31), 5, -5]])
def test_row_starts_outside_the_batch_reach_no_other_memory(n, starts):
    """Starts in units of n rows: those within the batch (3 n rows) give the
    sequences their rows, the others end at its first and last row."""
    g = torch.Generator().manual_seed(n)
    cache, _, _ = filled(g, 60, 16, 2, 128, "int8")
    table = torch.randperm(60, generator=g).to(torch.int32).view(3, 20).cuda()
    lens = torch.tensor([300, 260, 91], dtype=torch.int32).cuda()
    q = torch.randn(3 * n, 8, 128, generator=g).to(torch.bfloat16).cuda()
    ints = [s * n if abs(s) < 1000 else s for s in starts]
    out = torch.full_like(q, 7.0)
    got = cache.attend(q, table, lens, query_start=torch.tensor(ints, dtype=torch.int32).cuda(), max_query=n, out=out)
    assert bool(torch.isfinite(got).all())
    held = [min(max(s, 0), 3 * n) for s in ints]
    if held == [0, n, 2 * n, 3 * n]:
        want = cache.attend(q, table, lens, query_start=torch.tensor(held, dtype=torch.int32).cuda(), max_query=n)
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    if all(a >= b for a, b in zip(held, held[1:])):
        assert bool((got == 7.0).all())
    k = torch.randn(3 * n, 2, 128, generator=g).cuda()
    held = cache.append(k, k, table, lens, q=k, query_start=torch.tensor(ints, dtype=torch.int32).cuda())
    assert bool(torch.isfinite(held).all())
    from se12_b200.device import device_status

    device_status()  # positions past the page table may have been met


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 2, 2**20])
@pytest.mark.parametrize("n", [1, 5, 70])
def test_attend_windows_longer_than_any_sequence(window, n):
    """Such a window hides nothing, also where rows lie before the sequence."""
    g = torch.Generator().manual_seed(n)
    lens = [300, max(n - 4, 1), 2]
    table, pool = random_tables(g, lens, 16)
    cache, _, _ = filled(g, pool, 16, 2, 128, "int8")
    q = torch.randn(3 * n, 8, 128, generator=g).to(torch.bfloat16).cuda()
    args = (table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    start = torch.tensor([0, n, 2 * n, 3 * n], dtype=torch.int32).cuda()
    want = cache.attend(q, *args, query_start=start, max_query=n)
    assert torch.equal(cache.attend(q, *args, query_start=start, max_query=n, window=window), want)


def test_overlapped_kernels_load_coherently():
    """These kernels begin while the kernel before them may still write what
    they read: none of their loads is a non-coherent one."""
    from se12_b200 import _build

    for name in ("se12_kv.cu", "se12_attend.cu", "se12_attend_tile.cu", "se12_logprobs.cu", "se12_device.cuh"):
        code = [line.split("//")[0] for line in (_build.PACKAGE_DIR / "csrc" / name).read_text().splitlines()]
        assert not any("global.nc" in line or "__ldg" in line for line in code), name


# ------------------------------------------------------------------ caps of any size


def capped_case(seed, kind, page, dim, group, cap, reach, counts, lens, sign):
    """Keys along one direction, so that the raw logits of every row are
    sign * cap * reach(position) with a little noise. Tolerance as above, plus
    2^-20 |s| of sum_j p_j |v_j| for the fp32 roundings of logits past 100
    (eight of 2^-24 each, for two logits)."""
    from se12_b200.kv_cache import PagedKvCache

    g = torch.Generator().manual_seed(seed)
    heads = 2
    table, pool = random_tables(g, lens, page)
    k = torch.zeros(pool, heads, page, dim)
    for b, ln in enumerate(lens):
        for j in range(ln):
            k[table[b, j // page], :, j % page] = reach(j / max(ln - 1, 1))
    k += 0.004 * torch.randn(k.shape, generator=g)
    v = torch.randn(pool, heads, page, dim, generator=g)
    tensors = []
    for x in (k, v):
        s = torch.tensor([[least_scale(m, kind) for m in row] for row in x.abs().amax(dim=(2, 3)).tolist()])
        tensors.append((code_of(x / s[:, :, None, None], kind), s))
    (kc, ks), (vc, vs) = tensors
    cache = PagedKvCache.from_tensors(kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), kind)
    keys, values = (value_of(c, kind).double() * s.double()[:, :, None, None] for c, s in tensors)
    starts = starts_of(counts)
    q = torch.full((starts[-1], heads * group, dim), sign * cap * dim**-0.5) * (1 + 0.01 * torch.randn(starts[-1], heads * group, 1, generator=g))
    q = q.to(torch.bfloat16)
    got = cache.attend(q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                       query_start=torch.tensor(starts, dtype=torch.int32).cuda(), max_query=max(counts), softcap=cap)
    want, size, biggest = plain_attend(q, keys, values, table, lens, starts, dim**-0.5, cap, 0)
    tol = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=1e-300))) - 8) + (2.0**-10 + 2.0**-20 * cap) * size + (
        2.0**-24 * max(lens) * biggest)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).nan_to_num(nan=math.inf).max()):.2f} of the tolerance"


# Where the logits lie, as a share of the cap, from the first position to the last.
REACH = {
    "rising": lambda t: 0.5 + 0.2 * t,
    "falling": lambda t: 0.7 - 0.2 * t,
    "level": lambda t: 0.6 + 0.001 * (t * 7919 % 1),
}


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [5.0, 30.0, 80.0, 120.0, 200.0, 1000.0])
@pytest.mark.parametrize("reach", sorted(REACH))
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dim,kind", [(128, "int8"), (256, "e4m3")])
@pytest.mark.parametrize("rows", ["few", "many"])
def test_attend_caps_of_any_size(cap, reach, sign, dim, kind, rows):
    """All of a row's logits near the cap's bend, on either side of zero; rows
    that see one token, a few, and many."""
    counts = [1, 1, 2] if rows == "few" else [40, 70, 1]
    capped_case(int(cap * 10), kind, 16, dim, 4, cap, REACH[reach], counts, [40, 333, 129], sign)


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [0.5, 1.0, 2.0, 5.0, 20.0, 50.0, 100.0])
@pytest.mark.parametrize("deep", [1.0, 1.3, 1.6, 3.0])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dim,kind", [(128, "int8"), (256, "e4m3")])
@pytest.mark.parametrize("rows", ["few", "many"])
def test_attend_logits_on_both_sides_of_a_cap(cap, deep, sign, dim, kind, rows):
    """Raw logits from 0.4 of the cap down to `deep` times it below zero (and
    the other way round): with a small cap the deep ones still weigh."""
    counts = [1, 1, 2] if rows == "few" else [40, 70, 1]
    capped_case(int(cap * 10), kind, 16, dim, 4, cap, lambda t: 0.4 - (0.4 + deep) * (t * 104729 % 1), counts, [40, 333, 129], sign)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("spread,q_scale", [(40.0, 2.0**-41), (18.0, 2.0**-15), (6.0, 0.1)])
def test_attend_tiles_of_very_different_scales(kind, dim, softcap, spread, q_scale):
    """Rows of many queries over blocks whose scales are 2^(+-spread): tiles
    where rows raise their references and then turn out to be unusual."""
    attend_case(int(spread), kind, 16, 2, 8, dim, [700, 60], [40, 50], softcap=softcap, spread=spread, q_scale=q_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("n,q_heads", [(1, 8), (3, 8), (70, 8), (140, 2)])
@pytest.mark.parametrize("what,bad", [("k_scales", math.nan), ("k_scales", 0.0), ("v_scales", math.nan), ("v_scales", math.inf),
                                      ("v_scales", 0.0)])
def test_attend_blocks_outside_the_window_may_hold_anything(dim, n, q_heads, what, bad):
    """A block that is not finite reaches the rows that see it, and no row
    whose window ends above it; a scale of zero makes no row NaN."""
    g = torch.Generator().manual_seed(dim + n)
    length, window, page = 400, 100, 16
    table, pool = random_tables(g, [length], page)
    cache, _, _ = filled(g, pool, page, 2, dim, "int8")
    q = torch.randn(n, q_heads, dim, generator=g).to(torch.bfloat16).cuda()
    args = (table.cuda(), torch.tensor([length], dtype=torch.int32).cuda())
    start = torch.tensor([0, n], dtype=torch.int32).cuda()
    want = cache.attend(q, *args, query_start=start, window=window)
    for block in ((length - n - window + 1) // page, (length - n - window + 1) // page + 2):
        scales = getattr(cache, what)
        kept = scales.clone()
        scales[int(table[0, block])] = bad
        got = cache.attend(q, *args, query_start=start, window=window)
        scales.copy_(kept)
        last = block * page + page - 1  # the block's last position
        for i in range(n):
            pos = length - n + i
            if pos - last >= window:  # the block lies below this row's window
                # (only the order of the sums may differ: the unusual tile's weights are summed apart)
                assert torch.allclose(got[i].float(), want[i].float(), rtol=2.0**-6, atol=2.0**-8), (block, i)
            else:
                assert bool((torch.isfinite(got[i]) == (bad == 0.0)).all()), (block, i)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("n", [1, 3, 8, 70])
@pytest.mark.parametrize("length,window", [(400, 100), (777, 513), (130, 1), (97, 97)])
def test_attend_pages_given_back_below_the_window(dim, n, length, window):
    """Page table entries below the first position a batch's rows see are
    not read: no status, the same output."""
    from se12_b200.device import device_status

    g = torch.Generator().manual_seed(length)
    page = 16
    lens, counts = [length, 45, length - 7], [n, 1, n]
    table, pool = random_tables(g, lens, page)
    cache, _, _ = filled(g, pool, page, 2, dim, "e4m3")
    q = torch.randn(sum(counts), 8, dim, generator=g).to(torch.bfloat16).cuda()
    start = torch.tensor(starts_of(counts), dtype=torch.int32).cuda()
    dev_lens = torch.tensor(lens, dtype=torch.int32).cuda()
    want = cache.attend(q, table.cuda(), dev_lens, query_start=start, max_query=n, window=window, softcap=20.0)
    for b in range(3):
        first = max(lens[b] - counts[b] - window + 1, 0)
        table[b, : first // page] = -1
    got = cache.attend(q, table.cuda(), dev_lens, query_start=start, max_query=n, window=window, softcap=20.0)
    assert device_status() == 0
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e3, 1e4, 1e6, 1e9])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("n", [1, 40])
def test_attend_caps_far_above_the_logits(cap, dim, n):
    """A cap that hardly bends the logits costs them no precision."""
    attend_case(dim + n, "int8", 16, 2, 8, dim, [300, 41], [n, n], softcap=cap, q_scale=2.0, max_query=n)


# ------------------------------------------------------------------ rotation tables


@pytest.mark.gpu
@pytest.mark.parametrize("dim,rotary,interleaved", [(128, 128, False), (64, 32, True)])
@pytest.mark.parametrize("rope_rows", [1, 12, 16, 17])
def test_append_past_the_rotation_table_stores_neither_half(dim, rotary, interleaved, rope_rows):
    """Tokens the table reaches are stored, keys and values; the others are
    not, neither half, and set the status."""
    from se12_b200.device import device_status

    g = torch.Generator().manual_seed(dim)
    n, page, heads, q_heads = 20, 16, 2, 4
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    cos, sin = rope(g, rope_rows, rotary // 2)
    y = torch.randn(n, q_heads + 2 * heads, dim, generator=g)
    q, k, v = y[:, :q_heads], y[:, q_heads : q_heads + heads], y[:, q_heads + heads :]
    reached = min(n, rope_rows)
    prompt, plain = make_pair(3, page, heads, dim, "int8")
    want = torch.zeros(n, q_heads, dim, dtype=torch.bfloat16)
    want[:reached] = plain.append(k[:reached], v[:reached], table, [reached], [0, reached], cos, sin, interleaved, q[:reached])
    got = prompt.append(k.cuda(), v.cuda(), table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), q=q.cuda(), cos=cos.cuda(),
                        sin=sin.cuda(), query_start=torch.tensor([0, n], dtype=torch.int32).cuda(), interleaved=interleaved)
    assert device_status() == 2
    assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
    same_cache(prompt, plain)
    step, plain = make_pair(3, page, heads, dim, "int8")  # one token at a time
    for i in range(n):
        got = step.append(k[i : i + 1].cuda(), v[i : i + 1].cuda(), table.cuda(), torch.tensor([i + 1], dtype=torch.int32).cuda(),
                          q=q[i : i + 1].cuda(), cos=cos.cuda(), sin=sin.cuda(), interleaved=interleaved)
        assert device_status() == (2 if i >= rope_rows else 0)
        if i < rope_rows:
            plain.append(k[i : i + 1], v[i : i + 1], table, [i + 1], [0, 1], cos, sin, interleaved)
        assert torch.equal(got.cpu()[0].view(torch.int16), want[i].view(torch.int16))
    same_cache(step, plain)


# ------------------------------------------------------------------ long prompts


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype,page,heads,q_heads,dim,rotary,interleaved", [
    ("int8", torch.float32, 32, 6, 6, 128, 128, False),    # heads that do not divide by the heads of a CTA
    ("e4m3", torch.bfloat16, 256, 5, 5, 256, 256, False),  # more tokens per page than stay in registers
    ("int8", torch.bfloat16, 16, 5, 10, 96, 32, False),    # scalar lanes
    ("e4m3", torch.float32, 128, 1, 2, 80, 80, True),
    ("int8", torch.float32, 64, 9, 9, 128, 0, False),
])
def test_append_thousands_of_tokens(kind, dtype, page, heads, q_heads, dim, rotary, interleaved):
    """Calls of more than 2048 tokens, on empty sequences and behind prefixes."""
    g = torch.Generator().manual_seed(page)
    steps = [[1900, 1, 0, 180], [700, 1200, 300, 7]]
    counts = [sum(s[b] for s in steps) for b in range(4)]
    table, pool = random_tables(g, counts, page)
    cache, plain = make_pair(pool, page, heads, dim, kind)
    cos, sin = rope(g, max(counts), rotary // 2) if rotary else (None, None)
    lens = [0] * 4
    for step, new in enumerate(steps):
        lens = [a + b for a, b in zip(lens, new)]
        starts = starts_of(new)
        y = (torch.randn(starts[-1], q_heads + 2 * heads, dim, generator=g) * 3.0**step).to(dtype)
        q, k, v = y[:, :q_heads], y[:, q_heads : q_heads + heads], y[:, q_heads + heads :]
        want = plain.append(k, v, table, lens, starts, cos, sin, interleaved, q)
        d = y.cuda()
        got = cache.append(d[:, q_heads : q_heads + heads], d[:, q_heads + heads :], table.cuda(),
                           torch.tensor(lens, dtype=torch.int32).cuda(), q=d[:, :q_heads],
                           query_start=torch.tensor(starts, dtype=torch.int32).cuda(), cos=None if cos is None else cos.cuda(),
                           sin=None if sin is None else sin.cuda(), interleaved=interleaved)
        assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
        same_cache(cache, plain)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [256, 257, 4100])
@pytest.mark.parametrize("kind,page,heads,dim", [("int8", 64, 9, 128), ("e4m3", 16, 3, 256), ("int8", 128, 5, 64)])
def test_append_heads_per_block_of_threads(tokens, kind, page, heads, dim):
    """One, two or four heads per CTA, by the tokens and the page; heads that
    do not divide by them."""
    g = torch.Generator().manual_seed(tokens)
    table, pool = random_tables(g, [tokens + 5], page)
    cache, plain = make_pair(pool, page, heads, dim, kind)
    cos, sin = rope(g, tokens + 5, dim // 2)
    for new, length in ((5, 5), (tokens, tokens + 5)):
        y = torch.randn(new, 2 * heads, dim, generator=g)
        plain.append(y[:, :heads], y[:, heads:], table, [length], [0, new], cos, sin)
        d = y.cuda()
        cache.append(d[:, :heads], d[:, heads:], table.cuda(), torch.tensor([length], dtype=torch.int32).cuda(),
                     query_start=torch.tensor([0, new], dtype=torch.int32).cuda(), cos=cos.cuda(), sin=sin.cuda())
        same_cache(cache, plain)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_attend_under_a_vanishing_cap_is_the_mean(n):
    """All weights are equal, a zero query's among them."""
    g = torch.Generator().manual_seed(n)
    table, pool = random_tables(g, [60], 16)
    cache, keys, values = filled(g, pool, 16, 2, 128, "int8")
    q = torch.randn(n, 8, 128, generator=g).to(torch.bfloat16)
    q[0, 1] = 0.0
    start = torch.tensor([0, n], dtype=torch.int32).cuda()
    got = cache.attend(q.cuda(), table.cuda(), torch.tensor([60], dtype=torch.int32).cuda(), query_start=start, softcap=1e-40)
    check_attend(got, *plain_attend(q, keys, values, table, [60], [0, n], 0.0, 0.0, 0), 60)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 20])
def test_attend_as_many_sequences_as_there_may_be(n):
    from se12_b200.kv_cache import MAX_SEQS

    g = torch.Generator().manual_seed(n)
    lens = [n + (i * 37) % 50 for i in range(MAX_SEQS)]
    table, pool = random_tables(g, lens, 16)
    cache, _, _ = filled(g, pool, 16, 1, 64, "int8")
    q = torch.randn(n * MAX_SEQS, 2, 64, generator=g).to(torch.bfloat16).cuda()
    got = cache.attend(q, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), max_query=n,
                       query_start=torch.tensor(starts_of([n] * MAX_SEQS), dtype=torch.int32).cuda())
    some = list(range(0, MAX_SEQS, 97)) + [MAX_SEQS - 1]
    rows = torch.cat([torch.arange(b * n, b * n + n) for b in some]).cuda()
    check_on_gpu(cache, q[rows], table[some].cuda(), [lens[b] for b in some], [n] * len(some), got[rows], 0.0, 0)


@pytest.mark.gpu
def test_windows_and_row_counts_past_32_bits():
    """A window of any length is a window; a row count past the batch's is
    refused as any other is."""
    from se12_b200.kv_cache import PagedKvCache

    cache = PagedKvCache(4, 16, 2, 64)
    x = torch.randn(2, 2, 64, device="cuda")
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    q = cache.append(x, x, table, lens, q=x)
    want = cache.attend(q, table, lens)
    for window in (2**31 - 1, 2**31, 2**63):
        assert torch.equal(cache.attend(q, table, lens, window=window), want)
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError):
        cache.attend(q, table, lens, query_start=start, max_query=2**40)
