"""The paged 4-bit key/value cache: the stored codes, scales and offsets bit
for bit against elementary fp32 operations (their order is the kernel's:
subtract, multiply, round), the values they stand for against the formula."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch
from test_kv_cache import random_tables, rope, rotate, starts_of
from test_kv_norms import normalise

GROUP = 64


# ------------------------------------------------------------------ plain implementation (CPU)


def quantise(x, values):
    """x [..., dim] fp32 as (codes, scales, offsets, E): uint8 [..., dim], fp16 [..., groups] twice, fp32 [...]."""
    e = torch.zeros(x.shape[:-1])
    bad = ~torch.isfinite(x).all(-1)
    if values:
        amax = x.abs().amax(-1)
        bad |= ~(amax < 2.0**34)
        x = torch.where(bad[..., None], torch.zeros_like(x), x)
        amax = x.abs().amax(-1)
        e = torch.where(amax > 0, torch.frexp(amax).exponent.float() - 4, torch.full_like(e, -30)).clamp(min=-30)
        x = x * torch.exp2(-e)[..., None]
        e = torch.where(bad, torch.full_like(e, math.nan), e)
    x = x.unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(-1), x.amax(-1)
    scale = ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32)).half()
    offset = (lo + 8 * scale.float()).half()
    inverse = torch.where(scale > 0, 1 / scale.float(), torch.zeros_like(lo))
    u = torch.round((x - offset.float()[..., None]) * inverse[..., None]) + 8
    u = u.clamp(0, 15).nan_to_num(0).to(torch.uint8).flatten(-2)
    if not values:
        lost = ~(torch.maximum(lo.abs(), hi.abs()) <= 65000.0)
        scale, offset = (torch.where(lost, torch.full_like(t, math.nan), t) for t in (scale, offset))
    return u, scale, offset, e


def line(u, scale, offset):
    """What codes stand for, in 64 bits."""
    x = u.double().unflatten(-1, (-1, GROUP)) - 8
    return (x * scale.double()[..., None] + offset.double()[..., None]).flatten(-2)


class Plain4:
    """The same cache in elementary CPU operations, one token of a head at a time."""

    def __init__(self, pages, page_size, heads, dim):
        self.page_size, self.heads, self.dim, self.groups = page_size, heads, dim, dim // GROUP
        shape = (pages, heads, page_size)
        self.u = {w: torch.zeros(*shape, dim, dtype=torch.uint8) for w in "kv"}
        self.scale = {w: torch.zeros(*shape, self.groups, dtype=torch.float16) for w in "kv"}
        self.offset = {w: torch.zeros(*shape, self.groups, dtype=torch.float16) for w in "kv"}
        self.e = torch.zeros(shape)

    def append(self, k, v, table, lens, starts, cos=None, sin=None, interleaved=False, q=None, q_norm=None, k_norm=None, eps=0.0):
        out = None if q is None else torch.zeros(q.shape, dtype=torch.bfloat16)
        for b, ln in enumerate(lens):
            n = starts[b + 1] - starts[b]
            for i in range(n):
                pos, t = ln - n + i, starts[b] + i
                if pos < 0:
                    continue
                turn = (lambda x: x) if cos is None else (lambda x, p=pos: rotate(x, cos[p], sin[p], interleaved))
                if q is not None:
                    out[t] = turn(normalise(q[t], q_norm, eps)).to(torch.bfloat16)
                page, slot = int(table[b, pos // self.page_size]), pos % self.page_size
                self.put("k", page, slot, turn(normalise(k[t], k_norm, eps)))
                self.put("v", page, slot, v[t].float())
        return out

    def put(self, w, page, slot, x):
        u, scale, offset, e = quantise(x, w == "v")
        self.u[w][page, :, slot], self.scale[w][page, :, slot], self.offset[w][page, :, slot] = u, scale, offset
        if w == "v":
            self.e[page, :, slot] = e

    def values(self, w):
        x = line(self.u[w], self.scale[w], self.offset[w])
        return x * torch.exp2(self.e.double())[..., None] if w == "v" else x

    def tensors(self):
        """The four tensors of a PagedKvCache."""
        def packed(u):
            words = u.unflatten(-1, (self.groups, 8, 8)).transpose(-3, -2)
            return (words[..., 0::2] | (words[..., 1::2] << 4)).flatten(-3).contiguous()

        k_scales = torch.stack((self.scale["k"], self.offset["k"]), -1)
        both = torch.cat((self.scale["v"], self.offset["v"]), -1).unflatten(2, (-1, 8, 2)).transpose(-1, -2).flatten(-3)
        v_scales = torch.cat((both, self.e.half().unflatten(2, (-1, 16))), -1)
        return packed(self.u["k"]), packed(self.u["v"]), k_scales, v_scales


def make_pair(pages, page, heads, dim):
    from se12_b200.kv_cache import PagedKvCache

    return PagedKvCache(pages, page, heads, dim, "int4"), Plain4(pages, page, heads, dim)


def same_bits(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num().view(torch.int16), b.nan_to_num().view(torch.int16))


def same_cache(cache, plain):
    k_codes, v_codes, k_scales, v_scales = plain.tensors()
    assert torch.equal(cache.k_codes.cpu(), k_codes) and same_bits(cache.k_scales.cpu(), k_scales), "keys"
    assert torch.equal(cache.v_codes.cpu(), v_codes) and same_bits(cache.v_scales.cpu(), v_scales), "values"


# ------------------------------------------------------------------ CPU


def test_the_line_holds_its_group():
    """Half a step, of a step that is rounded to FP16 (2^-11 of it at the ends,
    7.5 steps away), and the offset's rounding."""
    g = torch.Generator().manual_seed(4)
    for values in (False, True):
        for size in (1e-3, 1.0, 300.0):
            x = torch.randn(200, 128, generator=g) * size * (1 + 9 * torch.rand(128, generator=g)) + size * torch.randn(128, generator=g)
            u, scale, offset, e = quantise(x, values)
            y = line(u, scale, offset) * torch.exp2(e.double())[:, None]
            group = x.double().unflatten(-1, (-1, GROUP))
            step = (group.amax(-1) - group.amin(-1)) / 15
            slack = step * (0.5 + 8 * 2.0**-11) + 2.0**-11 * group.abs().amax(-1) + 2.0**-24
            assert bool(((y - x.double()).abs().unflatten(-1, (-1, GROUP)) <= slack[..., None]).all())


@pytest.mark.parametrize("args", [dict(head_dim=96), dict(head_dim=32), dict(head_dim=512), dict(head_dim=80), dict(page_size=8),
                                  dict(kv_heads=0)])
def test_cache_refuses_bad_shapes(args):
    from se12_b200.kv_cache import PagedKvCache

    with pytest.raises(ValueError):
        PagedKvCache(**{**dict(pages=4, page_size=16, kv_heads=2, head_dim=64, kind="int4"), **args})


def test_cache_refuses_tensors_of_other_shapes():
    from se12_b200.kv_cache import PagedKvCache

    good = list(Plain4(3, 16, 2, 128).tensors())
    for i, bad in ((0, good[0].float()), (0, good[0][..., :48]), (1, good[1][:2]), (2, good[2].float()), (2, good[2][..., 0]),
                   (3, good[3][..., :-1]), (3, good[3].transpose(0, 1).contiguous()), (2, good[2].transpose(0, 1))):
        tensors = list(good)
        tensors[i] = bad
        with pytest.raises(ValueError):
            PagedKvCache.from_tensors(*tensors, kind="int4")


def test_abi_refuses_bad_arguments_without_a_device():
    from se12_b200 import _build, _lib

    _build.build()
    lib = _lib.load()
    handle = ctypes.c_void_p()
    good = dict(pages=4, page_size=16, kv_heads=2, head_dim=64, kind=4, k_codes=256, v_codes=256, k_scales=256, v_scales=256)

    def create(**changed):
        return lib.se12_kv_cache_create(ctypes.byref(_lib.Se12KvPagesStruct(**{**good, **changed})), ctypes.byref(handle))

    assert create(head_dim=96) == 1 and b"64, 128 or 256" in lib.se12_last_error()
    assert create(kind=3) == 2 and create(k_scales=264) == 3 and create(v_scales=260) == 3 and create(v_scales=None) == 1


# ------------------------------------------------------------------ append and reading back


APPEND = [
    # dtype, page, heads, q_heads, dim, rotary (0: none), interleaved, norm weights' type (None: no norms)
    (torch.float32, 16, 2, 4, 256, 256, False, torch.float32),
    (torch.float32, 32, 3, 7, 128, 128, False, None),
    (torch.bfloat16, 64, 3, 3, 128, 128, False, torch.bfloat16),
    (torch.bfloat16, 16, 1, 8, 256, 64, False, torch.float32),   # part of the row, in halves
    (torch.float32, 16, 2, 5, 64, 64, False, torch.bfloat16),
    (torch.float32, 16, 5, 2, 64, 32, False, None),
    (torch.bfloat16, 128, 2, 2, 128, 128, True, torch.float32),  # neighbouring pairs
    (torch.float32, 16, 2, 2, 256, 96, True, None),
    (torch.float32, 16, 1, 2, 128, 12, False, torch.float32),    # halves that are no vectors
    (torch.bfloat16, 16, 1, 2, 64, 2, True, None),
    (torch.float32, 256, 2, 2, 128, 0, False, torch.float32),    # no rotation
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,page,heads,q_heads,dim,rotary,interleaved,w_dtype", APPEND)
@pytest.mark.parametrize("steps", [
    [[1, 1, 1, 1, 1]] * 3,                                    # next tokens
    [[40, 1, 0, 17, 3], [1, 16, 33, 0, 2], [5, 5, 5, 5, 5]],  # prompts, continued
    [[300, 0, 0, 0, 1], [1, 1, 1, 1, 1]],
])
def test_append_stores_the_same_codes(dtype, page, heads, q_heads, dim, rotary, interleaved, w_dtype, steps):
    g = torch.Generator().manual_seed(dim + page + rotary)
    counts = [sum(s[b] for s in steps) for b in range(5)]
    table, pool = random_tables(g, counts, page)
    cache, plain = make_pair(pool, page, heads, dim)
    cos, sin = rope(g, max(counts), rotary // 2) if rotary else (None, None)
    q_norm, k_norm = ((1 + 0.5 * torch.randn(dim, generator=g)).to(w_dtype) if w_dtype else None for _ in "qk")
    lens = [0] * 5
    for step, new in enumerate(steps):
        lens = [a + b for a, b in zip(lens, new)]
        starts = starts_of(new)
        y = (torch.randn(starts[-1], q_heads + 2 * heads, dim, generator=g) * 3.0**step * (1 + 9 * torch.rand(dim, generator=g))).to(dtype)
        q, k, v = y[:, :q_heads], y[:, q_heads : q_heads + heads], y[:, q_heads + heads :]
        want = plain.append(k, v, table, lens, starts, cos, sin, interleaved, q, q_norm, k_norm, 1e-6)
        d = y.cuda()
        start = None if all(n == 1 for n in new) else torch.tensor(starts, dtype=torch.int32).cuda()
        got = cache.append(d[:, q_heads : q_heads + heads], d[:, q_heads + heads :], table.cuda(),
                           torch.tensor(lens, dtype=torch.int32).cuda(), q=d[:, :q_heads], query_start=start,
                           cos=None if cos is None else cos.cuda(), sin=None if sin is None else sin.cuda(), interleaved=interleaved,
                           q_norm=None if q_norm is None else q_norm.cuda(), k_norm=None if k_norm is None else k_norm.cuda())
        assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
        same_cache(cache, plain)
    keys, values = cache.decode()
    # rounded to fp32 once and then to BF16
    for got, want in ((keys, plain.values("k")), (values, plain.values("v"))):
        assert torch.equal(got.cpu().view(torch.int16), want.float().to(torch.bfloat16).view(torch.int16))
    some = torch.tensor([int(table[0, 0]), 0, int(table[0, 0])], dtype=torch.int32)
    again = cache.decode(some.cuda())
    assert torch.equal(again[0], keys[some.long().cuda()]) and torch.equal(again[1], values[some.long().cuda()])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens_each", [1, 3])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_append_takes_any_strides(tokens_each, dim):
    """Rows at odd offsets, an output with its own strides, a rotation table cut
    from a wider one, one query row for all heads: the same codes."""
    g = torch.Generator().manual_seed(5)
    heads, q_heads, seqs, page = 2, 4, 3, 16
    lens = [20, 7, 33]
    table, pool = random_tables(g, lens, page)
    cache, plain = make_pair(pool, page, heads, dim)
    cos, sin = rope(g, 40, dim // 2)
    starts = starts_of([tokens_each] * seqs)
    t = starts[-1]
    start = None if tokens_each == 1 else torch.tensor(starts, dtype=torch.int32).cuda()

    def odd(x):  # the same values, one element past an aligned address, head stride dim + 3
        wide = torch.zeros(t, x.shape[1], dim + 3)
        wide[:, :, 1 : dim + 1] = x
        return wide.cuda()[:, :, 1 : dim + 1]

    q = torch.randn(t, 1, dim, generator=g).expand(t, q_heads, dim)
    k, v = torch.randn(t, heads, dim, generator=g), torch.randn(t, heads, dim, generator=g)
    norm = torch.randn(dim + 1, generator=g)
    want = plain.append(k, v, table, lens, starts, cos, sin, False, q, norm[1:], None, 1e-6)
    out = torch.full((t, q_heads, dim + 5), 7.0, dtype=torch.bfloat16, device="cuda")
    wide = torch.zeros(2, 40, dim // 2 + 1)
    wide[0, :, 1:], wide[1, :, 1:] = cos, sin
    wide = wide.cuda()
    got = cache.append(odd(k), odd(v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                       q=q[:, :1].cuda().expand(t, q_heads, dim), query_start=start, cos=wide[0][:, 1:], sin=wide[1][:, 1:],
                       q_out=out[:, :, 2 : dim + 2], q_norm=norm.cuda()[1:])
    assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
    assert bool((out[:, :, :2] == 7).all()) and bool((out[:, :, dim + 2 :] == 7).all())
    same_cache(cache, plain)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_that_do_not_fit(dim):
    """A key group with a value that is not finite or beyond FP16 is NaN, a token
    with such values is NaN as a whole through E alone, and nobody else is."""
    cache, plain = make_pair(3, 16, 1, dim)
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(14, 1, dim, generator=g), torch.randn(14, 1, dim, generator=g)
    for i, x in enumerate((math.inf, -math.inf, math.nan, 65001.0, -1e30)):
        k[i, 0, (7 * i) % dim] = x
    k[5] = 64999.0
    for i, x in enumerate((math.inf, -math.inf, math.nan, 2.0**34, -1e30)):
        v[6 + i, 0, (9 * i) % dim] = x
    v[11, 0, 3] = 2.0**34 * 0.999
    v[12], k[12] = 0.0, 0.0
    v[13] *= 1e-12
    table = torch.tensor([[2]], dtype=torch.int32)
    starts = torch.tensor([0, 14], dtype=torch.int32).cuda()
    plain.append(k, v, table, [14], [0, 14])
    cache.append(k.cuda(), v.cuda(), table.cuda(), torch.tensor([14], dtype=torch.int32).cuda(), query_start=starts)
    same_cache(cache, plain)
    keys, values = cache.decode()
    assert bool(torch.isfinite(keys[2, 0, 5:14]).all()) and bool(torch.isnan(keys[2, 0, :5]).any(-1).all())
    assert bool(torch.isnan(values[2, 0, 6:11]).all())
    assert bool(torch.isfinite(values[2, 0, :6]).all()) and bool(torch.isfinite(values[2, 0, 11:]).all())
    assert bool((values[2, 0, 12] == 0).all()) and bool((keys[2, 0, 12] == 0).all())
    assert bool(torch.isfinite(cache.v_scales[..., : dim // 2]).all())


@pytest.mark.gpu
def test_append_stays_within_its_tokens_and_pages():
    """Padding rows, a page id out of range, positions past the page table and
    past the rotation table store nothing (and set the status); other pages and
    slots keep their bytes; queries without a position are zeros."""
    from se12_b200.device import device_status

    g = torch.Generator().manual_seed(8)
    page, dim, heads = 16, 128, 2
    cache, plain = make_pair(6, page, heads, dim)
    for t in (cache.k_codes, cache.v_codes):
        t.random_(0, 255)
    for t in (cache.k_scales, cache.v_scales):
        t.uniform_(-1, 1)
    before = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)]
    cos, sin = rope(g, 30, 64)
    x = torch.randn(6, heads, dim, generator=g).cuda()
    table = torch.tensor([[0, 1], [2, 9], [3, -4], [4, 5], [1, 1], [5, 5]], dtype=torch.int32).cuda()
    lens = torch.tensor([0, 17, 32, 31, 33, -7], dtype=torch.int32).cuda()  # padding, bad pages, past the rotation, past the table
    q = cache.append(x, x, table, lens, q=x, cos=cos.cuda(), sin=sin.cuda())
    assert device_status(clear=True) == 2
    for t, b in zip((cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales), before):
        assert torch.equal(t, b)
    zero = [bool((q[i] == 0).all()) for i in range(6)]
    assert zero[0] and zero[3] and zero[4] and zero[5] and not zero[1]
    # three tokens into slots 14, 15 of one page and 0 of the next
    starts = torch.tensor([0, 3], dtype=torch.int32).cuda()
    cache.append(x[:3], x[:3], table[:1], torch.tensor([17], dtype=torch.int32).cuda(), query_start=starts)
    changed = {(int(p), int(s)) for p, _, s, _ in (cache.k_codes != before[0]).nonzero().cpu()}
    assert changed == {(0, 14), (0, 15), (1, 0)}
    assert {(int(p), int(s)) for p, _, s, _, _ in (cache.k_scales != before[2]).nonzero().cpu()} == changed


@pytest.mark.gpu
def test_decode_of_pages_that_are_not_there_is_zero():
    from se12_b200.device import device_status

    cache, _ = make_pair(3, 16, 2, 64)
    cache.k_scales.fill_(1.0)
    keys, values = cache.decode(torch.tensor([1, 3, -1], dtype=torch.int32).cuda())
    assert device_status(clear=True) == 2
    assert bool((keys[0] != 0).any()) and bool((keys[1:] == 0).all()) and bool((values[1:] == 0).all())
