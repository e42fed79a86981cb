"""Attention over 4-bit pages whose tokens' values differ much in size: each row
against its own 64-bit sum, with a tolerance of what that row sees alone.

Tolerance, elementwise, p the weights of a row and v = s + o its values (codes
times scale, and offsets). BF16's rounding of the output, half a unit in its last
place. Weights are rounded to FP16 and for s once more times the scale: 2^-10 of
p @ |s|, 2^-11 of p @ |o|; fp32 errors of logits, exponential and sums: 2^-12 of
p @ |v|. FP16 ends at 2^-24 of a row's reference, which is the largest p 2^E
that the row sees or less: with |v| <= S 2^E a token is off by 2^-25 (S + 8) of
that at most (weight; 8 codes times the rounded product of weight and scale).
Few rows: what mma.sync cuts off a sum of 16 products of codes, 2^-16 of a step
of the largest, 2^-14 of p @ scale in all.
Many rows: values are rounded to FP16 (2^-11 of p @ |v|), and those of a cell of
16 tokens within 2^6 of each other stand beside the largest, seen or not: up to
2^6 times the reference, and scale, offset and value off by 2^-25 of it. Keys are
rounded to FP16: a logit moves by 2^-11 of scale sum_d |q k|, and with it the
token's weight and the sum of all."""

from __future__ import annotations

import math

import pytest
import torch
from test_kv_cache import starts_of
from test_kv_int4 import GROUP, Plain4, quantise

SPREAD = 6  # powers of two that the tokens of a cell of 16 may differ by without a way of their own


def by_tiles(rows, dim):
    """Which kernel a call of so many query rows per KV head takes."""
    return rows > {64: 128, 128: 48, 256: 32}[dim]


class Sized:
    """Sequences whose token j has values of about 2^powers[j], and on the GPU in 64 bits what their cache holds."""

    def __init__(self, g, page, heads, dim, powers, key=None):
        from se12_b200.kv_cache import PagedKvCache

        need = [(len(p) + page - 1) // page for p in powers]
        pool = sum(need) + 1
        order = torch.randperm(pool, generator=g)
        plain = Plain4(pool, page, heads, dim)
        self.table = torch.full((len(powers), max(need)), -1, dtype=torch.int32)
        self.k, self.s, self.o, self.e, self.step = [], [], [], [], []
        at = 0
        for b, (power, n) in enumerate(zip(powers, need)):
            ids = order[at : at + n]
            at += n
            self.table[b, :n] = ids
            length = len(power)
            k = torch.randn(heads, length, dim, generator=g) if key is None else key(b, power)
            v = torch.randn(heads, length, dim, generator=g) * torch.exp2(power)[:, None]
            v *= torch.exp2(-torch.randint(0, 7, (heads, length, dim // GROUP), generator=g).float()).repeat_interleave(GROUP, -1)
            for w, x in (("k", k), ("v", v)):
                u, scale, offset, e = quantise(x, w == "v")
                for held, new in ((plain.u[w], u), (plain.scale[w], scale), (plain.offset[w], offset)) + (((plain.e, e),) if w == "v" else ()):
                    padded = torch.zeros(heads, n * page, *new.shape[2:], dtype=held.dtype)
                    padded[:, :length] = new
                    held[ids] = padded.unflatten(1, (n, page)).transpose(0, 1)
                steps = (u.double().unflatten(-1, (-1, GROUP)) - 8) * scale.double()[..., None]
                offsets = offset.double().repeat_interleave(GROUP, -1)
                if w == "k":
                    self.k.append((steps.flatten(-2) + offsets).cuda())
                else:
                    p = torch.exp2(e.double())[..., None]
                    self.s.append((steps.flatten(-2) * p).cuda())
                    self.o.append((offsets * p).cuda())
                    self.step.append((scale.double().repeat_interleave(GROUP, -1) * p).cuda())
                    self.e.append(e.double().cuda())
        self.heads, self.dim, self.page, self.plain = heads, dim, page, plain
        self.cache = PagedKvCache.from_tensors(*(t.cuda() for t in plain.tensors()), "int4")
        self.lens = [len(p) for p in powers]

    def attend(self, q, counts, **call):
        return self.cache.attend(q.cuda(), self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda(),
                                 query_start=torch.tensor(starts_of(counts), dtype=torch.int32).cuda(), max_query=max(counts), **call)

    def check(self, q, counts, got, softcap=0.0, window=0, skip=None):
        dim, group = self.dim, q.shape[1] // self.heads
        tiles, scale, starts = by_tiles(max(counts) * group, dim), dim**-0.5, starts_of(counts)
        q, got = q.cuda(), got.double()
        for b, ln in enumerate(self.lens):
            i, j = torch.arange(ln - counts[b], ln, device="cuda"), torch.arange(ln, device="cuda")
            seen = j[None, :] <= i[:, None]
            if window:
                seen &= i[:, None] - j[None, :] < window
            for h in range(self.heads):
                k, s, o, e, step = self.k[b][h], self.s[b][h], self.o[b][h], self.e[b][h], self.step[b][h]
                v, power = s + o, torch.exp2(e)
                largest = float((v.abs() / power[:, None]).max())
                for r in range(h * group, (h + 1) * group):
                    x = q[starts[b] : starts[b + 1], r].double()
                    logits = x @ k.T * scale
                    if softcap:
                        logits = softcap * torch.tanh(logits / softcap)
                    p = torch.softmax(logits.masked_fill(~seen, -math.inf), -1)
                    want, size = p @ v, p @ v.abs()
                    tol = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=1e-300))) - 8)
                    tol = tol + 2.0**-10 * (p @ s.abs()) + 2.0**-11 * (p @ o.abs()) + 2.0**-12 * size
                    reference = (p * power).amax(-1, keepdim=True) * seen.sum(-1, keepdim=True)
                    tol = tol + 2.0 ** (-25 + (SPREAD if tiles else 0)) * (largest + 8 + (10 if tiles else 0)) * reference
                    if tiles:
                        moved = torch.expm1(2.0**-11 * scale * (x.abs() @ k.abs().T))
                        moved = p * moved.masked_fill(~seen, 0)
                        tol = tol + 2.0**-11 * size + moved @ v.abs() + moved.sum(-1, keepdim=True) * size
                    else:
                        tol = tol + 2.0**-14 * (p @ step)
                    err = (got[starts[b] : starts[b + 1], r] - want).abs()
                    if skip is not None:
                        err[skip] = 0
                    assert bool((err <= tol).all()), (b, r, float((err / tol).nan_to_num(math.inf).max()))


LENS, COUNTS = [150, 161, 333], [150, 140, 130]


def sizes(pattern, g, length):
    power = torch.zeros(length)
    if pattern == "one larger token":  # the last of its 16, for the others
        power[15::48] = 26.0
    elif pattern == "any size":
        power = torch.randint(-30, 27, (length,), generator=g).float()
    elif pattern == "near each other":  # cells on both sides of SPREAD
        power = torch.cat([torch.randint(0, 4 + n % 8, (16,), generator=g).float() for n in range(length // 16 + 1)])[:length]
    elif pattern == "first of all":  # left behind by a window
        power[: length // 2 : 5] = 28.0
    return power


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("pattern", ["one larger token", "any size", "near each other", "first of all"])
@pytest.mark.parametrize("softcap,window", [(0.0, 0), (0.0, 21), (5.0, 0), (30.0, 40)])
def test_rows_by_tiles_have_their_own_size(dim, pattern, softcap, window):
    """A row that does not see a large token has its own values' precision; so
    have tokens that follow a large one, once it is outside the window."""
    g = torch.Generator().manual_seed(dim + window)
    f = Sized(g, 16 if dim == 128 else 64, 2, dim, [sizes(pattern, g, n) for n in LENS])
    q = torch.randn(sum(COUNTS), 4, dim, generator=g).to(torch.bfloat16)
    f.check(q, COUNTS, f.attend(q, COUNTS, softcap=softcap, window=window), softcap, window)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 12, 160])
@pytest.mark.parametrize("softcap", [0.0, 400.0])
def test_large_tokens_of_no_weight(dim, n, softcap):
    """Every row sees the large tokens, at logits of about -200: they count nothing."""
    g = torch.Generator().manual_seed(n)
    way = torch.randn(dim, generator=g)
    way *= dim**0.5 / way.norm()

    def key(b, power):
        away = -200 * dim**-0.5 * way
        return torch.where((power > 10)[None, :, None], away, 0.5 * torch.randn(2, len(power), dim, generator=g))

    lens, counts = [200, 333], [n, n]
    f = Sized(g, 32, 2, dim, [torch.where(torch.arange(ln) % 7 == 3, 24.0, 0.0) for ln in lens], key)
    q = (way + 0.1 * torch.randn(2 * n, 4, dim, generator=g)).to(torch.bfloat16)
    f.check(q, counts, f.attend(q, counts, softcap=softcap), softcap)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_large_tokens_in_a_long_sequence(dim):
    """Tiles of several CTAs: references of very different size are joined."""
    g = torch.Generator().manual_seed(dim)
    powers = [torch.where(torch.rand(n, generator=g) < 0.01, 25.0, 0.0) for n in (6001, 900)]
    powers[0][: 16 * 150] = -9.0
    counts = [200, 70]
    f = Sized(g, 128, 1, dim, powers)
    q = torch.randn(sum(counts), 3, dim, generator=g).to(torch.bfloat16)
    f.check(q, counts, f.attend(q, counts))
    f.check(q, counts, f.attend(q, counts, window=300), window=300)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_tokens_that_are_nan_or_zero_beside_large_ones(dim):
    """In a cell of 16 tokens of very different sizes, too, a token that is NaN
    reaches the rows that see it and no others, and one of zeros weighs."""
    g = torch.Generator().manual_seed(dim)
    n = 140
    f = Sized(g, 16, 1, dim, [sizes("one larger token", g, n)])
    for t in (*f.plain.scale.values(), *f.plain.offset.values()):
        assert bool(t.isfinite().all())
    zero = 5
    page, slot = int(f.table[0, 0]), zero
    f.plain.u["v"][page, 0, slot], f.plain.scale["v"][page, 0, slot], f.plain.offset["v"][page, 0, slot] = 8, 0, 0
    f.plain.e[page, 0, slot] = -30
    f.s[0][0, zero], f.o[0][0, zero], f.step[0][0, zero], f.e[0][0, zero] = 0, 0, 0, -30
    f.cache = type(f.cache).from_tensors(*(t.cuda() for t in f.plain.tensors()), "int4")
    q = torch.randn(n, 2, dim, generator=g).to(torch.bfloat16)
    f.check(q, [n], f.attend(q, [n]))
    lost, window = 20, 30
    page, slot = int(f.table[0, 1]), lost - 16
    f.plain.u["v"][page, 0, slot], f.plain.scale["v"][page, 0, slot], f.plain.offset["v"][page, 0, slot] = 8, 0, 0
    f.plain.e[page, 0, slot] = math.nan
    f.cache = type(f.cache).from_tensors(*(t.cuda() for t in f.plain.tensors()), "int4")
    got = f.attend(q, [n], window=window)
    sees = torch.zeros(n, dtype=torch.bool)
    sees[lost : lost + window] = True
    assert bool(got[sees.cuda()].isnan().all()) and not bool(got[~sees.cuda()].isnan().any())
    f.check(q, [n], got, window=window, skip=sees.cuda())


# Rows per KV head that the kernel of few rows takes, past its first tile of 16: no key is rounded there.
FEW = [(64, 8, 3), (64, 4, 17), (64, 8, 16), (64, 1, 100), (128, 8, 3), (128, 1, 33), (128, 8, 6), (128, 12, 4), (256, 8, 3),
       (256, 1, 32), (256, 4, 8), (256, 17, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,group,n", FEW)
@pytest.mark.parametrize("pattern", ["all alike", "any size"])
@pytest.mark.parametrize("softcap,window", [(0.0, 0), (5.0, 33)])
def test_several_tiles_of_few_rows(dim, group, n, pattern, softcap, window):
    assert not by_tiles(n * group, dim) and n * group > 16
    g = torch.Generator().manual_seed(dim + n)
    counts = [n, max(n - 1, 1), 1, n]
    f = Sized(g, 16 if dim == 256 else 64, 2, dim, [sizes(pattern, g, max(length, n)) for length in (700, 61, 17, n)])
    q = (2 * torch.randn(sum(counts), 2 * group, dim, generator=g)).to(torch.bfloat16)
    f.check(q, counts, f.attend(q, counts, softcap=softcap, window=window), softcap, window)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 70])
def test_the_largest_scales_and_offsets(dim, n):
    """Of tensors that append did not write: scales up to 128, offsets beside which
    the codes stay in FP16's range, and weights up to 2^8 of the reference."""
    g = torch.Generator().manual_seed(dim + n)
    length = 300
    f = Sized(g, 16, 1, dim, [torch.zeros(length)])
    ids = f.table[0].long()
    plain = f.plain
    plain.scale["v"][ids] = (127.9 * torch.rand(plain.scale["v"][ids].shape, generator=g) ** 4).half()
    plain.offset["v"][ids] = (30000 * (2 * torch.rand(plain.offset["v"][ids].shape, generator=g) - 1)).half()
    plain.e[ids] = -12.0
    # the first tokens' logits are 5 below the rest: weights pass the reference without raising it
    plain.u["k"][ids[0]], plain.scale["k"][ids[0]] = 8, 0
    plain.offset["k"][ids[0]] = -5 * dim**-0.5
    plain.u["k"][ids[1:]], plain.scale["k"][ids[1:]], plain.offset["k"][ids[1:]] = 8, 0, 0
    flat = lambda t: t[ids, 0].flatten(0, 1)[:length]  # noqa: E731
    power = 2.0**-12
    f.k[0][0] = flat(plain.values("k"))
    steps = (flat(plain.u["v"]).double().unflatten(-1, (-1, GROUP)) - 8) * flat(plain.scale["v"]).double()[..., None]
    f.s[0][0] = steps.flatten(-2) * power
    f.o[0][0] = flat(plain.offset["v"]).double().repeat_interleave(GROUP, -1) * power
    f.step[0][0] = flat(plain.scale["v"]).double().repeat_interleave(GROUP, -1) * power
    f.e[0][0] = -12.0
    f.cache = type(f.cache).from_tensors(*(t.cuda() for t in plain.tensors()), "int4")
    q = torch.ones(n, 2, dim).to(torch.bfloat16)
    f.check(q, [n], f.attend(q, [n]))
