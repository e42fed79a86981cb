"""Norms of queries and keys per head in front of the position rotation, in
the append to the 8-bit cache: the same codes, scales and rotated queries as
elementary fp32 operations give on normalised rows (the norm's factor from
64-bit sums, as the kernels have it), bit for bit."""

from __future__ import annotations

import pytest
import torch
from test_kv_cache import make_pair, random_tables, rope, rotate, same_cache, starts_of


def normalise(x, weight, eps):
    """x [..., dim] as fp32: x f w, f = 1 / sqrt(mean(x^2) + eps) rounded to fp32."""
    if weight is None:
        return x.float()
    f = 1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps)
    return (x.float() * f.float()) * weight.float()


def test_the_plain_norm_and_rotation_are_the_formulas():
    """Against 64 bits: two products and a rounded factor (3 half units of 2^-24
    each), then two products and a sum (2 more, of |a| + |b|)."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(50, 128, generator=g) * 4, torch.randn(128, generator=g)
    cos, sin = rope(g, 1, 64)
    y = rotate(normalise(x, w, 1e-6), cos[0], sin[0], False)
    z = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-6) * w.double()
    a, b, c, s = z[:, :64], z[:, 64:], cos.double(), sin.double()
    want = torch.cat((a * c - b * s, b * c + a * s), -1)
    size = torch.cat((a.abs() + b.abs(), a.abs() + b.abs()), -1)
    assert bool(((y.double() - want).abs() <= 5 * 2.0**-24 * 1.01 * size).all())


CASES = [
    # kind, dtype, page, heads, q_heads, dim, rotary (0: none), interleaved, weights' type, which norms
    ("int8", torch.float32, 16, 2, 4, 256, 256, False, torch.float32, "qk"),
    ("e4m3", torch.bfloat16, 32, 2, 6, 128, 128, False, torch.bfloat16, "qk"),
    ("int8", torch.bfloat16, 64, 3, 3, 128, 128, False, torch.float32, "k"),
    ("e4m3", torch.float32, 16, 1, 8, 256, 256, False, torch.bfloat16, "q"),
    ("int8", torch.float32, 16, 2, 2, 96, 32, False, torch.float32, "qk"),    # partial rotation
    ("e4m3", torch.bfloat16, 16, 2, 2, 80, 80, True, torch.bfloat16, "qk"),   # neighbouring pairs
    ("int8", torch.float32, 128, 1, 2, 128, 128, True, torch.float32, "qk"),
    ("e4m3", torch.float32, 16, 1, 1, 16, 2, False, torch.bfloat16, "qk"),
    ("int8", torch.float32, 256, 2, 2, 128, 0, False, torch.float32, "qk"),   # norms alone
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype,page,heads,q_heads,dim,rotary,interleaved,w_dtype,which", CASES)
@pytest.mark.parametrize("steps", [
    [[1, 1, 1, 1, 1]] * 3,                                    # next tokens
    [[40, 1, 0, 17, 3], [1, 16, 33, 0, 2], [5, 5, 5, 5, 5]],  # prompts, continued
    [[300, 0, 0, 0, 1], [1, 1, 1, 1, 1]],
])
def test_append_with_norms_stores_the_same_codes(kind, dtype, page, heads, q_heads, dim, rotary, interleaved, w_dtype, which, steps):
    g = torch.Generator().manual_seed(3 * dim + page)
    counts = [sum(s[b] for s in steps) for b in range(5)]
    table, pool = random_tables(g, counts, page)
    cache, plain = make_pair(pool, page, heads, dim, kind)
    cos, sin = rope(g, max(counts), rotary // 2) if rotary else (None, None)
    q_norm, k_norm = ((1 + 0.5 * torch.randn(dim, generator=g)).to(w_dtype) if w in which else None for w in "qk")
    eps, lens = 1e-5, [0] * 5
    for step, new in enumerate(steps):
        lens = [a + b for a, b in zip(lens, new)]
        starts = starts_of(new)
        y = (torch.randn(starts[-1], q_heads + 2 * heads, dim, generator=g) * 3.0**step * (1 + 9 * torch.rand(dim, generator=g))).to(dtype)
        q, k, v = y[:, :q_heads], y[:, q_heads : q_heads + heads], y[:, q_heads + heads :]
        want = plain.append(normalise(k, k_norm, eps), v, table, lens, starts, cos, sin, interleaved, normalise(q, q_norm, eps))
        d = y.cuda()
        start = None if all(n == 1 for n in new) else torch.tensor(starts, dtype=torch.int32).cuda()
        got = cache.append(d[:, q_heads : q_heads + heads], d[:, q_heads + heads :], table.cuda(),
                           torch.tensor(lens, dtype=torch.int32).cuda(), q=d[:, :q_heads], query_start=start,
                           cos=None if cos is None else cos.cuda(), sin=None if sin is None else sin.cuda(), interleaved=interleaved,
                           q_norm=None if q_norm is None else q_norm.cuda(), k_norm=None if k_norm is None else k_norm.cuda(),
                           norm_eps=eps)
        assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
        same_cache(cache, plain)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "int4"])
def test_norms_of_odd_rows(kind):
    """Zero rows stay zero, tiny and huge ones (whose squares pass fp32's range)
    are normalised like others, weights may lie at odd addresses, a padding row
    gives zeros, and keys may be appended without queries."""
    from se12_b200.kv_cache import PagedKvCache

    g = torch.Generator().manual_seed(9)
    dim, page = 128, 16
    cache = PagedKvCache(4, page, 1, dim, kind)
    sizes = torch.tensor([0.0, 1e-18, 1.0, 1e25, 3.0])
    x = torch.randn(5, 1, dim, generator=g) * sizes[:, None, None]
    weight = torch.randn(dim + 1, generator=g)
    eps = 1e-38
    want = normalise(x, weight[1:], eps)
    table = torch.zeros(5, 1, dtype=torch.int32)
    table[:4, 0] = torch.arange(4)
    lens = torch.tensor([1, 1, 1, 1, 0], dtype=torch.int32)
    w = weight.cuda()[1:]
    got = cache.append(x.cuda(), x.cuda() * 0, table.cuda(), lens.cuda(), q=x.cuda(), q_norm=w, k_norm=w, norm_eps=eps)
    assert torch.equal(got[:4].cpu().view(torch.int16), want[:4].to(torch.bfloat16).view(torch.int16))
    assert bool((got[4] == 0).all())
    first = cache.decode()[0][:, 0, 0].cpu()
    assert bool((first[0] == 0).all()) and bool(torch.isfinite(first).all())
    # a step of the code's grid, and BF16's rounding of what is read back
    step = want[:4, 0].abs().amax(-1, keepdim=True) * (2 / 127 if kind == "int8" else 2 / 15)
    assert bool(((first.float() - want[:4, 0]).abs() <= 0.51 * step + 2.0**-8 * want[:4, 0].abs()).all())
    before = cache.k_codes.clone()
    assert cache.append(x.cuda(), x.cuda() * 0, table.cuda(), lens.cuda(), k_norm=w, norm_eps=eps) is None
    assert torch.equal(before, cache.k_codes)


def test_refusals_of_norms_come_before_the_device():
    """The checks of the weights, without a GPU: they only look at the tensors."""
    from se12_b200.kv_cache import PagedKvCache

    cache = PagedKvCache.__new__(PagedKvCache)
    cache.device, cache.head_dim, cache.kv_heads = torch.device("cpu"), 64, 1
    good = torch.ones(64)
    assert cache._norm_weight(None, "q_norm") == (0, False)
    assert cache._norm_weight(good, "q_norm") == (good.data_ptr(), False)
    assert cache._norm_weight(good.bfloat16(), "q_norm")[1] is True
    for bad in (torch.ones(63), torch.ones(1, 64), torch.ones(64, dtype=torch.float16), torch.ones(128)[::2]):
        with pytest.raises(ValueError):
            cache._norm_weight(bad, "q_norm")
    k = torch.ones(1, 1, 64)
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            cache.append(k, k, None, None, q=k, q_out=k.bfloat16(), q_norm=good, norm_eps=eps)
    with pytest.raises(ValueError):
        cache.append(k, k, None, None, q_norm=good)


def test_abi_refuses_bad_norms():
    from se12_b200 import _build, _lib

    _build.build()
    lib = _lib.load()
    assert lib.se12_kv_append_normed(None, None, None, None, None) == 1
    assert _lib.KV_NORMS.size == 32


def test_abi_refuses_misaligned_weights():
    """Before anything else of the call is looked at on the device: the handle is
    one made without a GPU's work (its pointers are never followed)."""
    from se12_b200 import _build, _lib

    _build.build()
    lib = _lib.load()
    if torch.cuda.is_available():
        from se12_b200.kv_cache import PagedKvCache

        x = torch.zeros(1, 1, 64, device="cuda")
        cache, ints = PagedKvCache(1, 16, 1, 64), torch.ones(1, 1, dtype=torch.int32, device="cuda")
        batch = _lib.KV_BATCH.pack(1, 1, ints.data_ptr(), 0, ints.data_ptr(), 1, 1)
        args = _lib.KV_APPEND.pack(False, 1, x.data_ptr(), x.data_ptr(), x.data_ptr(), *[64] * 6, 0, 0, 0, 0, 0, False, x.data_ptr(), 64, 64)
        for q, k, bf16, want in ((x.data_ptr() + 2, 0, 0, 3), (0, x.data_ptr() + 1, 1, 3)):
            norms = _lib.KV_NORMS.pack(q, k, bf16, bf16, 1e-6)
            assert lib.se12_kv_append_normed(cache.handle, batch, args, norms, None) == want
        assert lib.se12_kv_append_normed(cache.handle, batch, args, _lib.KV_NORMS.pack(0, 0, 0, 0, -1.0), None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("tokens", [40, 300])
def test_rows_behind_the_last_sequence_are_not_stored(kind, tokens):
    """query_start ends before the batch does, and begins after its first rows:
    those rows' queries are zeros, their keys and values are nowhere."""
    from se12_b200.kv_cache import PagedKvCache

    g = torch.Generator().manual_seed(tokens)
    dim, heads, page = 128, 2, 16
    n = tokens - 13
    table = torch.arange(40, dtype=torch.int32).view(2, 20).cuda()
    lens = torch.tensor([n - 5, 5], dtype=torch.int32).cuda()
    start = torch.tensor([3, n - 2, n + 3], dtype=torch.int32).cuda()
    x = torch.randn(tokens, heads, dim, generator=g).cuda()
    w = torch.randn(dim, generator=g).cuda()
    cos, sin = (t.cuda() for t in rope(g, 400, dim // 2))
    whole, part = (PagedKvCache(40, page, heads, dim, kind) for _ in range(2))
    q = whole.append(x, x, table, lens, q=x, query_start=start, cos=cos, sin=sin, q_norm=w, k_norm=w)
    rows = slice(3, n + 3)
    again = part.append(x[rows], x[rows], table, lens, q=x[rows], query_start=start - 3, cos=cos, sin=sin, q_norm=w, k_norm=w)
    assert torch.equal(q[rows], again) and not q[:3].any() and not q[n + 3 :].any()
    assert torch.equal(whole.k_codes, part.k_codes) and torch.equal(whole.v_codes, part.v_codes)
    assert torch.equal(whole.k_scales, part.k_scales) and torch.equal(whole.v_scales, part.v_scales)
