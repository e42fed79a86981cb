"""Token log probabilities against 64-bit sums over the same logits.

Tolerance of a log probability or an entropy, absolute: a term exp(z - M)
carries 2^-22 (the exponential) and the rounding of (z - M) log2(e) (2^-24 of
at most 200), sums of a few dozen roundings of 2^-24, so below 1e-5 of the
sum, plus 2^-21 of the result; capped logits are off by at most 2^-20 of the
cap (the exponential's and the quotient's 2^-22 and the argument's rounding).
Ids are exact.
"""

from __future__ import annotations

import math

import pytest
import torch

from se12_b200.logprobs import MAX_TOP, token_logprobs


def plain(x: torch.Tensor, tokens: torch.Tensor, top: int, softcap: float):
    x64 = x.double()
    z = x64 if not softcap else torch.where(x64 == -math.inf, x64, softcap * torch.tanh(x64 / softcap))
    logp = torch.log_softmax(z, -1)
    p = logp.exp()
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(-1)
    safe = tokens.clamp(0, x.shape[1] - 1)
    lp = logp.gather(1, safe[:, None])[:, 0]
    lp = torch.where((tokens < 0) | (tokens >= x.shape[1]), torch.full_like(lp, math.nan), lp)
    order = torch.where(x64.isnan(), torch.full_like(x64, math.inf), x64.clamp(-1e308, 1e307))  # NaN above +inf
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices[:, :top]
    return lp, entropy, ids, logp.gather(1, ids)


def check(x: torch.Tensor, tokens: torch.Tensor, top: int, softcap: float = 0.0, device_logits=None):
    got = token_logprobs(x.cuda() if device_logits is None else device_logits, tokens.cuda(), top=top, softcap=softcap)
    want = plain(x, tokens, top, softcap)
    assert got.top_ids.shape == (x.shape[0], top) and got.top_ids.dtype == torch.int64
    assert torch.equal(got.top_ids.cpu(), want[2])
    for g, w in ((got.logprob, want[0]), (got.entropy, want[1]), (got.top_logprobs, want[3])):
        g = g.double().cpu()
        assert torch.equal(g.isnan(), w.isnan()) and torch.equal(g.isinf(), w.isinf())
        fine = torch.isfinite(w)
        tol = 1e-5 + 2.0**-20 * softcap + 2.0**-21 * w.abs()
        assert bool(((g - w).abs() <= tol)[fine].all()), float(((g - w).abs() / tol)[fine].max())
    return got


def logits(seed: int, rows: int, vocab: int, dtype=torch.float32, spread: float = 3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * spread).to(dtype)
    return x, torch.randint(0, vocab, (rows,), generator=g)


# ------------------------------------------------------------------ CPU: refusals


def test_refusals():
    x, t = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64)
    for call in (
        lambda: token_logprobs(x[0], t),
        lambda: token_logprobs(x.half(), t),
        lambda: token_logprobs(x.double(), t),
        lambda: token_logprobs(x.t().contiguous().t(), t),
        lambda: token_logprobs(x, t.int()),
        lambda: token_logprobs(x, t[:1]),
        lambda: token_logprobs(x, t, top=-1),
        lambda: token_logprobs(x, t, top=11),
        lambda: token_logprobs(torch.zeros(2, 100), t, top=MAX_TOP + 1),
        lambda: token_logprobs(x, t, softcap=-1.0),
        lambda: token_logprobs(x, t, softcap=math.inf),
        lambda: token_logprobs(x, t, softcap=math.nan),
        lambda: token_logprobs(x, t),  # not on a GPU
    ):
        with pytest.raises(ValueError):
            call()


def test_abi_refuses_bad_arguments_without_a_device():
    from se12_b200 import _build, _lib

    _build.build()
    lib = _lib.load()
    need = lib.se12_token_logprobs_workspace_bytes()

    def call(logits=256, rows=2, vocab=10, ld=10, tokens=256, top=2, softcap=0.0, ids=256, ws=256, size=need):
        return lib.se12_token_logprobs(logits, 0, rows, vocab, ld, tokens, top, softcap, 256, 256, ids, 256, ws, size, None)

    assert call(logits=None) == 1 and call(tokens=None) == 1 and call(rows=0) == 1 and call(ld=9) == 1 and call(top=33) == 1
    assert call(top=11) == 1 and call(ids=None) == 1 and call(softcap=-1.0) == 1 and call(softcap=math.nan) == 1
    assert call(ws=None) == 4 and call(size=need - 1) == 4 and call(ws=264) == 3


# ------------------------------------------------------------------ GPU


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 31), (2, 33), (5, 1000), (4, 8191), (4, 8192), (4, 8193), (1, 100003),
                                        (2, 256000), (700, 4099), (301, 16384), (1, 1000000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_sizes(rows, vocab, dtype, softcap):
    x, t = logits(rows + vocab, rows, vocab, dtype)
    for top in sorted({0, min(1, vocab), min(5, vocab), min(32, vocab)}):
        check(x, t, top, softcap)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [50, 9000, 70000])
def test_equal_values_go_to_the_lowest_id(vocab):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randint(-3, 3, (6, vocab), generator=g).to(torch.float32)
    x[0] = 1.0                       # a constant row
    x[1] = torch.where(torch.rand(vocab, generator=g) < 0.5, 0.0, -0.0)  # zeros of both signs are equal
    x[2, 7:] = -math.inf
    t = torch.randint(0, vocab, (6,), generator=g)
    check(x, t, 20)
    check(x.to(torch.bfloat16), t, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [300, 40000])
def test_sorted_rows(vocab):
    """Every value of an ascending row enters the list."""
    x = torch.linspace(-20, 20, vocab)[None].repeat(3, 1)
    x[1] = x[1].flip(0)
    x[2] = x[2].roll(vocab // 2)
    check(x, torch.tensor([0, 1, vocab - 1]), 32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("period,equal", [(2048, 300), (1024, 100), (4096, 40), (2048, 2000)])
def test_equal_values_of_a_stripe_of_columns(dtype, period, equal):
    """Thousands of equal values at the top, all of them in a few (or most) of
    the threads that share a row; rows with NaN and +inf among them."""
    rows, vocab = 600, 40007
    x, t = logits(period + equal, rows, vocab, dtype)
    stripe = torch.arange(vocab) % period < equal
    x[:, stripe] = 64.0
    x[1, 30000] = math.inf
    x[2, ::5000] = math.inf
    x[3, 5000:5010] = math.nan
    x[4, ~stripe] = -math.inf
    x[5, stripe] = -math.inf
    check(x, t, 20)
    wide = torch.zeros(rows, vocab + 4, dtype=dtype, device="cuda")[:, 1 : vocab + 1]  # not on 16 bytes
    check(x, t, 32, device_logits=wide.copy_(x))


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("vocab", [40, 20000, 200000])
def test_banned_tokens(vocab, softcap):
    g = torch.Generator().manual_seed(1)
    x, t = logits(3, 6, vocab)
    x[0, torch.rand(vocab, generator=g) < 0.9] = -math.inf
    x[1] = -math.inf
    x[1, vocab // 2] = 2.0               # one token left
    x[2] = -math.inf
    x[2, -3:] = torch.tensor([1.0, 1.0, -4.0])
    x[3, : vocab // 2] = -math.inf
    x[4, 5:] = -math.inf                 # fewer tokens than alternatives
    t[0] = int((x[0] == -math.inf).nonzero()[0, 0])  # a banned token: -inf
    check(x, t, 20, softcap)
    check(x.to(torch.bfloat16), t, 20, softcap)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 20000])
def test_masks_of_the_lowest_value_and_empty_rows(vocab):
    low = torch.finfo(torch.float32).min
    x, t = logits(4, 7, vocab)
    x[0, ::2] = low
    x[1] = low                           # uniform
    x[2] = -math.inf                     # nothing left: NaN
    x[3] = low
    x[3, 3] = -math.inf
    x[4] = low
    x[4, 9] = 0.5
    x[5] = -3.0e38
    x[6, 11] = 3.0e38                    # forced
    got = check(x, t, 5)
    assert bool(got.logprob[2].isnan()) and got.top_ids[2].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("vocab", [100, 20000])
def test_values_that_are_not_finite_stay_in_their_rows(vocab, bad):
    x, t = logits(5, 4, vocab)
    x[1, vocab - 1] = bad
    x[2, 0] = bad
    x[2, 60] = bad
    got = check(x, t, 8)
    assert bool(got.logprob[1].isnan()) and bool(got.entropy[2].isnan()) and not bool(got.logprob[0].isnan())
    assert int(got.top_ids[1, 0]) == vocab - 1 and got.top_ids[2, :2].tolist() == [0, 60]


@pytest.mark.gpu
def test_tokens_outside_the_vocabulary():
    from se12_b200.device import device_status

    x, _ = logits(6, 3, 500)
    check(x, torch.tensor([-1, 5, -100]), 3)
    assert device_status() == 0
    check(x, torch.tensor([499, 500, 1 << 40]), 3)
    assert device_status() == 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (5, 1), (0, 3)])
def test_strides_and_alignment(dtype, pad, offset):
    x, t = logits(7, 5, 9001, dtype)
    wide = torch.full((5, 9001 + pad + offset), 99.0, dtype=dtype)
    wide[:, offset : offset + 9001] = x
    check(x, t, 10, device_logits=wide.cuda()[:, offset : offset + 9001])


@pytest.mark.gpu
def test_large_and_small_logits():
    for spread in (1e-3, 100.0, 1e4):
        x, t = logits(8, 3, 30000, spread=spread)
        check(x, t, 5)
    x, t = logits(9, 3, 30000)
    check(x + 1000.0, t, 5)


@pytest.mark.gpu
def test_streams_and_graphs():
    x, t = logits(10, 2, 150000)
    dx, dt = x.cuda(), t.cuda()
    want = token_logprobs(dx, dt, top=7, softcap=30.0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = token_logprobs(dx, dt, top=7, softcap=30.0)
        for _ in range(3):
            graph.replay()
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    y, _ = logits(11, 2, 150000)
    dx.copy_(y.cuda())
    want = token_logprobs(dx, dt, top=7, softcap=30.0)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_rows_past_31_bits_of_values():
    """More than 2^31 logits: the last rows are the last rows."""
    rows, vocab = 16400, 131072
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    y, t = logits(12, 2, vocab, torch.bfloat16)
    x[-2:] = y.cuda()
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    tokens[-2:] = t.cuda()
    got = token_logprobs(x, tokens, top=3)
    want = plain(y, t, 3, 0.0)
    assert torch.equal(got.top_ids[-2:].cpu(), want[2]) and got.top_ids[:-2].unique().tolist() == [0, 1, 2]
    assert bool(((got.logprob[-2:].cpu().double() - want[0]).abs() <= 1e-5 + 2.0**-21 * want[0].abs()).all())
    assert bool(((got.logprob[:-2].double() + math.log(vocab)).abs() < 1e-5).all())


@pytest.mark.gpu
def test_no_rows():
    got = token_logprobs(torch.zeros(0, 10, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), top=3)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 3)


def test_abi_takes_one_row_for_several_tokens():
    """A row stride of zero passes the checks (the next one is the workspace's)."""
    from se12_b200 import _build, _lib

    _build.build()

    def call(ld):
        return _lib.load().se12_token_logprobs(256, 0, 2, 10, ld, 256, 2, 0.0, 256, 256, 256, 256, None, 0, None)

    assert call(0) == 4 and call(-10) == 1 and call(9) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 33, 5000, 70000])
def test_expanded_and_overlapping_rows(dtype, vocab):
    """Several candidates against one expanded row, rows that overlap, one row
    of any stride: as for a copy of them."""
    x, t = logits(16, 5, vocab + 8, dtype)
    t = t % vocab
    row = x[1:2, :vocab]
    check(row.expand(5, -1), t, min(4, vocab), device_logits=x.cuda()[1:2, :vocab].expand(5, -1))
    flat = x.reshape(-1)[: vocab + 8]
    for step in (1, 2):
        view = flat.cuda().as_strided((5, vocab), (step, 1))
        check(flat.as_strided((5, vocab), (step, 1)), t, min(4, vocab), device_logits=view)
    check(row, t[:1], min(4, vocab), device_logits=x.cuda()[1:2, :vocab].as_strided((1, vocab), (0, 1), x.shape[1]))
    check(x[:, :vocab], t, min(4, vocab), device_logits=x.cuda()[:, :vocab])


@pytest.mark.gpu
def test_workspace_is_prepared_on_the_logits_device(monkeypatch):
    """With another GPU current (here by what the library is told), the
    workspace is cleared and the kernel launched with the logits' GPU current."""
    from se12_b200 import _lib, logprobs

    x, t = logits(17, 2, 5000)
    dx, dt = x.cuda(), t.cuda()
    want = token_logprobs(dx, dt, top=3)
    inside, seen = [], []
    real_device, real_pool = torch.cuda.device, logprobs._WORKSPACES

    class Device(real_device):
        def __enter__(self):
            inside.append(1)
            return super().__enter__()

        def __exit__(self, *args):
            inside.pop()
            return super().__exit__(*args)

    class Pool:
        def get(self, device, stream, nbytes):
            seen.append(len(inside))
            return real_pool.get(device, stream, nbytes)

    monkeypatch.setattr(logprobs, "_WORKSPACES", Pool())
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0 if inside else 1)
    got = token_logprobs(dx, dt, top=3)
    assert seen == [1] and _lib.is_loaded()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("others", [-20.0, -60.0])
def test_certain_rows_have_no_positive_log_probability(softcap, dtype, others):
    """Rows with one token of probability 1 but for 1e-9 or less: a log
    probability is never above zero, an entropy never below."""
    g = torch.Generator().manual_seed(13)
    rows, vocab = 2000, 1000
    x = others + torch.randn(rows, vocab, generator=g) * 0.3
    t = torch.randint(0, vocab, (rows,), generator=g)
    x.scatter_(1, t[:, None], 5.0 + 40.0 * torch.rand(rows, 1, generator=g))
    got = check(x.to(dtype), t, 3, softcap)
    assert bool((got.logprob <= 0).all()), float(got.logprob.max())
    assert bool((got.top_logprobs <= 0).all()) and bool((got.entropy >= 0).all()), float(got.entropy.min())


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [0.5, 30.0, 1e3, 1e5, 1e8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("banned", [0.0, 0.3])
def test_caps_of_any_size(softcap, dtype, banned):
    """Caps far below and far above the logits, with and without banned
    tokens: a capped logit is off by a few roundings of its own size (six of
    2^-23), not of the cap's."""
    x, t = logits(14, 6, 30011, dtype)
    g = torch.Generator().manual_seed(15)
    ban = torch.rand(x.shape, generator=g) < banned
    ban.scatter_(1, t[:, None], False)
    x[ban] = -math.inf
    got = token_logprobs(x.cuda(), t.cuda(), top=8, softcap=softcap)
    want = plain(x, t, 8, softcap)
    assert torch.equal(got.top_ids.cpu(), want[2])
    largest = min(softcap, 20.0)
    for a, b in ((got.logprob, want[0]), (got.entropy, want[1]), (got.top_logprobs, want[3])):
        tol = 1e-5 + 6 * 2.0**-23 * largest + 2.0**-21 * b.abs()
        assert bool(((a.double().cpu() - b).abs() <= tol).all()), float(((a.double().cpu() - b).abs() / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [100, 20000])
def test_infinite_logits_under_a_cap(vocab):
    """+inf is a logit of the cap there, NaN stays NaN."""
    x, t = logits(18, 4, vocab)
    x[1, vocab - 1] = math.inf
    x[2, 0] = math.nan
    x[3] = -math.inf
    x[3, 7] = math.inf
    got = check(x, t, 8, softcap=30.0)
    assert bool(torch.isfinite(got.entropy[1])) and bool(got.entropy[2].isnan())


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [1e-20, 1e-38, 1e-40])
def test_a_vanishing_cap_makes_all_tokens_equal(softcap):
    x, t = logits(19, 2, 500)
    x[0, 3] = 0.0
    got = token_logprobs(x.cuda(), t.cuda(), top=2, softcap=softcap)
    for v in (got.logprob, got.top_logprobs):
        assert bool(((v.double() + math.log(500)).abs() < 1e-5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [40, 9001, 70000])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("top", [0, 9])
def test_rows_that_are_summed_again(dtype, vocab, softcap, top):
    """Empty rows, masks of the lowest value alone, values near the largest
    and infinities, among ordinary rows, aligned and not."""
    x, t = logits(20, 9, vocab, dtype)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x[1] = -math.inf
    x[2] = low
    x[3] = low
    x[3, 5:30] = -math.inf
    x[4, 7] = high
    x[5, 3] = x[5, 30] = high
    x[6, 11] = math.inf
    x[7] = low / 2
    x[7, 20:] = low / 2 * (1 + 2.0**-6)
    check(x, t, top, softcap)
    wide = torch.zeros(9, vocab + 3, dtype=dtype, device="cuda")[:, 1 : vocab + 1]
    check(x, t, top, softcap, device_logits=wide.copy_(x))


@pytest.mark.gpu
def test_an_empty_row_does_not_hold_up_the_others():
    """One row with nothing left among 16 takes no more than a few times the
    others' time (it was seventy times: one warp went over the row twice)."""
    x, t = logits(21, 16, 256000)
    plain_rows, with_empty = x.cuda(), x.cuda()
    with_empty[3] = -math.inf
    t = t.cuda()

    def time(logits_):
        for _ in range(3):
            token_logprobs(logits_, t, top=5)
        best = math.inf
        for _ in range(5):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(10):
                token_logprobs(logits_, t, top=5)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end))
        return best

    assert time(with_empty) < 10 * time(plain_rows)
