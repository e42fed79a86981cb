"""Calls of different sizes from several host threads: a kernel's limit of dynamic
shared memory is one for all of them."""

from __future__ import annotations

import re
import sys
import threading

import pytest
import torch

from se12_b200 import _build


def test_the_limit_is_set_in_one_place_to_one_value():
    """Whoever sets it to a call's own size may lower it between another thread's
    setting and launch."""
    found = [(p.name, line.strip()) for p in _build.sources() for line in p.read_text().splitlines()
             if re.search(r"cudaFuncSetAttribute|cuFuncSetAttribute", line)]
    assert [name for name, _ in found] == ["se12_launch.h"], found
    assert "kMaxSmemPerCta - fixed" in found[0][1]


def in_threads(calls, times):
    """Each call again and again, all at once, each by a thread with a stream of its own."""
    errors, gate = [], threading.Barrier(len(calls))

    def work(call):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait(60)
                for _ in range(times):
                    call()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    try:
        threads = [threading.Thread(target=work, args=(c,)) for c in calls]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    assert not errors, errors[0]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,n", [("int4", 1), ("int4", 64), ("int8", 1), ("int8", 64)])
def test_attention_over_few_and_many_sequences_at_once(kind, n):
    """By the C entry, so that little else than launches is done."""
    from se12_b200 import _lib
    from se12_b200.kv_cache import PagedKvCache

    g = torch.Generator().manual_seed(n)
    lib = _lib.load()
    cache = PagedKvCache(4, 16, 1, 128, kind)
    x = torch.randn(64, 1, 128, generator=g).cuda()
    table = torch.arange(4, dtype=torch.int32)[None].cuda()
    cache.append(x, x, table, torch.tensor([64], dtype=torch.int32).cuda(), query_start=torch.tensor([0, 64], dtype=torch.int32).cuda())
    calls, outs = [], []
    need = lib.se12_kv_attend_call_bytes(cache.handle, 2, n)
    for seqs in (1, 2000, 1, 1000):
        # (of many sequences one has queries: a call that takes no time)
        lens, start = torch.full((seqs,), 64, dtype=torch.int32).cuda(), torch.tensor([0] + [n] * seqs, dtype=torch.int32).cuda()
        q = torch.randn(n, 2, 128, generator=g).to(torch.bfloat16).cuda()
        want = cache.attend(q, table.expand(seqs, 4), lens, query_start=start, max_query=n)
        out, space = torch.empty_like(q), torch.zeros(need, dtype=torch.uint8, device="cuda")
        batch = _lib.KV_BATCH.pack(seqs, n, lens.data_ptr(), start.data_ptr(), table.data_ptr(), 0, 4)
        args = _lib.KV_ATTEND.pack(q.data_ptr(), 256, 128, out.data_ptr(), 256, 128, 2, n, 0, 128**-0.5, 0.0)

        def call(batch=batch, args=args, space=space, keep=(lens, start, q)):
            stream = torch._C._cuda_getCurrentRawStream(0)
            for _ in range(1000):
                assert lib.se12_kv_attend(cache.handle, batch, args, space.data_ptr(), need, stream) == 0, lib.se12_last_error()

        calls.append(call)
        outs.append((out, want))
    torch.cuda.synchronize()
    in_threads(calls, 20)
    torch.cuda.synchronize()
    for out, want in outs:
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))


@pytest.mark.gpu
def test_products_of_several_widths_at_once():
    from se12_b200.codec import encode_device

    g = torch.Generator().manual_seed(0)
    calls = []
    for cols in (256, 2048, 4096):
        m = encode_device((torch.randn(64, cols, generator=g) / 16).to(torch.bfloat16).cuda())
        x = torch.randn(1, cols, generator=g).to(torch.bfloat16).cuda()
        calls.append(lambda m=m, x=x: m.gemv(x))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    in_threads(calls, 3000)
    for call, w in zip(calls, want):
        assert torch.equal(call(), w)
