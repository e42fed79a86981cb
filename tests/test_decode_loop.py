"""The decode-loop example: cache, attention and log probabilities together
with the SE12 GEMVs, eagerly and as a replayed graph."""

from __future__ import annotations

import pathlib
import sys

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "examples"))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_greedy_tokens_and_their_log_probabilities(kind):
    from decode_loop import Decoder, Shape, generate

    prompts = [[(7 * i + 3 * j) % 4096 for j in range(n)] for i, n in enumerate((5, 100, 33, 1))]
    eager_ids, eager = generate(Decoder(Shape(kind=kind)), prompts, 10)
    graph_ids, graph = generate(Decoder(Shape(kind=kind)), prompts, 10, graph=True)
    assert torch.equal(eager_ids, graph_ids)
    for ids, a, b in zip(eager_ids.unbind(1), eager, graph):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
        # the greedy token is the first alternative, with the same log probability
        assert torch.equal(a.top_ids[:, 0], ids) and torch.equal(a.top_logprobs[:, 0], a.logprob)
        assert bool((a.logprob <= 0).all()) and bool((a.entropy > 0).all())
        assert bool((a.top_logprobs[:, :-1] >= a.top_logprobs[:, 1:]).all())


@pytest.mark.gpu
def test_the_first_layer_sees_what_plain_attention_sees():
    """One layer's new row against 64-bit attention over the cache's values:
    projections, rotation, store and attention in one path. The tolerance is
    the attention tests'."""
    from decode_loop import Decoder, Shape, norm

    s = Shape(layers=1)
    model = Decoder(s, slots=2, positions=96)
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    model.prefill([list(range(40)), list(range(7, 60))], lens, chunk=16)
    lens.add_(1)
    layer = model.layers[0]
    x = model.embed(torch.tensor([11, 12], device="cuda")).float() * s.hidden**0.5
    y = layer.qkv.gemv(norm(x)).view(2, -1, s.head_dim)
    q = layer.cache.append(y[:, s.q_heads : s.q_heads + s.kv_heads], y[:, s.q_heads + s.kv_heads :], model.table, lens,
                           q=y[:, : s.q_heads], cos=model.cos, sin=model.sin)
    got = layer.cache.attend(q, model.table, lens, softcap=s.attn_softcap)
    keys, values = (t.double() for t in layer.cache.decode())
    for b in range(2):
        n = int(lens[b])
        pages = model.table[b, : (n + s.page - 1) // s.page].long()
        for h in range(s.q_heads):
            k, v = (t[pages, h * s.kv_heads // s.q_heads].reshape(-1, s.head_dim)[:n] for t in (keys, values))
            logits = k @ q[b, h].double() * s.head_dim**-0.5
            p = torch.softmax(s.attn_softcap * torch.tanh(logits / s.attn_softcap), 0)
            want, size = p @ v, p @ v.abs()
            half_unit = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=1e-300))) - 8)
            assert bool(((got[b, h].double() - want).abs() <= half_unit + 2.0**-10 * size + 2.0**-24 * n * v.abs().max()).all())


def test_the_captured_step_waits_for_its_inputs(monkeypatch):
    """generate(graph=True) with a model that records what runs on which
    stream: the side stream waits after the ids it reads have been written."""
    import contextlib

    import decode_loop

    log, current = [], ["main"]

    class Stream:
        def __init__(self, name="side"):
            self.name = name

        def wait_stream(self, other):
            log.append(("wait", self.name, other.name))

    class Ids(torch.Tensor):
        def clone(self):
            log.append(("clone", current[0]))
            return torch.Tensor.clone(self).as_subclass(torch.Tensor)

    @contextlib.contextmanager
    def on(stream):
        before, current[0] = current[0], stream.name
        yield
        current[0] = before

    class Graph:
        def replay(self):
            pass

    class Cuda:
        CUDAGraph = Graph

        def __init__(self):
            self.Stream, self.stream = Stream, on

        def current_stream(self):
            return Stream(current[0])

        def graph(self, captured, stream=None):
            return on(stream)

    class Torch:  # torch, on the CPU, with the streams above
        cuda = Cuda()

        def __getattr__(self, name):
            return getattr(torch, name)

        def zeros(self, *shape, device=None, **rest):
            return torch.zeros(*shape, **rest)

    class Model:
        shape = decode_loop.Shape()

        def prefill(self, prompts, lens):
            return torch.zeros(len(prompts), 4)

        def forward(self, ids, lens):
            log.append(("forward", current[0]))
            return torch.zeros(len(ids), 4)

        def logits(self, x):
            return x.as_subclass(Ids)

    monkeypatch.setattr(decode_loop, "torch", Torch())
    monkeypatch.setattr(decode_loop, "token_logprobs",
                        lambda logits, ids, **_: decode_loop.TokenLogprobs(*(torch.zeros(len(logits)) for _ in range(4))))
    decode_loop.generate(Model(), [[1], [2]], 2, graph=True)
    assert ("clone", "main") in log and ("forward", "side") in log
    assert log.index(("clone", "main")) < log.index(("wait", "side", "main")) < log.index(("forward", "side"))
