"""A small decoder served from SE12 weights: prompts in chunks, then one token
at a time, with a paged 8-bit cache and log probabilities.

Everything between the input ids and the log probabilities that is not a
norm, an activation or a sum runs in this package's kernels:

    CompressedEmbedding -> [qkv GEMV -> PagedKvCache.append -> PagedKvCache.attend
    -> o GEMV -> gate/up GEMV -> down GEMV] per layer -> LM head GEMV -> token_logprobs

The weights are random (seeded): the point is the calls and their shapes.
The decode step can be captured in a CUDA graph: lengths, page tables and
token ids are device tensors that the captured calls read anew each replay.

    python examples/decode_loop.py --layers 2 --new 12 --graph
"""

from __future__ import annotations

import argparse
import dataclasses
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent))

from se12_b200.codec import encode_device  # noqa: E402
from se12_b200.device import DeviceSe12Matrix  # noqa: E402
from se12_b200.kv_cache import PagedKvCache  # noqa: E402
from se12_b200.logprobs import TokenLogprobs, token_logprobs  # noqa: E402
from se12_b200.runtime import CompressedEmbedding  # noqa: E402


@dataclasses.dataclass(frozen=True)
class Shape:
    hidden: int = 512
    q_heads: int = 4
    kv_heads: int = 2
    head_dim: int = 128
    intermediate: int = 1024
    vocab: int = 4096
    layers: int = 2
    attn_softcap: float = 50.0
    final_softcap: float = 30.0
    window: int = 64  # of every other layer
    page: int = 16
    kind: str = "int8"


class Layer:
    def __init__(self, s: Shape, weights, pages: int, window: int):
        q, k, v = (weights(n * s.head_dim, s.hidden) for n in (s.q_heads, s.kv_heads, s.kv_heads))
        self.qkv = DeviceSe12Matrix.concatenate([encode_device(w) for w in (q, k, v)])
        self.o = encode_device(weights(s.hidden, s.q_heads * s.head_dim))
        self.gate_up = DeviceSe12Matrix.concatenate([encode_device(weights(s.intermediate, s.hidden)) for _ in range(2)])
        self.down = encode_device(weights(s.hidden, s.intermediate))
        self.cache = PagedKvCache(pages, s.page, s.kv_heads, s.head_dim, s.kind)
        self.window = window


def norm(x: torch.Tensor) -> torch.Tensor:
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)


class Decoder:
    """``slots`` sequences of up to ``positions`` tokens; every sequence owns
    its pages from the start."""

    def __init__(self, shape: Shape = Shape(), slots: int = 4, positions: int = 256, seed: int = 0):
        s, self.shape = shape, shape
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weights(rows: int, cols: int) -> torch.Tensor:
            return (torch.randn(rows, cols, generator=g, device="cuda") * cols**-0.5).to(torch.bfloat16)

        columns = (positions + s.page - 1) // s.page
        order = torch.randperm(slots * columns, generator=g, device="cuda").to(torch.int32)
        self.table = order.view(slots, columns).contiguous()
        self.layers = [Layer(s, weights, slots * columns, s.window if i % 2 else 0) for i in range(s.layers)]
        self.embed = CompressedEmbedding(encode_device(weights(s.vocab, s.hidden)))
        self.head = encode_device(weights(s.vocab, s.hidden))
        angle = torch.arange(positions, device="cuda")[:, None] * 1e4 ** (
            -torch.arange(0, s.head_dim, 2, device="cuda") / s.head_dim)[None, :]
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    def forward(self, ids: torch.Tensor, lens: torch.Tensor, query_start: torch.Tensor | None = None,
                max_query: int = 1) -> torch.Tensor:
        """Hidden states [tokens, hidden] of new tokens; ``lens`` counts them."""
        s = self.shape
        x = self.embed(ids).float() * s.hidden**0.5
        for layer in self.layers:
            y = layer.qkv.gemv(norm(x)).view(-1, s.q_heads + 2 * s.kv_heads, s.head_dim)
            q = layer.cache.append(y[:, s.q_heads : s.q_heads + s.kv_heads], y[:, s.q_heads + s.kv_heads :], self.table, lens,
                                   q=y[:, : s.q_heads], cos=self.cos, sin=self.sin, query_start=query_start)
            a = layer.cache.attend(q, self.table, lens, query_start=query_start, max_query=max_query,
                                   softcap=s.attn_softcap, window=layer.window)
            x = x + layer.o.gemv(a.view(-1, s.q_heads * s.head_dim))
            gate, up = layer.gate_up.gemv(norm(x)).chunk(2, dim=-1)
            x = x + layer.down.gemv((torch.nn.functional.gelu(gate, approximate="tanh") * up).to(torch.bfloat16))
        return x

    def logits(self, x: torch.Tensor) -> torch.Tensor:
        return self.head.gemv(norm(x))

    def prefill(self, prompts: list, lens: torch.Tensor, chunk: int = 48) -> torch.Tensor:
        """Runs the prompts (lists of ids) in chunks of up to ``chunk`` tokens of
        each; returns the last token's hidden state of each sequence."""
        last = torch.zeros(len(prompts), self.shape.hidden, device="cuda")
        for at in range(0, max(len(p) for p in prompts), chunk):
            parts = [p[at : at + chunk] for p in prompts]
            counts = [len(p) for p in parts]
            starts = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
            lens.add_(torch.tensor(counts, dtype=torch.int32, device="cuda"))
            x = self.forward(torch.tensor([t for p in parts for t in p], device="cuda"), lens, starts, max(counts))
            for i, n in enumerate(counts):
                if n:
                    last[i] = x[int(starts[i + 1]) - 1]
        return last


def generate(model: Decoder, prompts: list, new: int, top: int = 5, graph: bool = False) -> tuple:
    """Greedy continuation: (ids [slots, new], TokenLogprobs of each step)."""
    lens = torch.zeros(len(prompts), dtype=torch.int32, device="cuda")
    logits = model.logits(model.prefill(prompts, lens))
    ids = logits.argmax(-1)
    out, scores = [], []

    def step(ids, lens):
        logits = model.logits(model.forward(ids, lens))
        chosen = logits.argmax(-1)
        return chosen, token_logprobs(logits, chosen, top=top, softcap=model.shape.final_softcap)

    scores.append(token_logprobs(logits, ids, top=top, softcap=model.shape.final_softcap))
    out.append(ids)
    captured = None
    if graph:
        held = ids.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            scratch = torch.zeros_like(lens)
            step(held, scratch)  # padding rows: nothing is stored
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured, stream=side):
                chosen, score = step(held, lens)
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(new - 1):
        lens.add_(1)
        if captured is None:
            ids, s = step(ids, lens)
        else:
            held.copy_(ids)
            captured.replay()
            ids, s = chosen.clone(), TokenLogprobs(*(t.clone() for t in score))
        out.append(ids)
        scores.append(s)
    return torch.stack(out, 1), scores


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--new", type=int, default=12)
    p.add_argument("--kind", choices=("int8", "e4m3"), default="int8")
    p.add_argument("--graph", action="store_true", help="replay the decode step as one CUDA graph")
    a = p.parse_args()
    model = Decoder(Shape(layers=a.layers, kind=a.kind))
    prompts = [[(7 * i + 3 * j) % 4096 for j in range(n)] for i, n in enumerate((5, 100, 33, 1))]
    ids, scores = generate(model, prompts, a.new, graph=a.graph)
    for i, prompt in enumerate(prompts):
        line = " ".join(f"{int(t)}({float(s.logprob[i]):.2f})" for t, s in zip(ids[i], scores))
        print(f"prompt of {len(prompt)} tokens -> {line}; entropy of the last step {float(scores[-1].entropy[i]):.2f}")


if __name__ == "__main__":
    main()
