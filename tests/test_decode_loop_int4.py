"""The decode-loop example with a 4-bit cache and normalised queries and keys."""

from __future__ import annotations

import pathlib
import subprocess
import sys

import pytest
import torch

from se12_b200 import _build

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "examples"))


@pytest.mark.gpu
@pytest.mark.parametrize("kind,qk_norm", [("int4", False), ("int4", True), ("int8", True)])
def test_greedy_tokens_eagerly_and_as_a_graph(kind, qk_norm):
    from decode_loop import Decoder, Shape, generate

    prompts = [[(7 * i + 3 * j) % 4096 for j in range(n)] for i, n in enumerate((5, 100, 33, 1))]
    shape = Shape(kind=kind, qk_norm=qk_norm)
    eager_ids, eager = generate(Decoder(shape), prompts, 10)
    graph_ids, graph = generate(Decoder(shape), prompts, 10, graph=True)
    assert torch.equal(eager_ids, graph_ids)
    for ids, a, b in zip(eager_ids.unbind(1), eager, graph):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
        assert torch.equal(a.top_ids[:, 0], ids) and torch.equal(a.top_logprobs[:, 0], a.logprob)


@pytest.mark.gpu
def test_one_layer_of_all_operators_against_plain_sums():
    """Norms, rotation, store and attention in one path: the new row against
    64-bit attention over what the pages hold (rounded to BF16 as they are read
    back, 2^-8 of a key or value: the logits move by that of their terms' sizes,
    the output by that of its terms' plus twice what the logits do)."""
    from decode_loop import Decoder, Shape, norm

    s = Shape(layers=1, kind="int4", qk_norm=True)
    model = Decoder(s, slots=2, positions=96)
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    model.prefill([list(range(40)), list(range(7, 60))], lens, chunk=16)
    lens.add_(1)
    layer = model.layers[0]
    x = model.embed(torch.tensor([11, 12], device="cuda")).float() * s.hidden**0.5
    y = layer.qkv.gemv(norm(x)).view(2, -1, s.head_dim)
    q = layer.cache.append(y[:, s.q_heads : s.q_heads + s.kv_heads], y[:, s.q_heads + s.kv_heads :], model.table, lens,
                           q=y[:, : s.q_heads], cos=model.cos, sin=model.sin, q_norm=layer.q_norm, k_norm=layer.k_norm)
    got = layer.cache.attend(q, model.table, lens, softcap=s.attn_softcap)
    keys, values = (t.double() for t in layer.cache.decode())
    for b in range(2):
        n = int(lens[b])
        # the queries as the formula has them: a norm, then pairs (i, i + dim / 2) turned
        z = y[b, : s.q_heads].double()
        z = z / torch.sqrt(z.square().mean(-1, keepdim=True) + 1e-6) * layer.q_norm.double()
        c, sn, half = model.cos[n - 1].double(), model.sin[n - 1].double(), s.head_dim // 2
        turned = torch.cat((z[:, :half] * c - z[:, half:] * sn, z[:, half:] * c + z[:, :half] * sn), -1)
        assert bool(((q[b].double() - turned).abs() <= 2.0**-8 * turned.abs() + 2.0**-20).all())
        pages = model.table[b, : (n + s.page - 1) // s.page].long()
        for h in range(s.q_heads):
            k, v = (t[pages, h * s.kv_heads // s.q_heads].reshape(-1, s.head_dim)[:n] for t in (keys, values))
            row, scale = q[b, h].double(), s.head_dim**-0.5
            logits = k @ row * scale
            p = torch.softmax(s.attn_softcap * torch.tanh(logits / s.attn_softcap), 0)
            moved = 2.0**-8 * scale * (k.abs() @ row.abs()).max()
            want, size = p @ v, p @ v.abs()
            assert bool(((got[b, h].double() - want).abs() <= 2.0**-8 * want.abs() + (2.0**-8 + 2.0**-9 + 2 * moved) * size + 1e-6).all())


def test_the_4_bit_kernel_files_compile_by_themselves(tmp_path):
    runs = [(name, subprocess.Popen([_build.nvcc_path(), "-std=c++17", "-gencode", _build.GENCODE, "--cuda", "-o",
                                     str(tmp_path / f"{name}.ii"), str(_build.PACKAGE_DIR / "csrc" / name)],
                                    stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
            for name in ("se12_kv4.cu", "se12_attend4.cu")]
    for name, run in runs:
        output, _ = run.communicate()
        assert run.returncode == 0, f"{name}:\n{output}"
