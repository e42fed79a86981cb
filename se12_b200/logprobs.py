"""Log probabilities of chosen tokens from the LM head's logits.

``token_logprobs`` takes rows of logits as the LM head leaves them (the fused
GEMV's fp32 output, or the exact mode's BF16) and gives, in one pass over
them, each row's log probability of a given token, its entropy and its top
alternatives: what a server returns beside the tokens it sampled, and what
scoring a prompt needs. The kernel is libse12_b200's; nothing here has a CPU
path.
"""

from __future__ import annotations

import typing

import torch

from . import _lib
from .device import _WorkspacePool
from .kv_cache import _launch

MAX_TOP = 32

_WORKSPACES = _WorkspacePool()


class TokenLogprobs(typing.NamedTuple):
    logprob: torch.Tensor       # fp32 [rows]
    entropy: torch.Tensor       # fp32 [rows], in nats
    top_ids: torch.Tensor       # int64 [rows, top], most likely first, ties to the lowest id
    top_logprobs: torch.Tensor  # fp32 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, softcap: float = 0.0) -> TokenLogprobs:
    """``logits``: fp32 or BF16 [rows, vocab] (any row stride: an expanded row
    is read as it is, rows that overlap are copied), ``tokens``: int64 [rows] ids; a negative id asks for none (its log probability is
    NaN), one past the vocabulary is NaN too and sets the device status.
    ``top``: alternatives per row, up to 32. ``softcap`` > 0 caps the logits
    (softcap * tanh(x / softcap)) first, -inf (a banned token) staying -inf."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("logits must be an fp32 or BF16 [rows, vocab] tensor")
    rows, vocab = logits.shape
    if vocab < 1 or logits.stride(1) != 1:
        raise ValueError("logits need a column or more and unit column stride")
    if tokens.dtype != torch.int64 or tokens.dim() != 1 or tokens.shape[0] != rows:
        raise ValueError(f"tokens must be an int64 tensor of {rows} ids")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be in 0..{min(MAX_TOP, vocab)}, got {top}")
    if not 0.0 <= softcap < 1e30:
        raise ValueError(f"softcap must be finite and not negative, got {softcap}")
    device = logits.device
    if device.type != "cuda" or tokens.device != device:
        raise ValueError("logits and tokens must be on one GPU")
    if tokens.stride(0) != 1 and rows > 1:
        tokens = tokens.contiguous()
    if rows > 1 and 0 < logits.stride(0) < vocab:
        logits = logits.contiguous()
    ld = logits.stride(0) if rows > 1 else vocab
    logprob = torch.empty(rows, dtype=torch.float32, device=device)
    entropy = torch.empty(rows, dtype=torch.float32, device=device)
    ids = torch.empty(rows, top, dtype=torch.int64, device=device)
    top_logprobs = torch.empty(rows, top, dtype=torch.float32, device=device)
    if rows:
        lib = _lib.load()
        need = lib.se12_token_logprobs_workspace_bytes()
        _launch(device, lib.se12_token_logprobs, "se12_token_logprobs", logits.data_ptr(), logits.dtype == torch.bfloat16, rows,
                vocab, ld, tokens.data_ptr(), top, softcap, logprob.data_ptr(), entropy.data_ptr(),
                ids.data_ptr(), top_logprobs.data_ptr(), workspace=(_WORKSPACES, need))
    return TokenLogprobs(logprob, entropy, ids, top_logprobs)


__all__ = ["MAX_TOP", "TokenLogprobs", "token_logprobs"]
