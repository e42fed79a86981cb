"""A paged key/value cache in 8 or 4 bits, and attention over it.

``PagedKvCache`` holds one layer's keys and values as 8-bit codes (int8 or
e4m3) with one fp32 scale per block (a page of one KV head), or as 4-bit codes
with a scale and an offset per token and 64 dimensions. ``append`` stores a
step's new keys and values, normalised and rotated to their positions, and does
the same to the queries in the same pass; ``attend`` is the attention of those queries
over the sequences' pages; ``decode`` reads pages back as BF16. They take the
grouped q/k/v GEMV's fp32 output as it is and give the BF16 rows the o
projection's GEMV takes, so that a decode step is

    y = qkv.gemv(x).view(tokens, q_heads + 2 * kv_heads, head_dim)
    q = cache.append(y[:, q_heads:-kv_heads], y[:, -kv_heads:], table, lens, q=y[:, :q_heads], cos=cos, sin=sin)
    x = o_proj.gemv(cache.attend(q, table, lens).view(tokens, -1))

Lengths and page tables are read on the device: a captured CUDA graph follows
their contents. The caller owns the pages (which sequence has which, when one
is copied or given back); two sequences of one call must not append to the
same page. Everything runs in kernels of libse12_b200 on the current torch
stream; nothing here has a CPU path.
"""

from __future__ import annotations

import ctypes
import math
import weakref

import torch

from . import _lib
from .device import _WorkspacePool

KINDS = {"int8": 0, "e4m3": 1, "int4": 4}
INT4_GROUP = 64  # dimensions that share a scale and an offset in 4 bits
INT4_HEAD_DIMS = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_SEQS = 2048
COUNTER_BYTES = 4096  # SE12_COUNTER_BYTES: the part of a workspace that must be zero before a call

_INT_MAX = 2**31 - 1
_FLOATS = (torch.float32, torch.bfloat16)
_BF16 = (torch.bfloat16,)

_WORKSPACES = _WorkspacePool()


def _workspace(pool: _WorkspacePool, device: torch.device, stream: int, nbytes: int) -> int:
    """Address of a workspace for this call, its counters zero; ``device`` is
    the current one. While a graph is captured it belongs to the graph (the
    clearing is captured with it); otherwise it is the stream's, which every
    call leaves zeroed."""
    if torch.cuda.is_current_stream_capturing():
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        buf[:COUNTER_BYTES].zero_()
        return buf.data_ptr()
    return pool.get(device, stream, nbytes).data_ptr()


def _launch(device: torch.device, function, name: str, *args, workspace: tuple | None = None) -> None:
    """function(*args, current stream) on the GPU ``device``; with ``workspace``
    (pool, bytes) function(*args, workspace, bytes, current stream), the
    workspace prepared on that GPU too."""
    index = device.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return _launch(device, function, name, *args, workspace=workspace)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if workspace is not None:
        pool, nbytes = workspace
        args += (_workspace(pool, device, stream, nbytes), nbytes)
    status = function(*args, stream)
    if status:
        _lib.check(status, name)


def _rows(x: torch.Tensor, name: str, heads: int | None, dim: int, tokens: int | None, dtypes, device) -> torch.Tensor:
    if x.dim() != 3 or x.shape[2] != dim or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{name} must be [tokens, {heads if heads is not None else 'heads'}, {dim}], got {tuple(x.shape)}")
    if tokens is not None and x.shape[0] != tokens:
        raise ValueError(f"{name} has {x.shape[0]} tokens, expected {tokens}")
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {x.dtype}")
    if x.stride(2) != 1:
        raise ValueError(f"{name} must have unit stride in its last dimension")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, the cache on {device}")
    return x


def _index(x: torch.Tensor, name: str, dim: int, device) -> torch.Tensor:
    if x.dtype != torch.int32 or x.dim() != dim:
        raise ValueError(f"{name} must be an int32 tensor of {dim} dimension{'s' if dim > 1 else ''}")
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        raise ValueError(f"{name} must have unit stride in its last dimension")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, the cache on {device}")
    return x


class PagedKvCache:
    """``pages`` pages of ``page_size`` tokens (16, 32, 64, 128 or 256) of
    ``kv_heads`` heads of ``head_dim`` (a multiple of 16 up to 256) values,
    for keys and for values. ``kind``: "int8" (codes of 7 bits and a sign,
    for heads whose values spread evenly), "e4m3" (for wide ranges) or "int4"
    (4.6 bits a value with the scales; head_dim 64, 128 or 256).

    ``k_codes`` and ``v_codes`` are [pages, kv_heads, page_size, head_dim]
    int8 tensors (e4m3: the bit patterns), ``k_scales`` and ``v_scales`` [pages,
    kv_heads] fp32; a value is code * scale.

    "int4" quantises every token of a head by itself, in groups of 64
    dimensions: a value is (u - 8) * scale + offset, u its code 0..15.
    ``k_codes`` and ``v_codes`` are uint8 [pages, kv_heads, page_size,
    head_dim / 2]: words of 8 codes, the first in the lowest bits, word 8 g + r
    of a row at place r * groups + g. ``k_scales`` is fp16 [pages, kv_heads,
    page_size, groups, 2] (scale, offset); ``v_scales`` fp16 [pages, kv_heads,
    page_size / 16, 32 * groups + 16]: of 16 tokens, for each two neighbours
    the groups' scales and then their offsets (the two tokens' side by side),
    then a whole number E per token, -30 to 30: its values are 2^E times what
    scale and offset give. E is NaN for a token whose values are not finite or
    reach 2^34, a key group's scale and offset where it is not finite or passes
    65000. Keys have no E: a group whose values differ by less than 2^-10 keeps
    fewer bits, by less than 2^-21 its offset alone, and offsets end at 2^-24.

    Attention takes any scales and offsets (``from_tensors``) with which every
    code's (u - 8) * scale + offset is in FP16's range, values' scales below 128;
    those of hidden values have to be finite too."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, kind: str = "int8", device="cuda"):
        self._check(pages, page_size, kv_heads, head_dim, kind)
        device = torch.device(device)
        if kind == "int4":
            groups = head_dim // INT4_GROUP
            codes = (pages, kv_heads, page_size, head_dim // 2)
            self._adopt(torch.zeros(codes, dtype=torch.uint8, device=device), torch.zeros(codes, dtype=torch.uint8, device=device),
                        torch.zeros(pages, kv_heads, page_size, groups, 2, dtype=torch.float16, device=device),
                        torch.zeros(pages, kv_heads, page_size // 16, 32 * groups + 16, dtype=torch.float16, device=device), kind)
            return
        shape = (pages, kv_heads, page_size, head_dim)
        self._adopt(torch.zeros(shape, dtype=torch.int8, device=device), torch.zeros(shape, dtype=torch.int8, device=device),
                    torch.ones(shape[:2], dtype=torch.float32, device=device),
                    torch.ones(shape[:2], dtype=torch.float32, device=device), kind)

    @staticmethod
    def _check(pages, page_size, kv_heads, head_dim, kind) -> None:
        if kind not in KINDS:
            raise ValueError(f"kind must be one of {tuple(KINDS)}, got {kind!r}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if pages < 1 or kv_heads < 1:
            raise ValueError("pages and kv_heads must be positive")
        if kind == "int4":
            if head_dim not in INT4_HEAD_DIMS:
                raise ValueError(f"head_dim must be one of {INT4_HEAD_DIMS} in 4 bits, got {head_dim}")
        elif head_dim < 16 or head_dim > 256 or head_dim % 16:
            raise ValueError(f"head_dim must be a multiple of 16 up to 256, got {head_dim}")

    @classmethod
    def from_tensors(cls, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
                     kind: str = "int8") -> "PagedKvCache":
        """A cache over existing contiguous tensors (used in place, not copied).
        e4m3 codes are finite ones (append writes no others): attention multiplies
        a hidden token's values by a weight of zero."""
        if k_codes.dim() != 4 or k_codes.shape != v_codes.shape:
            raise ValueError("codes must be [pages, kv_heads, page_size, head_dim], the same for keys and values")
        pages, heads, page_size, dim = k_codes.shape
        dim *= 2 if kind == "int4" else 1
        cls._check(pages, page_size, heads, dim, kind)
        for t in (k_codes, v_codes):
            if t.dtype not in (torch.int8, torch.uint8, torch.float8_e4m3fn) or not t.is_contiguous():
                raise ValueError("codes must be contiguous 8-bit tensors")
        if kind == "int4":
            groups = dim // INT4_GROUP
            for t, name, shape in ((k_scales, "k_scales", (pages, heads, page_size, groups, 2)),
                                   (v_scales, "v_scales", (pages, heads, page_size // 16, 32 * groups + 16))):
                if t.dtype != torch.float16 or tuple(t.shape) != shape or not t.is_contiguous():
                    raise ValueError(f"{name} must be a contiguous fp16 tensor of shape {shape}, got {tuple(t.shape)}")
        else:
            for t in (k_scales, v_scales):
                if t.dtype != torch.float32 or tuple(t.shape) != (pages, heads) or not t.is_contiguous():
                    raise ValueError("scales must be contiguous fp32 [pages, kv_heads] tensors")
        if any(t.device != k_codes.device for t in (v_codes, k_scales, v_scales)):
            raise ValueError("codes and scales must be on one device")
        self = cls.__new__(cls)
        self._adopt(k_codes, v_codes, k_scales, v_scales, kind)
        return self

    def _adopt(self, k_codes, v_codes, k_scales, v_scales, kind) -> None:
        lib = _lib.load()
        self.k_codes, self.v_codes, self.k_scales, self.v_scales, self.kind = k_codes, v_codes, k_scales, v_scales, kind
        self.pages, self.kv_heads, self.page_size, self.head_dim = k_codes.shape
        if kind == "int4":
            self.head_dim *= 2
        self.device = k_codes.device
        s = _lib.Se12KvPagesStruct(self.pages, self.page_size, self.kv_heads, self.head_dim, KINDS[kind], k_codes.data_ptr(),
                                   v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr())
        handle = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            _lib.check(lib.se12_kv_cache_create(ctypes.byref(s), ctypes.byref(handle)), "se12_kv_cache_create")
        self._handle = handle
        self._finalizer = weakref.finalize(self, lib.se12_kv_cache_destroy, handle)
        self._lib = lib

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._handle

    # The checks of a call that is right cost as little as they can (a decode
    # step makes one such call per layer and operator); the functions that say
    # what is wrong are only called where something is.
    def _batch(self, tokens: int, block_table, lens, query_start) -> bytes:
        shape, stride, device = block_table.shape, block_table.stride(), self.device
        seqs = lens.numel()
        if not (block_table.dtype is torch.int32 and lens.dtype is torch.int32 and len(shape) == 2 and lens.dim() == 1
                and shape[0] == seqs and shape[1] >= 1 and (stride[1] == 1 or shape[1] == 1)
                and (seqs == 1 or lens.stride(0) == 1) and block_table.device == device and lens.device == device
                and 1 <= seqs <= MAX_SEQS):
            self._refuse_batch(block_table, lens)
        start = 0
        if query_start is None:
            if tokens != seqs:
                raise ValueError(f"without query_start there is one token per sequence: {tokens} tokens, {seqs} sequences")
        else:
            _index(query_start, "query_start", 1, device)
            if query_start.shape[0] != seqs + 1:
                raise ValueError(f"query_start must have {seqs + 1} entries, got {query_start.shape[0]}")
            start = query_start.data_ptr()
        return _lib.KV_BATCH.pack(seqs, tokens, lens.data_ptr(), start, block_table.data_ptr(), stride[0], shape[1])

    def _refuse_batch(self, block_table, lens) -> None:
        _index(block_table, "block_table", 2, self.device)
        _index(lens, "lens", 1, self.device)
        seqs = lens.shape[0]
        if block_table.shape[0] != seqs or block_table.shape[1] < 1:
            raise ValueError(f"block_table must have a row per sequence ({seqs}) and a column or more, got {tuple(block_table.shape)}")
        raise ValueError(f"1..{MAX_SEQS} sequences, got {seqs}")

    def _row_strides(self, x: torch.Tensor, name: str, heads: int | None, tokens: int | None, dtypes) -> tuple:
        """Token and head stride of [tokens, heads, head_dim] rows."""
        shape, stride = x.shape, x.stride()
        if (len(shape) == 3 and shape[2] == self.head_dim and (heads is None or shape[1] == heads)
                and (tokens is None or shape[0] == tokens) and x.dtype in dtypes and stride[2] == 1 and x.device == self.device):
            return stride[0], stride[1]
        _rows(x, name, heads, self.head_dim, tokens, dtypes, self.device)
        return stride[0], stride[1]

    def _norm_weight(self, w: torch.Tensor | None, name: str) -> tuple:
        if w is None:
            return 0, False
        if w.dim() != 1 or w.shape[0] != self.head_dim or w.dtype not in _FLOATS or w.stride(0) != 1 or w.device != self.device:
            raise ValueError(f"{name} must be fp32 or BF16 [{self.head_dim}] on {self.device}, with unit stride")
        return w.data_ptr(), w.dtype is torch.bfloat16

    # ------------------------------------------------------------------ operators
    def append(self, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
               q: torch.Tensor | None = None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
               query_start: torch.Tensor | None = None, interleaved: bool = False,
               q_out: torch.Tensor | None = None, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
               norm_eps: float = 1e-6) -> torch.Tensor | None:
        """Stores new keys and values (fp32 or BF16 [tokens, kv_heads,
        head_dim], any token and head strides) and returns the queries q
        [tokens, q_heads, head_dim] rotated, as BF16 (None without q).

        ``lens`` [seqs] counts the tokens of each sequence with the new ones,
        which are its last; ``query_start`` [seqs + 1] says where each
        sequence's rows begin (None: one row per sequence). ``block_table``
        [seqs, columns] (any row stride) holds page ids. A sequence with ``lens`` 0 is a padding
        row: nothing is stored, its queries are zeros. ``cos`` and ``sin``
        (fp32 [positions, rotary / 2]) rotate keys and queries by position,
        pairs (i, i + rotary / 2), or (2i, 2i + 1) when ``interleaved``.
        ``q_norm`` and ``k_norm`` (fp32 or BF16 [head_dim] weights) normalise
        each head's queries or keys before that: x / sqrt(mean(x^2) +
        ``norm_eps``) * weight, in fp32 (the mean from 64-bit sums) without a
        rounding in between. (Of a checkpoint whose norms multiply by 1 + w the
        caller passes 1 + w.)"""
        dtype = k.dtype
        k_strides = self._row_strides(k, "k", self.kv_heads, None, _FLOATS)
        tokens = k.shape[0]
        v_strides = self._row_strides(v, "v", self.kv_heads, tokens, (dtype,))
        q_ptr, q_heads, q_strides, out_ptr, out_strides = 0, 0, (0, 0), 0, (0, 0)
        if q is not None:
            q_strides = self._row_strides(q, "q", None, tokens, (dtype,))
            q_heads = q.shape[1]
            if q_heads < 1:
                raise ValueError("q has no heads")
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=torch.bfloat16, device=self.device)
                out_strides = (q_heads * self.head_dim, self.head_dim)
            else:
                out_strides = self._row_strides(q_out, "q_out", q_heads, tokens, _BF16)
            q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        norms = None
        if q_norm is not None or k_norm is not None:
            if q_norm is not None and q is None:
                raise ValueError("q_norm without q")
            if not 0.0 <= norm_eps < math.inf:
                raise ValueError(f"norm_eps must be finite and not negative, got {norm_eps}")
            (q_weight, q_bf16), (k_weight, k_bf16) = self._norm_weight(q_norm, "q_norm"), self._norm_weight(k_norm, "k_norm")
            norms = _lib.KV_NORMS.pack(q_weight, k_weight, q_bf16, k_bf16, norm_eps)
        if tokens == 0:
            return q_out
        batch = self._batch(tokens, block_table, lens, query_start)
        turn = (0, 0, 0, 0, 0)
        if cos is not None and sin is not None:
            shape, stride = cos.shape, cos.stride()
            if not (cos.dtype is torch.float32 and sin.dtype is torch.float32 and len(shape) == 2 and sin.shape == shape
                    and stride[1] == 1 and sin.stride() == stride and cos.device == self.device and sin.device == self.device
                    and 1 <= shape[1] <= self.head_dim // 2 and shape[0] >= 1):
                raise ValueError(f"cos and sin must be fp32 [positions, 1..{self.head_dim // 2}] tensors on {self.device} with the "
                                 "same shape and strides and unit column stride")
            turn = (cos.data_ptr(), sin.data_ptr(), stride[0], shape[0], 2 * shape[1])
        elif cos is not None or sin is not None:
            raise ValueError("cos and sin go together")
        args = _lib.KV_APPEND.pack(dtype is torch.bfloat16, q_heads, q_ptr, k.data_ptr(), v.data_ptr(), *q_strides, *k_strides,
                                   *v_strides, *turn, bool(interleaved), out_ptr, *out_strides)
        if norms is None:
            _launch(self.device, self._lib.se12_kv_append, "se12_kv_append", self._handle, batch, args)
        else:
            _launch(self.device, self._lib.se12_kv_append_normed, "se12_kv_append_normed", self._handle, batch, args, norms)
        return q_out

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, query_start: torch.Tensor | None = None,
               max_query: int | None = None, scale: float | None = None, softcap: float = 0.0, window: int = 0,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the rows q (BF16 [tokens, q_heads, head_dim]) over
        their sequences; batch arguments as for ``append``. Causal: a row at
        position p sees positions up to p, with ``window`` only the last
        ``window`` of them; page table entries below the first position that a
        sequence's rows see are not read (those pages may have been given
        back). Logits are ``scale`` (default head_dim ** -0.5) q . k, with
        ``softcap`` > 0 then softcap * tanh(logit / softcap). Rows that see
        nothing are zero; rows of ``out`` that ``query_start`` gives to no
        sequence are left as they are. ``max_query``: the most rows of one
        sequence (default: all tokens; tells the launch how many rows share a page).
        Returns BF16 like q."""
        q_strides = self._row_strides(q, "q", None, None, _BF16)
        tokens, q_heads, _ = q.shape
        if q_heads < 1 or q_heads % self.kv_heads:
            raise ValueError(f"q has {q_heads} heads, not a multiple of the cache's {self.kv_heads}")
        if out is None:
            out = torch.empty(q.shape, dtype=torch.bfloat16, device=self.device)
            out_strides = (q_heads * self.head_dim, self.head_dim)
        else:
            out_strides = self._row_strides(out, "out", q_heads, tokens, _BF16)
        if tokens == 0:
            return out
        batch = self._batch(tokens, block_table, lens, query_start)
        if max_query is None:
            max_query = 1 if query_start is None else tokens
        max_query = min(int(max_query), _INT_MAX)
        args = _lib.KV_ATTEND.pack(q.data_ptr(), *q_strides, out.data_ptr(), *out_strides, q_heads, max_query, min(int(window), _INT_MAX),
                                   self.head_dim ** -0.5 if scale is None else scale, softcap)
        need = self._lib.se12_kv_attend_call_bytes(self._handle, q_heads, max_query)
        _launch(self.device, self._lib.se12_kv_attend, "se12_kv_attend", self._handle, batch, args, workspace=(_WORKSPACES, need))
        return out

    def decode(self, pages: torch.Tensor | None = None) -> tuple:
        """Keys and values of the given pages (int32 ids; None: all) as BF16
        tensors [pages, kv_heads, page_size, head_dim], exact (int4: rounded)."""
        count = self.pages if pages is None else _index(pages, "pages", 1, self.device).shape[0]
        shape = (count, self.kv_heads, self.page_size, self.head_dim)
        k = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        v = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        if count:
            _launch(self.device, self._lib.se12_kv_decode, "se12_kv_decode", self._handle,
                    None if pages is None else pages.data_ptr(), count, k.data_ptr(), v.data_ptr())
        return k, v


__all__ = ["KINDS", "MAX_SEQS", "PAGE_SIZES", "PagedKvCache"]
