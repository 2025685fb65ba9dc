"""The 4-bit paged K/V cache and the attention that reads it, on top of the C ABI
(``b2_kv4_cache`` in ``include/riftco_b200.h``, where the format is defined).

``PagedKv4Pool`` is to this cache what ``PagedKvPool`` is to the FP32 one; exceptions
follow ``backend.py``. All tensors live on the current CUDA device; calls only enqueue
work on ``stream`` (default: torch's current stream) and report device-side errors in
``status`` (int32 [1], zeroed by the caller; ``_lib.ATTN_STATUS_*``).
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field

import torch

from . import _lib
from ._lib import Kv4CacheStruct, Kv4ScoreRulesStruct, lib
from .backend import _check, _stream_ptr

__all__ = ("PagedKv4Pool", "dequantize_kv4", "paged_chunk_attention_kv4", "paged_chunk_kv4_workspace_bytes",
           "paged_decode_attention_kv4", "paged_decode_kv4_workspace_bytes", "rope_append_kv4")

_INTS = (torch.int32, torch.uint32)
HEAD_WIDTHS = (64, 128, 256)


# Two of torch's own accessors without their wrappers, where this torch has them: a torch.cuda.Stream object for the
# current stream takes 3.7 us to build and its raw handle 0.1 us, a third of what a small call costs the host.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream(stream, device: int) -> int:
    if stream is None and _raw_stream is not None:
        return _raw_stream(device)
    return _stream_ptr(stream)


def _need(t, what: str, dtypes, shape, device: int) -> int:
    """The data pointer of a contiguous tensor of this type and shape on CUDA device `device`; raises
    otherwise."""
    if not isinstance(t, torch.Tensor) or t.get_device() != device:
        raise ValueError(f"{what} storage does not match its backend")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}")
    if t.shape != shape:
        raise RuntimeError(f"{what} storage size does not match dimensions")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return t.data_ptr()


_F32 = (torch.float32,)


def _u32(value: int, what: str) -> int:
    """`value`, which a uint32 of the C ABI has to hold: ctypes would pass on the lower half of a larger one."""
    if not 0 <= value <= 0xFFFFFFFF:
        raise ValueError(f"paged attention {what} must be between 0 and 2**32 - 1, got {value}")
    return value


@dataclass
class PagedKv4Pool:
    """One layer's 4-bit K/V pages: ``pages`` uint8 [physical_blocks, kv_heads,
    block_size / 16, 18 * head_width]."""

    pages: torch.Tensor
    block_size: int
    head_width: int
    device_index: int = field(init=False, repr=False, compare=False)   # -1: not on a GPU

    def __post_init__(self) -> None:
        if self.head_width not in HEAD_WIDTHS:
            raise ValueError(f"4-bit cache head width must be 64, 128 or 256, got {self.head_width}")
        if self.block_size <= 0 or self.block_size % 16 != 0:
            raise ValueError(f"4-bit cache block size must be a multiple of 16, got {self.block_size}")
        p = self.pages
        if not isinstance(p, torch.Tensor) or p.dtype != torch.uint8 or not p.is_contiguous() or p.dim() != 4:
            raise ValueError("4-bit cache pages must be contiguous uint8 [blocks, heads, block_size / 16, bytes]")
        if p.shape[2] != self.block_size // 16 or p.shape[3] != 18 * self.head_width:
            raise RuntimeError("4-bit cache storage size does not match dimensions")
        self.device_index = p.get_device()

    @classmethod
    def empty(cls, physical_blocks: int, kv_heads: int, block_size: int, head_width: int,
              device="cuda") -> "PagedKv4Pool":
        """A pool whose slots hold nothing yet (uninitialised memory)."""
        pages = torch.empty((physical_blocks, kv_heads, block_size // 16, 18 * head_width), dtype=torch.uint8,
                            device=device)
        return cls(pages, block_size, head_width)

    @property
    def physical_blocks(self) -> int:
        return self.pages.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.pages.shape[1]

    def bytes_per_token(self) -> int:
        """Bytes one token of a sequence takes in this layer."""
        return self.kv_heads * 18 * self.head_width // 16

    def struct(self, block_tables: torch.Tensor) -> Kv4CacheStruct:
        device = self.device_index
        if device < 0 or device != _current_device():
            raise ValueError("4-bit cache pages must be on the current CUDA device")
        dims = block_tables.shape
        if len(dims) != 2:
            raise ValueError("block tables must be [sequences, blocks]")
        tables = _need(block_tables, "block table", _INTS, dims, device)
        blocks, heads, _, _ = self.pages.shape
        return Kv4CacheStruct(self.pages.data_ptr(), tables, blocks, dims[0], dims[1], heads, self.head_width,
                              self.block_size, 0)


def _token_args(pool, block_tables, positions, token_seq):
    n = positions.shape[0]
    device = pool.device_index
    pos = _need(positions, "positions", _INTS, (n,), device)
    owner = None if token_seq is None else _need(token_seq, "token sequences", _INTS, (n,), device)
    if token_seq is None and n != block_tables.shape[0]:
        raise ValueError("without token sequences every sequence contributes one token")
    return n, pos, owner


def _status_ptr(status, device):
    return None if status is None else _need(status, "status", _INTS, (1,), device)


def rope_append_kv4(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, positions: torch.Tensor,
                    pool: PagedKv4Pool, block_tables: torch.Tensor, theta: float,
                    token_seq: torch.Tensor | None = None, queries_out: torch.Tensor | None = None,
                    status: torch.Tensor | None = None, stream=None) -> None:
    """Rotates queries [n, q_heads, d] (into ``queries_out``, default in place) and keys
    [n, kv_heads, d] at ``positions`` [n] and stores keys and values in the cache: token t in
    sequence ``token_seq[t]``, or in sequence t without ``token_seq``."""
    cache = pool.struct(block_tables)
    device, d = pool.device_index, pool.head_width
    n, pos, owner = _token_args(pool, block_tables, positions, token_seq)
    if queries.dim() != 3:
        raise ValueError("queries must be [tokens, heads, head width]")
    hq = queries.shape[1]
    q = _need(queries, "queries", _F32, (n, hq, d), device)
    out = q if queries_out is None else _need(queries_out, "rotated queries", _F32, (n, hq, d), device)
    k = _need(keys, "keys", _F32, (n, pool.kv_heads, d), device)
    v = _need(values, "values", _F32, (n, pool.kv_heads, d), device)
    _check(lib.b2_rope_append_kv4(C.byref(cache), q, out, k, v, pos, owner, n, hq, theta,
                                  _status_ptr(status, device), _stream(stream, device)))


def dequantize_kv4(pool: PagedKv4Pool, block_tables: torch.Tensor, positions: torch.Tensor, keys_out: torch.Tensor,
                   values_out: torch.Tensor, token_seq: torch.Tensor | None = None,
                   status: torch.Tensor | None = None, stream=None) -> None:
    """The stored keys and values of the given tokens, as FP32 [n, kv_heads, d]."""
    cache = pool.struct(block_tables)
    device = pool.device_index
    n, pos, owner = _token_args(pool, block_tables, positions, token_seq)
    shape = (n, pool.kv_heads, pool.head_width)
    k = _need(keys_out, "keys", _F32, shape, device)
    v = _need(values_out, "values", _F32, shape, device)
    _check(lib.b2_kv4_dequantize(C.byref(cache), pos, owner, n, k, v, _status_ptr(status, device),
                                 _stream(stream, device)))


def _rules(softcap, window, alibi_slopes, q_heads, device):
    if not softcap and not window and alibi_slopes is None:
        return None
    if softcap != 0 and not 1e-6 <= softcap <= 1e18:   # here too: one below FP32's range would become 0, no cap
        raise ValueError(f"paged attention score cap must be 0 or between 1e-6 and 1e18, got {softcap}")
    _u32(window, "window")
    slopes = None if alibi_slopes is None else _need(alibi_slopes, "slopes", _F32, (q_heads,), device)
    return C.byref(Kv4ScoreRulesStruct(softcap, window, slopes))


def _workspace(workspace, device):
    if workspace is None:
        return None, 0
    if workspace.get_device() != device or not workspace.is_contiguous():
        raise ValueError("workspace storage does not match its backend")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def paged_decode_kv4_workspace_bytes(n_seq: int, q_heads: int, kv_heads: int, head_width: int,
                                     max_seq_len: int) -> int:
    return lib.b2_paged_decode_kv4_workspace_bytes(_u32(n_seq, "sequences"), _u32(q_heads, "query heads"),
                                                   _u32(kv_heads, "KV heads"), _u32(head_width, "head width"),
                                                   _u32(max_seq_len, "max_seq_len"))


def paged_decode_attention_kv4(queries: torch.Tensor, pool: PagedKv4Pool, block_tables: torch.Tensor,
                               seq_lens: torch.Tensor, context: torch.Tensor | None, max_seq_len: int, *,
                               softcap: float = 0.0, window: int = 0, alibi_slopes: torch.Tensor | None = None,
                               context_bf16: torch.Tensor | None = None, status: torch.Tensor | None = None,
                               workspace: torch.Tensor | None = None, stream=None) -> None:
    """One query token per sequence: queries [n_seq, q_heads, d] FP32, ``context`` the same (None
    where only ``context_bf16`` is wanted), seq_lens [n_seq] the lengths with the new token."""
    _u32(max_seq_len, "max_seq_len")
    cache = pool.struct(block_tables)
    device = pool.device_index
    if queries.dim() != 3:
        raise ValueError("queries must be [sequences, heads, head width]")
    n, hq = block_tables.shape[0], queries.shape[1]
    shape = (n, hq, pool.head_width)
    q = _need(queries, "paged decode attention query", _F32, shape, device)
    ctx = None if context is None else _need(context, "paged decode attention context", _F32, shape, device)
    ctx16 = None if context_bf16 is None else _need(context_bf16, "paged decode attention context",
                                                    (torch.bfloat16,), shape, device)
    lens = _need(seq_lens, "sequence lengths", _INTS, (n,), device)
    rules = _rules(softcap, window, alibi_slopes, hq, device)
    ws, ws_bytes = _workspace(workspace, device)
    _check(lib.b2_paged_decode_attention_kv4(C.byref(cache), rules, q, lens, ctx, ctx16, hq, max_seq_len, ws, ws_bytes,
                                             _status_ptr(status, device), _stream(stream, device)))


def paged_chunk_kv4_workspace_bytes(n_seq: int, n_tokens: int, q_heads: int, kv_heads: int, head_width: int,
                                    max_chunk: int, max_seq_len: int) -> int:
    return lib.b2_paged_chunk_kv4_workspace_bytes(_u32(n_seq, "sequences"), _u32(n_tokens, "tokens"),
                                                  _u32(q_heads, "query heads"), _u32(kv_heads, "KV heads"),
                                                  _u32(head_width, "head width"), _u32(max_chunk, "max_chunk"),
                                                  _u32(max_seq_len, "max_seq_len"))


def paged_chunk_attention_kv4(queries: torch.Tensor, pool: PagedKv4Pool, block_tables: torch.Tensor,
                              seq_lens: torch.Tensor, chunk_starts: torch.Tensor, context_bf16: torch.Tensor,
                              max_chunk: int, max_seq_len: int, *, softcap: float = 0.0, window: int = 0,
                              alibi_slopes: torch.Tensor | None = None, prefix_lens: torch.Tensor | None = None,
                              status: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                              stream=None) -> None:
    """Several new tokens per sequence, already appended: queries [n_tokens, q_heads, d] FP32 and
    ``context_bf16`` the same in bf16, ``chunk_starts`` [n_seq + 1] the first row of each sequence's
    tokens, ``prefix_lens`` [n_seq] how much of a sequence is seen from all of it."""
    _u32(max_chunk, "max_chunk")
    _u32(max_seq_len, "max_seq_len")
    cache = pool.struct(block_tables)
    device = pool.device_index
    if queries.dim() != 3:
        raise ValueError("queries must be [tokens, heads, head width]")
    n_seq, (n, hq, d) = block_tables.shape[0], queries.shape
    shape = (n, hq, pool.head_width)
    q = _need(queries, "paged attention query", _F32, shape, device)
    ctx = _need(context_bf16, "paged attention context", (torch.bfloat16,), shape, device)
    lens = _need(seq_lens, "sequence lengths", _INTS, (n_seq,), device)
    starts = _need(chunk_starts, "chunk starts", _INTS, (n_seq + 1,), device)
    prefix = None if prefix_lens is None else _need(prefix_lens, "prefix lengths", _INTS, (n_seq,), device)
    rules = _rules(softcap, window, alibi_slopes, hq, device)
    ws, ws_bytes = _workspace(workspace, device)
    _check(lib.b2_paged_chunk_attention_kv4(C.byref(cache), rules, prefix, q, lens, starts, ctx, n, hq, max_chunk,
                                            max_seq_len, ws, ws_bytes, _status_ptr(status, device),
                                            _stream(stream, device)))
