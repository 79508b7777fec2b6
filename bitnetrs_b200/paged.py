"""The quantised paged key-value cache on the device: rows quantised into it,
rows read back, and attention over it.

:class:`PagedKV` describes a cache in device memory (the caller's own, or one
layer of a :class:`~bitnetrs_b200.model.KVCache`) and has one method for each
of the ``bitnet_cuda_kv_*_device`` entry points of ``include/bitnet_cuda.h``,
which also states the cache's layout.  As in ``decode_step_device``, tensors
are device addresses (e.g. torch ``data_ptr()``) and ``stream`` is a
``cudaStream_t``: 0 selects the context's own stream, and 1 is CUDA's name for
the legacy default stream (the one torch calls 0).  Calls return without
synchronising.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

from . import _native as N
from ._native import check
from .backend import CudaBackend

KV_I8 = 2
KV_I4 = 3
STATUS_NON_FINITE = 1
STATUS_BAD_CONTEXT = 4
STATUS_WAIT_TIMEOUT = 8


class PagedKV:
    """A paged cache of 8- or 4-bit keys and values (bitnet_cuda_kv_pages)."""

    def __init__(self, backend: CudaBackend, pool: int, page_table: int, *, pages: int, seqs: int, pages_per_seq: int,
                 kv_heads: int, head_dim: int, kv_dtype: int):
        self._init(backend, N.KvPages(pool, page_table, pages, seqs, pages_per_seq, kv_heads, head_dim, kv_dtype))

    def _init(self, backend, pages, owner=None):
        self.backend = backend
        self._lib = N.cuda_lib()
        self._pages = pages
        self._ref = C.byref(pages)
        self._kv_width = pages.kv_heads * pages.head_dim
        self._owner = owner  # keeps a model's cache alive
        self._store = self._lib.bitnet_cuda_kv_store_device
        self._load = self._lib.bitnet_cuda_kv_load_device
        self._attention = self._lib.bitnet_cuda_kv_attention_device
        self._prompt = self._lib.bitnet_cuda_kv_prompt_attention_device

    @classmethod
    def of_layer(cls, kv, layer: int) -> "PagedKV":
        """One layer of a model's quantised cache (bitnet_cuda_kv_layer_pages)."""
        pages = N.KvPages()
        check(N.cuda_lib().bitnet_cuda_kv_layer_pages(kv.handle, layer, C.byref(pages)))
        self = cls.__new__(cls)
        self._init(kv.model.backend, pages, kv)
        return self

    @staticmethod
    def block_bytes(kv_dtype: int, head_dim: int) -> int:
        """Bytes of one page of one kv head; a pool holds pages * kv_heads of them."""
        n = C.c_size_t()
        check(N.cuda_lib().bitnet_cuda_kv_block_bytes(kv_dtype, head_dim, C.byref(n)))
        return n.value

    def store(self, k: int, v: int, rows: int, row_seq: int, row_pos: int, status: int, *, ldk: Optional[int] = None,
              ldv: Optional[int] = None, bf16: bool = False, rope: Optional[Tuple[int, int, int]] = None,
              stream: int = 0) -> None:
        """Quantise ``rows`` rows of K and V (f32, or bf16) into positions ``row_pos`` of sequences ``row_seq``
        (device int32 arrays).  ``rope`` = (cos, sin, length): K is rotated first."""
        cos, sin, length = rope if rope is not None else (None, None, 0)
        w = self._kv_width
        code = self._store(
            self.backend._h, self._ref, k, w if ldk is None else ldk, v, w if ldv is None else ldv,
            int(bf16), rows, row_seq, row_pos, cos, sin, length, status, stream or None)
        if code:
            check(code)

    def load(self, k: int, v: int, rows: int, row_seq: int, row_pos: int, status: int, *, ldk: Optional[int] = None,
             ldv: Optional[int] = None, bf16: bool = False, stream: int = 0) -> None:
        """Read rows back into ``k`` and ``v``."""
        w = self._kv_width
        code = self._load(
            self.backend._h, self._ref, rows, row_seq, row_pos, k, w if ldk is None else ldk, v,
            w if ldv is None else ldv, int(bf16), status, stream or None)
        if code:
            check(code)

    def attention_workspace(self, n_heads: int) -> int:
        """Bytes of the workspace that one attention call in flight needs."""
        n = C.c_size_t()
        check(self._lib.bitnet_cuda_kv_attention_workspace(self._ref, n_heads, C.byref(n)))
        return n.value

    def attention(self, q: int, out: int, rows: int, n_heads: int, row_seq: int, row_len: int, max_len: int,
                  workspace: int, workspace_bytes: int, status: int, *, ldq: Optional[int] = None,
                  ldo: Optional[int] = None, bf16: bool = False, lse: int = 0, stream: int = 0) -> None:
        """Attention of single tokens: row r sees the first ``row_len[r]`` positions of sequence ``row_seq[r]``."""
        w = n_heads * self._pages.head_dim
        code = self._attention(
            self.backend._h, self._ref, q, w if ldq is None else ldq, int(bf16), rows, n_heads,
            row_seq, row_len, max_len, out, w if ldo is None else ldo, lse or None, workspace, workspace_bytes, status,
            stream or None)
        if code:
            check(code)

    def prompt_attention(self, q: int, out: int, rows: int, n_heads: int, n_seqs: int, seq_ids: int, cu_rows: int,
                         starts: int, max_len: int, workspace: int, workspace_bytes: int, status: int, *,
                         ldq: Optional[int] = None, ldo: Optional[int] = None, bf16: bool = False, lse: int = 0,
                         stream: int = 0) -> None:
        """Causal attention of prompts whose K and V are in the cache: rows ``cu_rows[i]`` to ``cu_rows[i + 1]`` are
        the positions from ``starts[i]`` of sequence ``seq_ids[i]``."""
        w = n_heads * self._pages.head_dim
        code = self._prompt(
            self.backend._h, self._ref, q, w if ldq is None else ldq, int(bf16), rows, n_heads, n_seqs,
            seq_ids, cu_rows, starts, max_len, out, w if ldo is None else ldo, lse or None, workspace,
            workspace_bytes, status, stream or None)
        if code:
            check(code)
