"""Key / value cache in 8 bits, in pages that sequences can share, on top of the C ABI's ``tpb_kv_*`` entry points: the counterpart of
the reference's cache and decode attention (src/core/kv_cache.zig, decode kernels of src/gpu/cuda/elt.zig).

A decode step of a model with one cache for all its layers:

    cache.extend(seqs, n_new)                      # once: room for the step's tokens
    for layer in range(layers):
        cache.append(layer, k, v, seqs, cu)        # this layer's new keys and values
        out = cache.attention(layer, q, seqs, cu, heads)
    cache.truncate(seqs, lens)                     # where drafted tokens were rejected

``seqs`` (int32 [n]) names the step's sequences, ``cu`` (int32 [n + 1]) the rows of the packed tensors that belong to each: for plain decoding
0, 1, .. n.  All arguments are tensors on the cache's device, and nothing here waits for the GPU: ``check()`` does, and raises what the
last page operation had to say.  Calls on one cache have to be ordered, by one stream or by events.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import KV_FORMAT, TPB_BF16, TPB_F16, TPB_F32, TPB_OK, TpbError

_ROWS = {torch.float32: TPB_F32, torch.bfloat16: TPB_BF16, torch.float16: TPB_F16}
_FORMAT = {torch.int8: KV_FORMAT["s8"], torch.float8_e4m3fn: KV_FORMAT["e4m3"]}
DTYPE = {"s8": torch.int8, "e4m3": torch.float8_e4m3fn}


class KvCache:
    """``k`` / ``v`` [layers][n_pages][kv_heads][page_tokens][head_dim], one f32 scale a page and head (``k_scale`` / ``v_scale``
    [layers][n_pages][kv_heads]), ``table`` [max_seqs][max_pages], ``lens`` and ``tail`` [max_seqs], ``refs`` [n_pages], ``result`` [4]: plain
    tensors, described at ``tpb_kv_cache`` in tpb200.h."""

    def __init__(self, backend, layers: int, n_pages: int, kv_heads: int, head_dim: int, max_seqs: int, max_pages: int,
                 page_tokens: int = 16, dtype: str = "s8"):
        if dtype not in DTYPE:
            raise TypeError(f"a cache holds s8 or e4m3 values (got {dtype})")
        if min(layers, n_pages, kv_heads, head_dim, max_seqs, max_pages, page_tokens) <= 0:
            raise ValueError("a cache's sizes must be positive")
        dev = backend.device
        shape = (layers, n_pages, kv_heads, page_tokens, head_dim)
        i32 = dict(dtype=torch.int32, device=dev)
        self._take(backend, torch.zeros(shape, dtype=torch.uint8, device=dev).view(DTYPE[dtype]),
                   torch.zeros(shape, dtype=torch.uint8, device=dev).view(DTYPE[dtype]), torch.zeros(shape[:3], device=dev),
                   torch.zeros(shape[:3], device=dev), torch.full((max_seqs, max_pages), -1, **i32), torch.zeros(max_seqs, **i32),
                   torch.zeros(n_pages, **i32), torch.zeros(max_seqs, **i32))

    @classmethod
    def wrap(cls, backend, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, table: torch.Tensor,
             lens: torch.Tensor, refs: torch.Tensor, tail: torch.Tensor) -> "KvCache":
        """A cache in tensors that the caller has (from a checkpoint of the pool, say); they are used as they are, not copied."""
        self = cls.__new__(cls)
        self._take(backend, k, v, k_scale, v_scale, table, lens, refs, tail)
        return self

    def _take(self, backend, k, v, k_scale, v_scale, table, lens, refs, tail):
        if k.dtype not in _FORMAT or v.dtype != k.dtype:
            raise TypeError(f"k and v must both be int8 or float8_e4m3fn (got {k.dtype}, {v.dtype})")
        if k.dim() != 5 or v.shape != k.shape:
            raise ValueError("k and v must be [layers][n_pages][kv_heads][page_tokens][head_dim]")
        if table.dim() != 2:
            raise ValueError("table must be [max_seqs][max_pages]")
        layers, n_pages, kv_heads, page_tokens, head_dim = k.shape
        max_seqs, max_pages = table.shape
        for name, t, dtype, shape in (("k", k, k.dtype, k.shape), ("v", v, k.dtype, k.shape),
                                      ("k_scale", k_scale, torch.float32, k.shape[:3]), ("v_scale", v_scale, torch.float32, k.shape[:3]),
                                      ("table", table, torch.int32, table.shape), ("lens", lens, torch.int32, (max_seqs,)),
                                      ("tail", tail, torch.int32, (max_seqs,)), ("refs", refs, torch.int32, (n_pages,))):
            if t.dtype != dtype:
                raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
            if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous, of shape {tuple(shape)} (got {tuple(t.shape)})")
            if t.device != backend.device:
                raise ValueError(f"{name} is on {t.device}, the backend on {backend.device}")
        self.be = backend
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.table, self.lens, self.refs, self.tail = table, lens, refs, tail
        self.layers, self.n_pages, self.kv_heads, self.page_tokens, self.head_dim = layers, n_pages, kv_heads, page_tokens, head_dim
        self.max_seqs, self.max_pages = max_seqs, max_pages
        self.result = torch.zeros(4, dtype=torch.int32, device=backend.device)
        nbytes = int(backend.lib.tpb_kv_scratch_bytes(n_pages, max_seqs))
        if nbytes == 0:
            raise ValueError(f"a cache of {n_pages} pages and {max_seqs} sequences is out of range")
        self._scratch = torch.empty(nbytes, dtype=torch.uint8, device=backend.device)
        self._calls, self._index, self._scale = backend._attn_calls, k.get_device(), head_dim ** -0.5
        self._no_workspace = _lib.KV_SHORT
        self._like = {}                    # empty tensors to make new ones by: half a microsecond less than torch.empty
        self._workspace_bytes = int(backend.lib.tpb_kv_attention_workspace_bytes(backend.h, head_dim))
        d = _lib.KvCacheDesc(k=k.data_ptr(), v=v.data_ptr(), k_scale=k_scale.data_ptr(), v_scale=v_scale.data_ptr(), table=table.data_ptr(),
                             lens=lens.data_ptr(), tail=tail.data_ptr(), refs=refs.data_ptr(), result=self.result.data_ptr(),
                             scratch=self._scratch.data_ptr(), n_pages=n_pages, layers=layers, kv_heads=kv_heads,
                             page_tokens=page_tokens, head_dim=head_dim, max_seqs=max_seqs, max_pages=max_pages, format=_FORMAT[k.dtype])
        self._desc, self._d = d, C.addressof(d)

    # -- arguments -------------------------------------------------------------------
    # A decode step makes two of these calls a layer, each about as long as its kernel: the checks ask every tensor for as little as they can.
    def _ints(self, name: str, t: torch.Tensor, n: int) -> int:
        if t.dtype is torch.int32 and t.dim() == 1 and t.shape[0] == n and t.is_contiguous() and t.get_device() == self._index:
            return t.data_ptr()
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32 (got {t.dtype})")
        raise ValueError(f"{name} must be a contiguous vector of {n} on {self.be.device} (got {tuple(t.shape)} on {t.device})")

    def _rows(self, name: str, t: torch.Tensor, rows: int, heads: int, dtype: torch.dtype) -> int:
        """Elements from one row to the next of [rows][heads * head_dim] or [rows][heads][head_dim]; columns are contiguous."""
        width = heads * self.head_dim
        s, st = t.shape, t.stride()
        if t.dtype is dtype and len(s) == 2 and s[1] == width and st[1] == 1 and s[0] == rows and t.get_device() == self._index:
            return st[0] if rows > 1 else width
        if t.dtype != dtype or dtype not in _ROWS:
            raise TypeError(f"{name} must be float32, bfloat16 or float16, like its partners (got {t.dtype})")
        if t.get_device() != self._index or s[0] != rows or not (
                len(s) == 3 and s[1] == heads and s[2] == self.head_dim and st[2] == 1 and (st[1] == self.head_dim or heads == 1)):
            raise ValueError(f"{name} must be [{rows}][{width}] on {self.be.device}, contiguous within a row (got {tuple(s)}, strides {st})")
        return st[0] if rows > 1 else width

    @staticmethod
    def _dtype(name: str, t: torch.Tensor) -> int:
        try:
            return _ROWS[t.dtype]
        except KeyError:
            raise TypeError(f"{name} must be float32, bfloat16 or float16 (got {t.dtype})") from None

    # -- tokens ----------------------------------------------------------------------
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, seqs: torch.Tensor, cu: torch.Tensor):
        """Quantises k and v ([rows][kv_heads * head_dim], f32, bf16 or f16) into the last cu[i + 1] - cu[i] places of each sequence: the
        tokens of its last ``extend``."""
        be, dtype = self.be, self._dtype("k", k)
        rows, n = k.shape[0], seqs.shape[0]
        ld_k, ld_v = self._rows("k", k, rows, self.kv_heads, k.dtype), self._rows("v", v, rows, self.kv_heads, k.dtype)
        ids, at = self._ints("seqs", seqs, n), self._ints("cu", cu, n + 1)
        rc = self._calls.tpb_kv_append(be._hv, be._stream(), self._d, layer, k.data_ptr(), ld_k, v.data_ptr(), ld_v, dtype, ids, at, n, rows)
        if rc != TPB_OK:
            be._check(rc)
        be.launches += n > 0 and rows > 0

    def read(self, layer: int, seqs: torch.Tensor, cu: torch.Tensor, rows: int, start: Optional[torch.Tensor] = None,
             dtype: torch.dtype = torch.float32, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values of tokens start[i] .. start[i] + cu[i + 1] - cu[i] - 1 of each sequence (from 0 without ``start``), packed into ``rows``
        rows; zero behind a sequence's end.  Rows of no sequence are not written."""
        be, n, width = self.be, seqs.shape[0], self.kv_heads * self.head_dim
        ids, at = self._ints("seqs", seqs, n), self._ints("cu", cu, n + 1)
        if out is None:
            like = self._like.get(dtype)
            if like is None:
                like = self._like[dtype] = torch.empty(0, dtype=dtype, device=be.device)
            k, v = like.new_empty((rows, width)), like.new_empty((rows, width))
            ld_k = ld_v = width
        else:
            k, v = out
            ld_k, ld_v = self._rows("k", k, rows, self.kv_heads, k.dtype), self._rows("v", v, rows, self.kv_heads, k.dtype)
        rc = self._calls.tpb_kv_read(be._hv, be._stream(), self._d, layer, k.data_ptr(), ld_k, v.data_ptr(), ld_v, self._dtype("k", k), ids,
                                     None if start is None else self._ints("start", start, n), at, n, rows)
        if rc != TPB_OK:
            be._check(rc)
        be.launches += n > 0 and rows > 0
        return k, v

    def attention(self, layer: int, q: torch.Tensor, seqs: torch.Tensor, cu: torch.Tensor, heads: int, scale: Optional[float] = None,
                  max_len: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of each sequence's last cu[i + 1] - cu[i] tokens, whose queries are q's rows ([rows][heads * head_dim], f32, bf16 or
        f16), over the sequence's cache; the result has q's type.  Scores, |scale * q . k|, stay below 2^22.  ``max_len``: an upper bound of the lengths, where the host knows one."""
        be, dtype = self.be, self._dtype("q", q)
        rows, n = q.shape[0], seqs.shape[0]
        ld_q = self._rows("q", q, rows, heads, q.dtype)
        if out is None:
            out = q.new_empty((rows, heads * self.head_dim))
            ld_out = heads * self.head_dim
        else:
            ld_out = self._rows("out", out, rows, heads, q.dtype)
        # of this call alone: another stream's call, or a captured one's replay, may run beside it.  Short sequences need none.
        work = None if 0 < max_len <= self._no_workspace else self._scratch.new_empty(self._workspace_bytes)
        ids, at = self._ints("seqs", seqs, n), self._ints("cu", cu, n + 1)
        rc = self._calls.tpb_kv_attention(be._hv, be._stream(), self._d, layer, out.data_ptr(), ld_out, q.data_ptr(), ld_q, dtype, ids, at, n, rows,
                                          heads, self._scale if scale is None else float(scale), max_len,
                                          None if work is None else work.data_ptr(), 0 if work is None else self._workspace_bytes)
        if rc != TPB_OK:
            be._check(rc)
        if n > 0 and rows > 0:
            be.launches += 1 if work is None else 2
        return out

    # -- pages -----------------------------------------------------------------------
    def extend(self, seqs: torch.Tensor, n_new: torch.Tensor):
        """Room for n_new[i] more tokens in sequence seqs[i]; lens counts them from here on."""
        n = seqs.shape[0]
        self.be._check(self.be.lib.tpb_kv_extend(self.be._hv, self.be._stream(), self._d, self._ints("seqs", seqs, n),
                                                 self._ints("n_new", n_new, n), n))
        self.be.launches += 1

    def truncate(self, seqs: torch.Tensor, lens: Optional[torch.Tensor] = None):
        """Cuts sequence seqs[i] to lens[i] tokens; without ``lens`` frees it."""
        n = seqs.shape[0]
        self.be._check(self.be.lib.tpb_kv_truncate(self.be._hv, self.be._stream(), self._d, self._ints("seqs", seqs, n),
                                                   None if lens is None else self._ints("lens", lens, n), n))
        self.be.launches += 1 if lens is None else 2

    def fork(self, src: torch.Tensor, dst: torch.Tensor, share: bool = True):
        """Makes the free sequence dst[i] a copy of src[i]: holding src's full pages and a copy of the part-filled one, or, with ``share``
        false, a copy of every page."""
        n = src.shape[0]
        self.be._check(self.be.lib.tpb_kv_fork(self.be._hv, self.be._stream(), self._d, self._ints("src", src, n), self._ints("dst", dst, n), n,
                                               int(share)))
        self.be.launches += 2

    def compact(self):
        """Moves the pages in use to the lowest indices."""
        self.be._check(self.be.lib.tpb_kv_compact(self.be._hv, self.be._stream(), self._d))
        self.be.launches += 2

    def check(self) -> int:
        """Waits for the device; the number of free pages after the last page operation.  Raises TpbError where that operation was
        refused (a refusal of an earlier one is written over), or where a kernel of this cache's backend, another cache's call among
        them, met a sequence, page or length that does not fit since the last poll."""
        self.be.status_poll()
        status, free, _, needed = self.result.tolist()
        if status != TPB_OK:
            raise TpbError(status, f"the page operation changed nothing: {free} pages are free, it needs {needed}"
                           if status == _lib.TPB_ERR_OOM else "the page operation changed nothing: its list does not fit the cache")
        return free
