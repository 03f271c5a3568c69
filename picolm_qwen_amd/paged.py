"""Attention over a paged KV cache, for a server of many requests (include/pqa.h, paged cache).

    att = PagedAttention(n_layers, n_pages, page_size, n_heads, n_kv_heads, head_dim, dtype="bf16", rope_base=1e6)
    batch = att.batch(max_seqs=64, max_tokens=2048)
    batch.set(n_new, lengths, page_lists)          # once per step, for every layer
    out = att.forward(layer, batch, q, k, v)       # append, then attend

Token rows are torch tensors on the handle's GPU, [n][heads * head_dim] with any distance between
rows. Calls run on torch's current stream of that GPU. Every call goes through libpqa.so; a
missing library raises.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._lib import PQAError, lib
from .attention import ROPE_NEOX_HALF, rope_table

_TYPES = {"f32": (0, "float32", "float16"), "f16": (1, "float16", "float16"), "bf16": (2, "bfloat16", "bfloat16")}


def _int_array(x, what: str):
    """x as a C-contiguous int32 array; values that int32 does not hold raise."""
    a = np.asarray(x)
    if a.size == 0:
        a = a.astype(np.int32)
    if a.dtype.kind not in "iu":
        raise ValueError(f"{what} must be whole numbers, got {a.dtype}")
    if a.size and (a.min() < -2**31 or a.max() >= 2**31):
        raise ValueError(f"{what} must fit int32")
    return np.ascontiguousarray(a, dtype=np.int32)


class PagedBatch:
    """Which tokens of which sequences the next calls are about (pqa_batch)."""

    def __init__(self, att: "PagedAttention", max_seqs: int, max_tokens: int, max_len: int):
        self.att = att  # keeps the handle alive
        self.max_seqs, self.max_tokens, self.max_len = max_seqs, max_tokens, max_len
        self.n_tokens = 0
        self._h = None
        h = C.c_void_p()
        att._check(lib().pqa_batch_create(att.handle, C.byref(h), max_seqs, max_tokens, max_len))
        self._h = h

    @property
    def handle(self):
        if self._h is None:
            raise RuntimeError("batch destroyed")
        return self._h

    def set(self, n_new, lengths, pages) -> None:
        """n_new[i] new tokens at the end of lengths[i] positions; pages: a list of page lists, or an integer
        array [n_seqs][stride]."""
        self.att.handle  # a closed cache raises
        n_new, lengths = _int_array(n_new, "n_new"), _int_array(lengths, "lengths")
        if n_new.ndim != 1 or lengths.shape != n_new.shape:
            raise ValueError("n_new and lengths must be lists of one length")
        if isinstance(pages, (list, tuple)):
            lists = [_int_array(p, "pages").reshape(-1) for p in pages]
            table = np.full((len(lists), max((p.size for p in lists), default=0)), -1, np.int32)
            for row, p in zip(table, lists):
                row[:p.size] = p
        else:
            table = _int_array(pages, "pages")
        if table.ndim != 2 or table.shape[0] != n_new.size:
            raise ValueError(f"expected the pages of {n_new.size} sequences")
        self.att._check(lib().pqa_batch_set(self.handle, n_new.size, n_new.ctypes.data, lengths.ctypes.data, table.ctypes.data,
                                            table.shape[1], self.att._stream()))
        self.n_tokens = int(n_new.sum())

    def close(self) -> None:
        if getattr(self, "_h", None) is not None:
            lib().pqa_batch_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


class PagedAttention:
    """The paged cache of a model's attention (pqa_paged) on the current GPU.

    dtype: "f32" (fp32 rows over fp16 pages), "f16" or "bf16". key_pages and val_pages
    [n_layers][n_pages][n_kv_heads][page_size][head_dim] (without the first axis for one layer), and
    key_bounds int8 [...][2][head_dim] with key_scales float32 [n_layers][n_pages][n_kv_heads], may be given as
    tensors; else they are made here, zeroed (bounds with bounds=True). rot_dim elements of a head are
    rotated (None: all), by tables [max_pos][rot_dim / 2] or by rope_base and max_pos; without either nothing is."""

    def __init__(self, n_layers: int, n_pages: int, page_size: int, n_heads: int, n_kv_heads: int, head_dim: int,
                 dtype: str = "f32", rope_style: int = ROPE_NEOX_HALF, rot_dim=None, rope_base=None, max_pos=None,
                 rope_cos=None, rope_sin=None, bounds: bool = False, key_pages=None, val_pages=None, key_bounds=None,
                 key_scales=None):
        import torch

        self._h = None
        if dtype not in _TYPES:
            raise ValueError(f"dtype must be one of {sorted(_TYPES)}, got {dtype!r}")
        code, io, page = _TYPES[dtype]
        self.dtype, self.io_type, self.page_type = dtype, getattr(torch, io), getattr(torch, page)
        self.n_layers, self.n_pages, self.page_size = n_layers, n_pages, page_size
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, n_kv_heads, head_dim
        self.q_dim, self.kv_dim = n_heads * head_dim, n_kv_heads * head_dim
        given = [x is not None for x in (key_pages, val_pages)]
        if any(given) != all(given) or (key_bounds is None) != (key_scales is None) or (key_bounds is not None and not all(given)):
            raise ValueError("give key_pages and val_pages together, and key_bounds and key_scales with them")
        device = None
        if all(given):
            device = key_pages.device
        elif torch.cuda.is_available():
            device = torch.device("cuda", torch.cuda.current_device())
        shape = (n_layers, n_pages, n_kv_heads)
        if all(given):
            for t, tail, kind, what in ((key_pages, (page_size, head_dim), self.page_type, "key_pages"),
                                        (val_pages, (page_size, head_dim), self.page_type, "val_pages"),
                                        (key_bounds, (2, head_dim), torch.int8, "key_bounds"),
                                        (key_scales, (), torch.float32, "key_scales")):
                if t is not None:
                    self._check_memory(t, shape + tail, kind, device, what)
            bounds = key_bounds is not None
        elif device is not None and min(shape) > 0 and page_size > 0 and head_dim > 0:
            key_pages = torch.zeros(shape + (page_size, head_dim), dtype=self.page_type, device=device)
            val_pages = torch.zeros_like(key_pages)
            if bounds:
                key_bounds = torch.zeros(shape + (2, head_dim), dtype=torch.int8, device=device)
                key_scales = torch.zeros(shape, dtype=torch.float32, device=device)
        self.key_pages, self.val_pages, self.key_bounds, self.key_scales = key_pages, val_pages, key_bounds, key_scales
        self.has_bounds = bool(bounds)
        self._device = device
        self._index = device.index if device is not None else -1
        ptr = [None if t is None else t.data_ptr() for t in (key_pages, val_pages, key_bounds, key_scales)]
        h = C.c_void_p()
        if device is not None:
            with torch.cuda.device(device):
                torch.cuda.current_stream().synchronize()  # the zeroed memory
                rc = lib().pqa_paged_create(C.byref(h), n_layers, n_pages, page_size, n_heads, n_kv_heads, head_dim, code,
                                            int(self.has_bounds), *ptr)
        else:
            rc = lib().pqa_paged_create(C.byref(h), n_layers, n_pages, page_size, n_heads, n_kv_heads, head_dim, code,
                                        int(self.has_bounds), *ptr)
        self._check(rc)
        self._h = h
        self._calls = lib()
        # one call costs the host some 3 us; what the wrapper looks up each time is kept short
        self._empty_like, self._zeros_like = torch.empty_like, torch.zeros_like
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        if rope_cos is not None or rope_sin is not None or rope_base is not None:
            self.set_rope(rope_style, rot_dim, rope_base, max_pos, rope_cos, rope_sin)

    @staticmethod
    def _check_memory(t, shape, kind, device, what) -> None:
        if t.dtype != kind:
            raise ValueError(f"{what}: expected {kind}, got {t.dtype}")
        if tuple(t.shape) != shape and not (shape[0] == 1 and tuple(t.shape) == shape[1:]):
            raise ValueError(f"{what}: expected shape {shape}, got {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous")
        if not t.is_cuda or t.device != device:
            raise ValueError(f"{what} must be on the GPU, all of the cache on one")

    # -- lifecycle ---------------------------------------------------------
    @property
    def handle(self):
        if self._h is None:
            raise RuntimeError("paged cache destroyed")
        return self._h

    def close(self) -> None:
        """Destroys the handle; its batches must be closed before."""
        if getattr(self, "_h", None) is not None:
            lib().pqa_paged_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def _check(self, rc: int) -> None:
        if rc:
            msg = lib().pqa_paged_last_error(self._h)
            raise PQAError(rc, msg.decode() if msg else "")

    def _stream(self) -> int:
        if self._raw_stream is not None:
            return self._raw_stream(self._index)
        import torch

        return torch.cuda.current_stream(self._device).cuda_stream

    def last_error(self) -> str:
        msg = lib().pqa_paged_last_error(self.handle)
        return msg.decode() if msg else ""

    # -- settings ------------------------------------------------------------
    def set_rope(self, rope_style: int = ROPE_NEOX_HALF, rot_dim=None, rope_base=None, max_pos=None, rope_cos=None,
                 rope_sin=None) -> None:
        """Rotation tables of the first rot_dim elements of a head (None: all; 0: no rotation), given or of rope_base."""
        rot = self.head_dim if rot_dim is None else int(rot_dim)
        if rot == 0:
            self._check(lib().pqa_paged_set_rope(self.handle, rope_style, 0, 0, None, None))
            return
        if rope_cos is None and rope_sin is None:
            if rope_base is None or max_pos is None:
                raise ValueError("give rope_cos and rope_sin, or rope_base and max_pos")
            if rot < 0 or rot % 2 or max_pos <= 0:
                raise ValueError("rot_dim must be even and max_pos positive")
            rope_cos, rope_sin = rope_table(rope_base, rot, max_pos)
        if rope_cos is None or rope_sin is None:
            raise ValueError("give both RoPE tables or neither")
        c = np.ascontiguousarray(rope_cos, dtype=np.float32)
        s = np.ascontiguousarray(rope_sin, dtype=np.float32)
        if c.ndim != 2 or c.shape != s.shape or c.shape[1] * 2 != rot or (max_pos is not None and c.shape[0] < max_pos):
            raise ValueError(f"RoPE tables must be [max_pos][{rot // 2}]")
        self._check(lib().pqa_paged_set_rope(self.handle, rope_style, rot, max_pos or c.shape[0], c.ctypes.data, s.ctypes.data))

    def set_qk_norm(self, layer: int, q_norm_w, k_norm_w) -> None:
        """Layer's QK-norm weights ([head_dim] each); None turns it off."""
        if q_norm_w is None and k_norm_w is None:
            self._check(lib().pqa_paged_set_qk_norm(self.handle, layer, None, None))
            return
        w = [None if x is None else np.ascontiguousarray(x, dtype=np.float32) for x in (q_norm_w, k_norm_w)]
        if any(x is not None and x.size != self.head_dim for x in w):
            raise ValueError(f"norm weights must have {self.head_dim} elements")
        self._check(lib().pqa_paged_set_qk_norm(self.handle, layer, *[None if x is None else x.ctypes.data for x in w]))

    def batch(self, max_seqs: int, max_tokens: int, max_len=None) -> PagedBatch:
        """A batch of at most max_seqs sequences and max_tokens new tokens; max_len: the longest sequence (None: the whole pool,
        for which the batch's page table takes 4 * max_seqs * n_pages bytes)."""
        if max_len is None:
            max_len = min(self.n_pages * self.page_size, 2**30)
        return PagedBatch(self, max_seqs, max_tokens, max_len)

    # -- calls ----------------------------------------------------------------
    def _rows(self, t, dim: int, n: int, what: str):
        """(address, row distance) of token rows the library reads or writes n of; anything that would make a kernel leave the
        tensor raises."""
        stride = t.stride()
        if (len(stride) == 2 and stride[1] == 1 and stride[0] >= dim and t.size(1) == dim and t.size(0) >= n
                and t.dtype is self.io_type and t.get_device() == self._index):
            return t.data_ptr(), stride[0]
        return self._unusual_rows(t, dim, n, what)

    def _unusual_rows(self, t, dim: int, n: int, what: str):
        if t.dim() != 2 or t.shape[1] != dim or t.shape[0] < n:
            raise ValueError(f"{what}: expected at least {n} rows of {dim}, got {tuple(t.shape)}")
        if t.dtype != self.io_type:
            raise ValueError(f"{what}: expected {self.io_type}, got {t.dtype}")
        if t.get_device() != self._index:
            raise ValueError(f"{what} must be on the cache's GPU")
        if t.stride(1) != 1 or t.shape[0] > 1:
            raise ValueError(f"{what}: elements of a row must lie side by side, rows apart")
        return t.data_ptr(), dim  # one row, whose distance to the next means nothing

    def _out(self, q, batch):
        # rows behind the batch's last token are not written
        return self._empty_like(q) if q.size(0) == batch.n_tokens else self._zeros_like(q)

    def _handles(self, batch):
        h, b = self._h, batch._h
        return (h, b) if h is not None and b is not None else (self.handle, batch.handle)  # the latter raise

    def append(self, layer: int, batch: PagedBatch, q, k, v, q_out=None):
        """K and V of the batch's new tokens into their pages; returns q normed and rotated (q_out may be q)."""
        n = batch.n_tokens
        a = self._rows(q, self.q_dim, n, "q")
        if q_out is None:
            q_out = self._out(q, batch)
        more = self._rows(k, self.kv_dim, n, "k") + self._rows(v, self.kv_dim, n, "v") + self._rows(q_out, self.q_dim, n, "q_out")
        rc = self._calls.pqa_paged_append(*self._handles(batch), layer, *a, *more, self._stream())
        if rc:
            self._check(rc)
        return q_out

    def attend(self, layer: int, batch: PagedBatch, q, out=None):
        """Causal attention of the new tokens over their sequences' pages, q as append returns it (out may be q)."""
        n = batch.n_tokens
        a = self._rows(q, self.q_dim, n, "q")
        if out is None:
            out = self._out(q, batch)
        o = self._rows(out, self.q_dim, n, "out")
        rc = self._calls.pqa_paged_attend(*self._handles(batch), layer, *a, *o, self._stream())
        if rc:
            self._check(rc)
        return out

    def forward(self, layer: int, batch: PagedBatch, q, k, v, out=None):
        """append, then attend."""
        n = batch.n_tokens
        a = self._rows(q, self.q_dim, n, "q")
        if out is None:
            out = self._out(q, batch)
        more = self._rows(k, self.kv_dim, n, "k") + self._rows(v, self.kv_dim, n, "v") + self._rows(out, self.q_dim, n, "out")
        rc = self._calls.pqa_paged_forward(*self._handles(batch), layer, *a, *more, self._stream())
        if rc:
            self._check(rc)
        return out

    def attend_sparse(self, layer: int, batch: PagedBatch, q, select: int, first: int = 1, last: int = 2, out=None, chosen=None):
        """attend with a budget of `select` pages per token and KV head; returns (out, chosen [n][n_kv_heads][select])."""
        import torch

        n = batch.n_tokens
        a = self._rows(q, self.q_dim, n, "q")
        if out is None:
            out = self._out(q, batch)
        if chosen is None:
            if select < 1:
                raise ValueError("select must be positive")
            make = torch.empty if q.shape[0] == n else torch.zeros
            chosen = make((q.shape[0], self.n_kv_heads, select), dtype=torch.int32, device=q.device)
        elif (chosen.dtype != torch.int32 or chosen.dim() != 3 or chosen.shape[0] < n
              or tuple(chosen.shape[1:]) != (self.n_kv_heads, select) or not chosen.is_contiguous()
              or chosen.get_device() != self._index):
            raise ValueError(f"chosen must be contiguous int32 [{n}][{self.n_kv_heads}][{select}] on the cache's GPU")
        o = self._rows(out, self.q_dim, n, "out")
        rc = self._calls.pqa_paged_attend_sparse(*self._handles(batch), layer, *a, select, first, last, chosen.data_ptr(), *o,
                                                 self._stream())
        if rc:
            self._check(rc)
        return out, chosen
