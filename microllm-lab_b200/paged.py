"""Host side of the paged serving operators (include/mllm.h: mllm_rope_append, mllm_paged_attn,
mllm_copy_pages, mllm_sample) on device pointers, and the page bookkeeping of a cache.

The reference keeps one contiguous cache per engine (engine/infer.js:348-358) and chooses ids greedily
(engine/infer.js:240-287); these operators serve many sequences whose caches grow page by page, share
the pages of a common prompt, and are sampled.  ``examples/paged_sampling.py`` runs them together.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from .engine import DTYPES, MllmError, load_library


class PagedKV(ctypes.Structure):
    """mllm_paged_kv: one layer's K/V page pool (see ``paged_kv``)."""

    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("page_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("pos_stride", ctypes.c_int64), ("dtype", ctypes.c_int32),
                ("n_pages", ctypes.c_int32), ("page_len", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32)]


def _check(rc: int) -> None:
    if rc:
        raise MllmError(rc, load_library().mllm_last_error(None).decode())


def paged_kv(k_ptr: int, v_ptr: int, dtype: str, n_pages: int, page_len: int, n_kv_heads: int, head_dim: int,
             strides=None) -> PagedKV:
    """Descriptor of one layer's page pool.  ``strides`` are the elements between pages, kv heads and
    positions; by default pages are contiguous and kv-head-major, [page][kvHead][position][dim]."""
    page, head, pos = strides or (n_kv_heads * page_len * head_dim, page_len * head_dim, head_dim)
    return PagedKV(k_ptr, v_ptr, page, head, pos, DTYPES[dtype], n_pages, page_len, n_kv_heads, head_dim)


def rope_append_device(kv: PagedKV, dtype: str, qkv_ptr: int, row_stride: int, n_tok: int, n_heads: int, seq_ptr: int,
                       pos_ptr: int, table_ptr: int, n_seq: int, table_stride: int, cos_ptr: int, sin_ptr: int,
                       n_pos: int, rope_dim: int, q_ptr: int, q_stride: int, interleaved: bool = False,
                       q_gain_ptr: int = 0, k_gain_ptr: int = 0, eps: float = 1e-6, stream: int = 0) -> None:
    """Per-head norm (with gains), rotation by position, q out, k and v into the cache's pages
    (mllm_rope_append).  ``seq_ptr`` 0: row t belongs to sequence t."""
    _check(load_library().mllm_rope_append(ctypes.byref(kv), DTYPES[dtype], qkv_ptr, row_stride, n_tok, n_heads,
                                           seq_ptr or None, pos_ptr, table_ptr, n_seq, table_stride,
                                           q_gain_ptr or None, k_gain_ptr or None, eps, cos_ptr or None,
                                           sin_ptr or None, n_pos, rope_dim, interleaved, q_ptr, q_stride,
                                           stream or None))


def paged_attn_workspace(n_seq: int, n_heads: int, head_dim: int) -> int:
    """Bytes of the workspace, zeroed once, that ``paged_attn_device`` needs (mllm_paged_attn_workspace).  One of
    the largest ``n_heads`` and ``head_dim`` serves calls of any shape, one after another."""
    return int(load_library().mllm_paged_attn_workspace(n_seq, n_heads, head_dim))


def paged_attn_device(kv: PagedKV, dtype: str, q_ptr: int, q_stride: int, n_seq: int, n_heads: int, len_ptr: int,
                      table_ptr: int, table_stride: int, scale: float, out_ptr: int, out_stride: int, ws_ptr: int,
                      ws_bytes: int, lse_ptr: int = 0, stream: int = 0) -> None:
    """Attention of one new token per sequence over its pages (mllm_paged_attn)."""
    _check(load_library().mllm_paged_attn(ctypes.byref(kv), DTYPES[dtype], q_ptr, q_stride, n_seq, n_heads, len_ptr,
                                          table_ptr, table_stride, scale, out_ptr, out_stride, lse_ptr or None,
                                          ws_ptr, ws_bytes, stream or None))


def _page_ids(ids) -> np.ndarray:
    """Page ids as contiguous int32, refused where that would change one."""
    ids = np.asarray(ids)
    if ids.dtype != np.int32 and ids.size:
        if ids.dtype.kind not in "iu":
            raise TypeError(f"page ids are whole numbers, not {ids.dtype}")
        low, high = int(ids.min()), int(ids.max())
        if low < -1 << 31 or high >= 1 << 31:
            raise ValueError(f"page ids from {low} to {high} do not fit 32 bits")
    return np.ascontiguousarray(ids, np.int32)


def copy_pages_device(kv: PagedKV, src, dst, n_layers: int = 1, layer_stride: int = 0, stream: int = 0) -> None:
    """Copy pages src[i] -> dst[i] (host ids) in every layer's pool (mllm_copy_pages)."""
    src, dst = _page_ids(src), _page_ids(dst)
    if src.shape != dst.shape or src.ndim != 1:
        raise ValueError("src and dst are page lists of one length")
    _check(load_library().mllm_copy_pages(ctypes.byref(kv), n_layers, layer_stride, src.ctypes.data, dst.ctypes.data,
                                          len(src), stream or None))


def sample_device(dtype: str, logits_ptr: int, row_stride: int, rows: int, vocab: int, u_ptr: int, id_ptr: int,
                  logprob_ptr: int = 0, kept_ptr: int = 0, probs_ptr: int = 0, temperature_ptr: int = 0,
                  top_k_ptr: int = 0, top_p_ptr: int = 0, min_p_ptr: int = 0, stream: int = 0) -> None:
    """Temperature / top-k / top-p / min-p sampling from one uniform number per row (mllm_sample)."""
    _check(load_library().mllm_sample(DTYPES[dtype], logits_ptr, row_stride, rows, vocab, temperature_ptr or None,
                                      top_k_ptr or None, top_p_ptr or None, min_p_ptr or None, u_ptr, id_ptr,
                                      logprob_ptr or None, kept_ptr or None, probs_ptr or None, stream or None))


def rope_tables(n_pos: int, rope_dim: int, theta: float = 10000.0, factor: float = 1.0, low: float = 0.0,
                high: float = 0.0, original: int = 0):
    """cos and sin tables [n_pos][rope_dim / 2] for ``rope_append_device``: f32 inverse frequencies and
    f64 angles, as buildRope does (engine/infer.js:185-206).  ``factor`` > 1 stretches them to longer
    contexts: with ``original`` 0 every frequency is divided by it; with the ``original`` context length,
    frequencies that turn fewer than ``low`` times over it are, those that turn more than ``high`` times
    stay, and the ones between are blended linearly in their number of turns."""
    half = rope_dim // 2
    inv = (1.0 / np.power(float(theta), 2.0 * np.arange(half) / max(rope_dim, 1))).astype(np.float32)
    if factor != 1.0:
        part = np.zeros(half)
        if original:
            turns = original * inv.astype(np.float64) / (2 * math.pi)
            part = np.clip((turns - low) / (high - low), 0.0, 1.0) if high > low else (turns >= high).astype(np.float64)
        inv = (inv * (part + (1.0 - part) / factor)).astype(np.float32)
    angle = np.arange(n_pos, dtype=np.float64)[:, None] * inv.astype(np.float64)[None, :]
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


class PageTable:
    """Which pages of a pool belong to which sequence: growth, forks that share pages, frees and
    compaction.  Page ids count references, so that forked sequences read the same pages until one of
    them writes.  Pure bookkeeping on the host: methods that need page contents moved return the
    (src, dst) lists for ``copy_pages_device``, which the caller runs before its next write."""

    def __init__(self, n_pages: int, page_len: int):
        if n_pages < 1 or page_len < 1:
            raise ValueError("a pool has at least one page of at least one position")
        self.n_pages, self.page_len = int(n_pages), int(page_len)
        self._refs = [0] * self.n_pages
        self._free = list(range(self.n_pages - 1, -1, -1))  # lowest id on top
        self._pages: dict[int, list[int]] = {}
        self._len: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages(self, seq: int) -> list[int]:
        return list(self._pages[seq])

    def length(self, seq: int) -> int:
        return self._len[seq]

    def new(self) -> int:
        """An empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def grow(self, seq: int, n: int = 1):
        """Room for ``n`` more positions.  Returns (src, dst): copies to run before they are written (the
        partly filled last page, where another sequence shares it).  Raises MemoryError, changing
        nothing, when the pool has too few free pages."""
        if n < 0:
            raise ValueError("n counts positions")
        pages, have = self._pages[seq], self._len[seq]
        more = -(-(have + n) // self.page_len) - len(pages)
        shared = n > 0 and have % self.page_len != 0 and self._refs[pages[-1]] > 1
        if more + shared > len(self._free):
            raise MemoryError(f"{more + shared} pages wanted, {len(self._free)} free")
        moved = ([], [])
        if shared:
            old, pages[-1] = pages[-1], self._take()
            self._refs[old] -= 1
            moved = ([old], [pages[-1]])
        pages.extend(self._take() for _ in range(more))
        self._len[seq] = have + n
        return moved

    def grow_all(self, seqs, n: int = 1):
        """``grow`` for each of ``seqs`` (each once), or for none: MemoryError when the pool has too few free
        pages for all of them.  Returns the copies of all as one (src, dst)."""
        if n < 0:
            raise ValueError("n counts positions")
        seqs = list(seqs)
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is there twice")
        want, refs = 0, {}  # refs: what those before leave of a shared last page's references
        for s in seqs:
            pages, have = self._pages[s], self._len[s]
            want += -(-(have + n) // self.page_len) - len(pages)
            if n and have % self.page_len:
                last = pages[-1]
                left = refs.get(last, self._refs[last])
                if left > 1:
                    want += 1
                    refs[last] = left - 1
        if want > len(self._free):
            raise MemoryError(f"{want} pages wanted, {len(self._free)} free")
        src, dst = [], []
        for s in seqs:
            a, b = self.grow(s, n)
            src += a
            dst += b
        return src, dst

    def fork(self, seq: int) -> int:
        """A new sequence with the same contents, sharing every page."""
        new = self.new()
        self._pages[new], self._len[new] = list(self._pages[seq]), self._len[seq]
        for p in self._pages[new]:
            self._refs[p] += 1
        return new

    def free(self, seq: int) -> None:
        """Give a sequence's pages back; those that another one shares stay."""
        self._len.pop(seq)
        for p in self._pages.pop(seq):
            self._refs[p] -= 1
            if not self._refs[p]:
                self._free.append(p)
        self._free.sort(reverse=True)

    def compact(self):
        """Move the pages in use to the lowest ids.  Returns (src, dst) to copy; no page is in both."""
        used = self.n_pages - len(self._free)
        holes = sorted(p for p in self._free if p < used)
        high = [p for p in range(used, self.n_pages) if self._refs[p]]
        to = dict(zip(high, holes))
        for pages in self._pages.values():
            pages[:] = [to.get(p, p) for p in pages]
        for a, b in to.items():
            self._refs[a], self._refs[b] = 0, self._refs[a]
        self._free = list(range(self.n_pages - 1, used - 1, -1))
        return high, holes

    def table(self, seqs, width: int = 0) -> np.ndarray:
        """Page ids [len(seqs)][width] as int32, -1 past a sequence's last page (width 0: the widest)."""
        rows = [self._pages[s] for s in seqs]
        width = width or max([1] + [len(r) for r in rows])
        out = np.full((len(rows), width), -1, np.int32)
        for r, pages in zip(out, rows):
            if len(pages) > width:
                raise ValueError(f"a sequence of {len(pages)} pages in a table of {width}")
            r[: len(pages)] = pages
        return out

    def _take(self) -> int:
        p = self._free.pop()
        self._refs[p] = 1
        return p
