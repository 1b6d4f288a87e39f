"""Serving many sequences from one paged key/value cache.

The reference leaves the cache to oMLX and attention to the model library, one sequence at a time; this module
is the part of a server that sits between the EXL3 projections:

  PagedKVCache      pool of fixed-size pages for all layers, pages handed to sequences as they grow
  PagedBatch        what one step feeds: new rows of some sequences, as device tables the kernels read
  paged_qkv_post    q/k RMSNorm + rotary embedding + append to the pages (exl3_paged_qkv_post)
  paged_attn        attention of the new rows over the pages, chunks and single tokens alike (exl3_paged_attn)

A batch is cu_rows (seqs + 1), lens (seqs) and page_table (seqs, cols), all int32 on the device: sequence s feeds
rows cu_rows[s] .. cu_rows[s + 1] - 1 and holds lens[s] positions once they are appended, so its row i is at
position lens[s] - rows[s] + i; position p lives in page page_table[s, p // page_size]. Rows at negative positions
are padding: nothing is appended and the output is zero (a captured graph's unused slots have lens 0). The
kernels read the tables themselves, so no call waits for the host and a captured graph follows their contents.

Calls run on the current stream. Tables that name something outside the pool set a bit in a per-device status
word, as a pipeline wait that gave up does: check_paged_status() raises on it.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import PagedDesc, check, dtype_code, lib, stream_ptr

_CACHE_DTYPES = (torch.float16, torch.bfloat16)
_status: dict = {}
_workspaces: dict = {}


def _status_word(device: torch.device) -> torch.Tensor:
    word = _status.get(device.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call a paged kernel once on this device before capturing it in a graph")
        word = torch.zeros(4, dtype=torch.int32, device=device)
        _status[device.index] = word
    return word


def paged_status(device: torch.device | None = None) -> int:
    """The device's status word of the paged kernels (0: nothing was out of range, no wait gave up); synchronises."""
    idx = torch.cuda.current_device() if device is None or device.index is None else device.index
    word = _status.get(idx)
    return 0 if word is None else int(word[0].item())


def check_paged_status(device: torch.device | None = None) -> None:
    """Raise RuntimeError if a paged kernel on `device` met a page, position or wait it could not serve, and clear
    the word. Synchronises."""
    value = paged_status(device)
    if value:
        idx = torch.cuda.current_device() if device is None or device.index is None else device.index
        _status[idx].zero_()
        what = [t for bit, t in ((8, "a table names a page or position outside its range"),
                                 (1, "a pipeline wait timed out")) if value & bit]
        raise RuntimeError(f"paged kernels: {'; '.join(what) or 'error'} (status 0x{value:x}); the outputs of the "
                           "failed call are invalid")


def _need(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


def _descriptor(k_pages, v_pages, page_table, cu_rows, lens, rows: int) -> PagedDesc:
    """Checked descriptor of the batch: what can be checked without reading device memory."""
    dt = k_pages.dtype
    if dt not in _CACHE_DTYPES or v_pages.dtype != dt:
        raise TypeError("k_pages and v_pages must both be fp16 or both bf16")
    if page_table.dtype != torch.int32 or cu_rows.dtype != torch.int32 or lens.dtype != torch.int32:
        raise TypeError("page_table, cu_rows and lens must be int32")
    dev = k_pages.device
    if dev.type != "cuda":
        raise ValueError("EXL3 kernels take CUDA tensors")
    _need(v_pages.device == dev and page_table.device == dev and cu_rows.device == dev and lens.device == dev,
          "the pages and the batch's tables must be on one device")
    shape = k_pages.shape
    _need(len(shape) == 4 and v_pages.shape == shape, "pages must be (num_pages, hkv, page_size, head_dim), K and V alike")
    _need(page_table.dim() == 2 and cu_rows.dim() == 1 and lens.dim() == 1, "page_table is 2-d, cu_rows and lens 1-d")
    seqs, cols = page_table.shape
    _need(seqs >= 1 and cu_rows.shape[0] == seqs + 1 and lens.shape[0] == seqs,
          "page_table (seqs, cols), cu_rows (seqs + 1) and lens (seqs) must agree")
    _need(k_pages.is_contiguous() and v_pages.is_contiguous(), "pages must be contiguous")
    _need(page_table.is_contiguous() and cu_rows.is_contiguous() and lens.is_contiguous(),
          "page_table, cu_rows and lens must be contiguous")
    return PagedDesc(k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), cu_rows.data_ptr(), lens.data_ptr(),
                     seqs, rows, cols, shape[0], shape[2], shape[1], shape[3], 0 if dt is torch.float16 else 1)


def _strided(x: torch.Tensor, width: int, name: str) -> int:
    """Row stride in elements of a (rows, width) view with contiguous rows."""
    _need(x.dim() == 2 and x.shape[1] == width, f"{name} must be (rows, {width})")
    _need(x.stride(1) == 1 and (x.shape[0] < 2 or x.stride(0) >= width), f"{name} needs contiguous, non-overlapping rows")
    return max(x.stride(0), width)


def paged_qkv_post(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_norm_w: torch.Tensor | None,
                   k_norm_w: torch.Tensor | None, eps: float, cos: torch.Tensor, sin: torch.Tensor,
                   k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, cu_rows: torch.Tensor,
                   lens: torch.Tensor, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Per-head q/k RMSNorm (skipped where the weight is None) and rotate-half rotary embedding at each row's
    position, k and v appended to the pages; returns q (rows, hq, head_dim) in the cache's dtype.

    q (rows, hq * head_dim), k and v (rows, hkv * head_dim), fp16 or bf16, one dtype; column views of a fused
    projection output are fine. cos / sin f32 (positions, rotated / 2): the first 2 * cos.shape[1] elements of a head
    are rotated. Computed in fp32 and rounded once, to the cache's dtype. Two live rows of a call must not share a position.
    """
    rows = q.shape[0]
    b = _descriptor(k_pages, v_pages, page_table, cu_rows, lens, rows)
    hd, dt = b.head_dim, q.dtype
    if dt not in _CACHE_DTYPES or k.dtype != dt or v.dtype != dt:
        raise TypeError("q, k and v must all be fp16 or all bf16")
    _need(k.shape[0] == rows and v.shape[0] == rows, "q, k and v must have the same rows")
    _need(q.dim() == 2 and q.shape[1] > 0 and q.shape[1] % (b.hkv * hd) == 0,
          "q's width must be a multiple of hkv * head_dim")
    hq = q.shape[1] // hd
    sq, sk, sv = _strided(q, hq * hd, "q"), _strided(k, b.hkv * hd, "k"), _strided(v, b.hkv * hd, "v")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("cos and sin must be fp32")
    _need(cos.dim() == 2 and cos.shape == sin.shape and cos.is_contiguous() and sin.is_contiguous(),
          "cos and sin must be contiguous (positions, rotated / 2)")
    dev = k_pages.device
    _need(q.device == dev and k.device == dev and v.device == dev and cos.device == dev and sin.device == dev,
          "all tensors must be on one device")
    for w in (q_norm_w, k_norm_w):
        if w is not None:
            if w.dtype != dt:
                raise TypeError("norm weights must have q's dtype")
            _need(w.numel() == hd and w.is_contiguous() and w.device == dev, "norm weights must be contiguous (head_dim)")
    if q_out is None:
        q_out = torch.empty((rows, hq, hd), dtype=k_pages.dtype, device=dev)
    else:
        _need(q_out.shape == (rows, hq, hd) and q_out.dtype == k_pages.dtype and q_out.is_contiguous()
              and q_out.device == dev, "q_out must be contiguous (rows, hq, head_dim) in the cache's dtype")
    with torch.cuda.device(dev):
        check(lib().exl3_paged_qkv_post(b, q.data_ptr(), k.data_ptr(), v.data_ptr(), sq, sk, sv,
                                        0 if dt is torch.float16 else 1, hq,
                                        None if q_norm_w is None else q_norm_w.data_ptr(),
                                        None if k_norm_w is None else k_norm_w.data_ptr(), eps, cos.data_ptr(),
                                        sin.data_ptr(), cos.shape[0], cos.shape[1], q_out.data_ptr(),
                                        _status_word(dev).data_ptr(), stream_ptr(dev)), "exl3_paged_qkv_post")
    return q_out


def _workspace(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    """Scratch of this device and stream: calls on different streams may overlap, calls on one stream run one after
    another. A captured call gets scratch of its own from the graph's pool: replays may run beside eager calls."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    ws = _workspaces.get((device.index, stream))
    if ws is None or ws.numel() < nbytes:
        ws = _workspaces[(device.index, stream)] = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws


def paged_attn(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
               cu_rows: torch.Tensor, lens: torch.Tensor, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q (rows, hq, head_dim) over the pages: row r sees positions up to its own of its sequence
    (grouped heads: head h reads kv head h // (hq // hkv)). scale defaults to 1 / sqrt(head_dim). Returns
    (rows, hq, head_dim) in q's dtype, which is the cache's. Rows at negative positions give zeros; what lies behind a
    sequence's end in its pages is never used.
    """
    rows = q.shape[0]
    b = _descriptor(k_pages, v_pages, page_table, cu_rows, lens, rows)
    dev = k_pages.device
    if q.dtype != k_pages.dtype:
        raise TypeError("q must have the cache's dtype")
    _need(q.dim() == 3 and q.shape[2] == b.head_dim and q.device == dev, "q must be (rows, hq, head_dim) on the pages' device")
    hq, hd = q.shape[1], b.head_dim
    _need(hq >= 1 and hq % b.hkv == 0 and hq // b.hkv <= 128, "hq must be a multiple of hkv, at most 128 heads per kv head")
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    _need(scale > 0 and math.isfinite(scale), "scale must be positive")
    if q.stride(2) != 1 or q.stride(1) != hd or q.stride(0) % 8 or q.stride(0) < hq * hd or q.data_ptr() % 16:
        q = q.contiguous()
    if out is None:
        out = torch.empty((rows, hq, hd), dtype=q.dtype, device=dev)
    else:
        _need(out.shape == (rows, hq, hd) and out.dtype == q.dtype and out.is_contiguous() and out.device == dev,
              "out must be contiguous (rows, hq, head_dim) in q's dtype")
    if rows == 0:
        return out
    with torch.cuda.device(dev):
        stream = stream_ptr(dev)
        need = ctypes.c_size_t()
        check(lib().exl3_paged_attn_workspace(b, hq, ctypes.byref(need)), "exl3_paged_attn_workspace")
        ws = _workspace(dev, stream, need.value)
        check(lib().exl3_paged_attn(b, q.data_ptr(), q.stride(0), hq, scale, out.data_ptr(), ws.data_ptr(), ws.numel(),
                                    _status_word(dev).data_ptr(), stream), "exl3_paged_attn")
    return out


# ------------------------------------------------------------------------------ cache and batches

class PagedBatch:
    """The rows one step feeds, as the kernels' device tables. `rows[i]` new rows of sequence i are at the end of
    its cached length `lens[i]`."""

    def __init__(self, rows: list[int], lens: list[int], pages: list[list[int]], device):
        self.rows, self.seqs, self.total_rows, self.max_rows = list(rows), len(rows), sum(rows), max(rows)
        cols = max(1, max(len(p) for p in pages))
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        flat = starts + list(lens)
        for p in pages:
            flat += p + [-1] * (cols - len(p))
        host = torch.tensor(flat, dtype=torch.int32)
        dev = torch.device(device)
        if dev.type == "cuda":
            host = host.pin_memory()
        buf = host.to(dev, non_blocking=True)                    # one copy for the three tables
        n = self.seqs
        self.cu_rows, self.lens = buf[:n + 1], buf[n + 1:2 * n + 1]
        self.page_table = buf[2 * n + 1:].view(n, cols)

    @property
    def tables(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        return self.page_table, self.cu_rows, self.lens


class PagedKVCache:
    """Pages of keys and values for all layers, (num_pages, n_kv, page_size, head_dim) each, and the sequences that
    hold them. A page is named by one index in every layer."""

    def __init__(self, n_layers: int, n_kv: int, head_dim: int, num_pages: int, page_size: int = 64, device=None,
                 dtype=torch.float16):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two, 16 or more")
        if num_pages < 1:
            raise ValueError("num_pages must be positive")
        shape = (num_pages, n_kv, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.page_size, self.num_pages = page_size, num_pages
        self.device = torch.device(device) if device is not None else self.k[0].device if self.k else torch.device("cpu")
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict = {}
        self._lens: dict = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq) -> int:
        return self._lens[seq]

    def add(self, seq) -> None:
        """A new, empty sequence under the key `seq`."""
        if seq in self._lens:
            raise ValueError(f"sequence {seq!r} is already in the cache")
        self._pages[seq], self._lens[seq] = [], 0

    def release(self, seq) -> None:
        """Forget a sequence and take its pages back."""
        self._free += reversed(self._pages.pop(seq))
        del self._lens[seq]

    def truncate(self, seq, length: int) -> None:
        """Keep the first `length` positions (drafts that were not accepted go)."""
        if not 0 <= length <= self._lens[seq]:
            raise ValueError(f"cannot cut sequence {seq!r} of {self._lens[seq]} positions to {length}")
        keep = -(-length // self.page_size)
        pages = self._pages[seq]
        self._free += reversed(pages[keep:])
        del pages[keep:]
        self._lens[seq] = length

    def extend(self, feeds: list[tuple[object, int]]) -> PagedBatch:
        """Room for `rows` new positions of each (sequence, rows); returns the batch that feeds them. Takes nothing
        and raises MemoryError if the pool has too few pages."""
        if not feeds or any(r < 1 for _, r in feeds):
            raise ValueError("extend needs at least one sequence, with one row or more each")
        if len({s for s, _ in feeds}) != len(feeds):
            raise ValueError("a sequence may be in a batch once")
        need = [-(-(self._lens[s] + r) // self.page_size) - len(self._pages[s]) for s, r in feeds]
        if sum(need) > len(self._free):
            raise MemoryError(f"the batch needs {sum(need)} pages, {len(self._free)} are free")
        for (s, r), n in zip(feeds, need):
            self._pages[s] += [self._free.pop() for _ in range(n)]
            self._lens[s] += r
        return PagedBatch([r for _, r in feeds], [self._lens[s] for s, _ in feeds], [list(self._pages[s]) for s, _ in feeds],
                          self.device)
