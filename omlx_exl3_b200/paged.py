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

from ._lib import PagedDesc, check, lib, stream_ptr

_status: dict = {}
_workspaces: dict = {}


_get_device = torch._C._cuda_getDevice
_capturing = torch._C._cuda_isCurrentStreamCapturing


def _status_word(index: int) -> int:
    """Address of the device's status word."""
    word = _status.get(index)
    if word is None:
        if _capturing():
            raise RuntimeError("call a paged kernel once on this device before capturing it in a graph")
        word = _status[index] = torch.zeros(4, dtype=torch.int32, device=torch.device("cuda", index))
    return word.data_ptr()


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


_F16, _BF16, _I32, _F32 = torch.float16, torch.bfloat16, torch.int32, torch.float32


def _descriptor(k_pages, v_pages, page_table, cu_rows, lens, rows: int) -> tuple:
    """Checked descriptor of the batch (what can be checked without reading device memory), its device, hkv and head_dim."""
    dt = k_pages.dtype
    if (dt is not _F16 and dt is not _BF16) or v_pages.dtype is not dt:
        raise TypeError("k_pages and v_pages must both be fp16 or both bf16")
    if not (page_table.dtype is cu_rows.dtype is lens.dtype is _I32):
        raise TypeError("page_table, cu_rows and lens must be int32")
    dev = k_pages.get_device()
    if dev < 0:
        raise ValueError("EXL3 kernels take CUDA tensors")
    if not (v_pages.get_device() == page_table.get_device() == cu_rows.get_device() == lens.get_device() == dev):
        raise ValueError("the pages and the batch's tables must be on one device")
    shape, table = k_pages.shape, page_table.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("pages must be (num_pages, hkv, page_size, head_dim), K and V alike")
    if len(table) != 2 or cu_rows.dim() != 1 or lens.dim() != 1:
        raise ValueError("page_table is 2-d, cu_rows and lens 1-d")
    seqs, cols = table
    if seqs < 1 or cu_rows.numel() != seqs + 1 or lens.numel() != seqs:
        raise ValueError("page_table (seqs, cols), cu_rows (seqs + 1) and lens (seqs) must agree")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("pages must be contiguous")
    if not (page_table.is_contiguous() and cu_rows.is_contiguous() and lens.is_contiguous()):
        raise ValueError("page_table, cu_rows and lens must be contiguous")
    num, hkv, ps, hd = shape
    return PagedDesc(k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), cu_rows.data_ptr(), lens.data_ptr(),
                     seqs, rows, cols, num, ps, hkv, hd, 0 if dt is _F16 else 1), dev, hkv, hd


def _row_stride(x: torch.Tensor, rows: int, width: int, name: str) -> int:
    """Row stride in elements of a (rows, width) view with contiguous rows."""
    if x.shape != (rows, width):
        raise ValueError(f"{name} must be ({rows}, {width})")
    s0, s1 = x.stride()
    if s1 == 1 and s0 >= width:
        return s0
    if rows > 1 or s1 != 1 and width > 1:
        raise ValueError(f"{name} needs contiguous, non-overlapping rows")
    return width


def _weight(w: torch.Tensor, dt: torch.dtype, hd: int, dev: int) -> int:
    if w.dtype is not dt:
        raise TypeError("norm weights must have q's dtype")
    if w.numel() != hd or not w.is_contiguous() or w.get_device() != dev:
        raise ValueError("norm weights must be contiguous (head_dim) on the pages' device")
    return w.data_ptr()


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
    rows, width = q.shape
    b, dev, hkv, hd = _descriptor(k_pages, v_pages, page_table, cu_rows, lens, rows)
    if _get_device() != dev:                      # the kernels launch on the current device
        with torch.cuda.device(dev):
            return paged_qkv_post(q, k, v, q_norm_w, k_norm_w, eps, cos, sin, k_pages, v_pages, page_table, cu_rows, lens, q_out)
    dt, kv_dt, nk = q.dtype, k_pages.dtype, hkv * hd
    if (dt is not _F16 and dt is not _BF16) or k.dtype is not dt or v.dtype is not dt:
        raise TypeError("q, k and v must all be fp16 or all bf16")
    if width == 0 or width % nk:
        raise ValueError("q's width must be a multiple of hkv * head_dim")
    hq = width // hd
    sq, sk, sv = _row_stride(q, rows, width, "q"), _row_stride(k, rows, nk, "k"), _row_stride(v, rows, nk, "v")
    if not (cos.dtype is sin.dtype is _F32):
        raise TypeError("cos and sin must be fp32")
    rope = cos.shape
    if len(rope) != 2 or sin.shape != rope or not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("cos and sin must be contiguous (positions, rotated / 2)")
    if not (q.get_device() == k.get_device() == v.get_device() == cos.get_device() == sin.get_device() == dev):
        raise ValueError("all tensors must be on one device")
    wq = None if q_norm_w is None else _weight(q_norm_w, dt, hd, dev)
    wk = None if k_norm_w is None else _weight(k_norm_w, dt, hd, dev)
    if q_out is None:
        q_out = q.new_empty((rows, hq, hd)) if kv_dt is dt else q.new_empty((rows, hq, hd), dtype=kv_dt)
    elif q_out.shape != (rows, hq, hd) or q_out.dtype is not kv_dt or not q_out.is_contiguous() or q_out.get_device() != dev:
        raise ValueError("q_out must be contiguous (rows, hq, head_dim) in the cache's dtype")
    status = lib().exl3_paged_qkv_post(b, q.data_ptr(), k.data_ptr(), v.data_ptr(), sq, sk, sv, 0 if dt is _F16 else 1, hq,
                                       wq, wk, eps, cos.data_ptr(), sin.data_ptr(), *rope, q_out.data_ptr(),
                                       _status_word(dev), stream_ptr(dev))
    if status:
        check(status, "exl3_paged_qkv_post")
    return q_out


def _workspace(index: int, stream: int, nbytes: int) -> torch.Tensor:
    """Scratch of this device and stream: calls on different streams may overlap, calls on one stream run one after
    another. A captured call gets scratch of its own from the graph's pool: replays may run beside eager calls."""
    if _capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", index))
    ws = _workspaces.get((index, stream))
    if ws is None or ws.numel() < nbytes:
        ws = _workspaces[(index, stream)] = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", index))
    return ws


_attn_bytes: dict = {}


def paged_attn(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
               cu_rows: torch.Tensor, lens: torch.Tensor, scale: float | None = None,
               out: torch.Tensor | None = None, max_rows: int = 0) -> torch.Tensor:
    """Attention of q (rows, hq, head_dim) over the pages: row r sees positions up to its own of its sequence
    (grouped heads: head h reads kv head h // (hq // hkv)). scale defaults to 1 / sqrt(head_dim). Returns
    (rows, hq, head_dim) in q's dtype, which is the cache's. Rows at negative positions give zeros; what lies behind a
    sequence's end in its pages is never used. max_rows, the most rows of any sequence where the caller knows it, may save
    a launch; it changes no result.
    """
    if q.dim() != 3:
        raise ValueError("q must be (rows, hq, head_dim)")
    rows, hq, hd = q.shape
    b, dev, hkv, head_dim = _descriptor(k_pages, v_pages, page_table, cu_rows, lens, rows)
    if _get_device() != dev:                      # the kernels launch on the current device
        with torch.cuda.device(dev):
            return paged_attn(q, k_pages, v_pages, page_table, cu_rows, lens, scale, out, max_rows)
    if q.dtype is not k_pages.dtype:
        raise TypeError("q must have the cache's dtype")
    if hd != head_dim or q.get_device() != dev:
        raise ValueError("q must be (rows, hq, head_dim) on the pages' device")
    if hq < 1 or hq % hkv or hq // hkv > 128:
        raise ValueError("hq must be a multiple of hkv, at most 128 heads per kv head")
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    elif not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive")
    s0, s1, s2 = q.stride()
    if s2 != 1 or s1 != hd or s0 % 8 or s0 < hq * hd or q.data_ptr() % 16:
        q = q.contiguous()
        s0 = hq * hd
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != (rows, hq, hd) or out.dtype is not q.dtype or not out.is_contiguous() or out.get_device() != dev:
        raise ValueError("out must be contiguous (rows, hq, head_dim) in q's dtype")
    if rows == 0:
        return out
    stream = stream_ptr(dev)
    need = _attn_bytes.get((dev, hd))
    if need is None:                              # depends on the device and the head size alone
        size = ctypes.c_size_t()
        check(lib().exl3_paged_attn_workspace(b, hq, size), "exl3_paged_attn_workspace")
        need = _attn_bytes[(dev, hd)] = size.value
    status = lib().exl3_paged_attn(b, q.data_ptr(), s0, hq, scale, max_rows, out.data_ptr(), _workspace(dev, stream, need).data_ptr(),
                                   need, _status_word(dev), stream)
    if status:
        check(status, "exl3_paged_attn")
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
