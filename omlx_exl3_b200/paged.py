"""Serving many sequences from one paged key/value cache.

The reference leaves the cache to oMLX and attention to the model library, one sequence at a time; this module
is the part of a server that sits between the EXL3 projections:

  PagedKVCache      pool of fixed-size pages for all layers, pages handed to sequences as they grow
  PagedBatch        what one step feeds: new rows of some sequences, as device tables the kernels read
  paged_qkv_post    q/k RMSNorm + rotary embedding + append to the pages (exl3_paged_qkv_post)
  paged_attn        attention of the new rows over the pages, chunks and single tokens alike (exl3_paged_attn)

A batch is cu_rows (seqs + 1), lens (seqs) and page_table (seqs, cols), all int32 on the device: sequence s feeds
rows cu_rows[s] .. cu_rows[s + 1] - 1 and holds lens[s] positions once they are appended, so its row i is at
position lens[s] - rows[s] + i; position p lives in page page_table[s, p // page_size]. Rows at negative positions,
rows before cu_rows[0] and rows from cu_rows[seqs] on are padding: nothing is appended and the output is zero (a captured
graph's unused slots have no rows, or lens 0). The kernels read the tables themselves, so no call waits for the host and a captured graph
follows their contents.

Calls run on the current stream. Tables that name something outside the pool, or a cu_rows that falls or passes the
call's rows, set a bit in a per-device status word, as a pipeline wait that gave up does: check_paged_status() raises on it.
"""
from __future__ import annotations

import torch

from ._lib import torch_calls


def _device_index(device: torch.device | None) -> int:
    return torch.cuda.current_device() if device is None or device.index is None else device.index


def paged_status(device: torch.device | None = None) -> int:
    """The device's status word of the paged kernels (0: nothing was out of range, no wait gave up). Waits for all of the
    device's streams."""
    index = _device_index(device)
    word = torch_calls().status(index)
    if word is None:
        return 0
    torch.cuda.synchronize(index)
    return int(word[0].item())


def check_paged_status(device: torch.device | None = None) -> None:
    """Raise RuntimeError if a paged kernel on `device` met a page, position or wait it could not serve, and clear
    the word. Waits for all of the device's streams."""
    index = _device_index(device)
    if torch_calls().status(index) is None:
        return
    torch.cuda.synchronize(index)
    value = int(torch_calls().take_status(index).item())
    if value:
        what = [t for bit, t in ((8, "a table names a page or position outside its range"),
                                 (1, "a pipeline wait timed out")) if value & bit]
        raise RuntimeError(f"paged kernels: {'; '.join(what) or 'error'} (status 0x{value:x}); the outputs of the "
                           "failed call are invalid")


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
    return torch_calls().paged_qkv_post(q, k, v, q_norm_w, k_norm_w, eps, cos, sin, k_pages, v_pages, page_table, cu_rows, lens,
                                        q_out)


def paged_attn(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
               cu_rows: torch.Tensor, lens: torch.Tensor, scale: float | None = None,
               out: torch.Tensor | None = None, max_rows: int = 0) -> torch.Tensor:
    """Attention of q (rows, hq, head_dim) over the pages: row r sees positions up to its own of its sequence
    (grouped heads: head h reads kv head h // (hq // hkv)). scale defaults to 1 / sqrt(head_dim). Returns
    (rows, hq, head_dim) in q's dtype, which is the cache's. Rows at negative positions give zeros; what lies behind a
    sequence's end in its pages is never used, whatever it is. Keys and values that a sequence does hold are taken to be
    finite: one that is not may reach rows of its own step that do not see its position. max_rows, the most rows of any
    sequence where the caller knows it, may save a launch; it changes no result.
    """
    return torch_calls().paged_attn(q, k_pages, v_pages, page_table, cu_rows, lens, scale, out, max_rows)


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
