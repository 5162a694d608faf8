"""Page operations of the paged caches (no counterpart in the reference, whose sequences each
own their pages): copies inside a pool in one launch, and the host bookkeeping of forked,
truncated and compacted sequences.
"""

from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..kernels import _lib


def device_ints(values, device: torch.device) -> torch.Tensor:
    """int32 tensor of ``values`` (a list or an int32 array) on ``device``. To a ROCm device
    it goes through pinned memory, behind the work queued there, without waiting for it
    (a captured stream keeps the waiting copy, which capture refuses)."""
    t = torch.from_numpy(np.asarray(values, dtype=np.int32))
    if device.type != "cuda" or t.numel() == 0 or torch.cuda.is_current_stream_capturing():
        return t.to(device)
    return t.pin_memory().to(device, non_blocking=True)


def _check_pairs(src: Sequence[int], dst: Sequence[int], num_pages: int) -> None:
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} source pages for {len(dst)} destinations")
    for page in (*src, *dst):
        if not 0 <= page < num_pages:
            raise IndexError(f"page {page} is outside the pool of {num_pages} pages")
    onto = set(dst)
    if len(onto) != len(dst):
        raise ValueError("a destination page appears twice")
    if not onto.isdisjoint(src):
        raise ValueError("a destination page is also a source")


def fastest_flash_copy_pages(
    k_pages: torch.Tensor,
    v_pages: Optional[torch.Tensor],
    src: Sequence[int] | torch.Tensor,
    dst: Sequence[int] | torch.Tensor,
) -> None:
    """Copy page ``src[i]`` of the pools (dim 0; ``v_pages`` may be None) onto page ``dst[i]``,
    all pairs in one launch.

    Destinations have to be distinct and none of them a source. Lists are checked (IndexError,
    ValueError); int32 tensors on the pools' device are read by the kernel as they are then,
    which leaves out pairs with an id outside the pool.
    """
    if v_pages is not None and (v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype
                                or v_pages.device != k_pages.device):
        raise ValueError("k_pages and v_pages must have one shape, dtype and device")
    if k_pages.dim() < 2 or not k_pages.is_contiguous() or not (v_pages is None or v_pages.is_contiguous()):
        raise ValueError("page pools must be contiguous, pages in dim 0")
    if k_pages.device.type != "cuda":
        raise RuntimeError("fastest_flash_attention_amd copies pages on ROCm tensors only; the pool is "
                           f"on {k_pages.device}")
    device = k_pages.device
    num_pages = k_pages.size(0)
    page_bytes = k_pages.numel() // num_pages * k_pages.element_size() if num_pages else 0
    if page_bytes % 2:
        raise TypeError(f"pages of {page_bytes} bytes are not supported")
    on_device = [isinstance(x, torch.Tensor) and x.is_cuda for x in (src, dst)]
    if all(on_device):
        if not src.dtype == dst.dtype == torch.int32:
            raise TypeError("src and dst must be int32")
        if src.dim() != 1 or src.shape != dst.shape:
            raise ValueError("src and dst must be 1D and of one length")
        if src.device != device or dst.device != device:
            raise RuntimeError("src and dst must be on the pools' device")
        src, dst, n = src.contiguous(), dst.contiguous(), src.numel()
        keep = None
    elif any(on_device):
        raise TypeError("src and dst must both be lists or both be device tensors")
    else:
        src, dst = [int(x) for x in src], [int(x) for x in dst]
        _check_pairs(src, dst, num_pages)
        n = len(src)
        keep = device_ints(src + dst, device)
        src, dst = keep[:n], keep[n:]
    if n == 0 or num_pages == 0:
        return
    a = _lib.PagedCopyArgs()
    a.k_pages = k_pages.data_ptr()
    a.v_pages = v_pages.data_ptr() if v_pages is not None else None
    a.src = src.data_ptr()
    a.dst = dst.data_ptr()
    a.page_bytes = page_bytes
    a.n_pairs = n
    a.num_pages = num_pages
    _lib.launch(_lib.load().ffa_paged_copy, a, device)


class PageBook:
    """Bookkeeping of pages that sequences share, for a cache with ``free_pages``, ``sequences``
    (``{"page_table": [...], "len": n}``), ``page_size``, ``max_pages``, ``allocate_page`` and
    ``_pools``. A page of several owners is copied before one of them writes into it.
    """

    def _init_pages(self) -> None:
        self._owners: Dict[int, int] = {}  # owners of pages that have more than one

    def _pools(self) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        raise NotImplementedError

    def _release(self, page: int) -> None:
        """One owner less: a page without any goes to the tail of the free list."""
        if page < 0:  # evicted
            return
        owners = self._owners.get(page, 1)
        if owners == 1:
            self.free_pages.append(page)
        elif owners == 2:
            del self._owners[page]
        else:
            self._owners[page] = owners - 1

    def _copy(self, src: List[int], dst: List[int]) -> None:
        k, v = self._pools()
        if k.device.type == "cuda":
            fastest_flash_copy_pages(k, v, src, dst)
            return
        _check_pairs(src, dst, self.max_pages)
        k[dst] = k[src]
        if v is not None:
            v[dst] = v[src]

    def copy_pages(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Copy physical pages ``src[i]`` onto ``dst[i]``, of every pool, in one launch."""
        self._copy([int(x) for x in src], [int(x) for x in dst])

    def _own_last_pages(self, seqs: Sequence[dict]) -> None:
        """Before tokens are appended to ``seqs``: a copy of its own, of a last page that is
        not full and shared, for each of them but the page's last owner. The caller has seen
        to the free pages (``_pages_to_own``)."""
        owners: Dict[int, int] = {}  # of the shared pages, less those that get a copy
        moves = []
        for seq in seqs:
            at, part = divmod(seq["len"], self.page_size)
            page = seq["page_table"][at] if part else -1
            if owners.setdefault(page, self._owners.get(page, 1)) > 1:
                owners[page] -= 1
                moves.append((seq, at, page, self.allocate_page()))
        if not moves:
            return
        try:
            self._copy([m[2] for m in moves], [m[3] for m in moves])
        except Exception:
            self.free_pages[:0] = [m[3] for m in moves]
            raise
        for seq, at, page, own in moves:
            seq["page_table"][at] = own
            self._release(page)

    def _pages_to_own(self, seqs: Sequence[dict]) -> int:
        """Free pages that ``_own_last_pages`` takes."""
        shared: Dict[int, int] = {}
        for seq in seqs:
            at, part = divmod(seq["len"], self.page_size)
            if part and seq["page_table"][at] in self._owners:
                page = seq["page_table"][at]
                shared[page] = shared.get(page, 0) + 1
        return sum(min(n, self._owners[page] - 1) for page, n in shared.items())

    def _sequence(self, seq_id: int) -> dict:
        if seq_id not in self.sequences:
            raise KeyError(f"no sequence {seq_id}")
        return self.sequences[seq_id]

    def fork_sequence(self, src_id: int, dst_id: int) -> None:
        """A new sequence ``dst_id`` with ``src_id``'s tokens, on the same pages: nothing is
        copied until one of the two appends into a page that both hold."""
        seq = self._sequence(src_id)
        if dst_id in self.sequences:
            raise ValueError(f"sequence {dst_id} exists already")
        # (pages past the tokens, of an append that failed, stay the first one's: both would write there)
        table = seq["page_table"][:-(-seq["len"] // self.page_size)]
        for page in table:
            if page >= 0:
                self._owners[page] = self._owners.get(page, 1) + 1
        self.sequences[dst_id] = {"page_table": table, "len": seq["len"]}

    def truncate_sequence(self, seq_id: int, length: int) -> None:
        """Keep the first ``length`` tokens of a sequence; pages behind them are released."""
        seq = self._sequence(seq_id)
        if not 0 <= length <= seq["len"]:
            raise ValueError(f"length {length} is not within the sequence's {seq['len']} tokens")
        keep = -(-length // self.page_size)
        if length % self.page_size and seq["page_table"][keep - 1] < 0:
            raise ValueError(f"the page of token {length - 1} has been evicted")
        for page in seq["page_table"][keep:]:
            self._release(page)
        del seq["page_table"][keep:]
        seq["len"] = length

    def compact(self) -> int:
        """Move the sequences' pages to the lowest ids, in one launch; returns how many moved.
        The free list is in order afterwards. Block tables made before no longer hold. (Pages
        taken with ``allocate_page`` outside any sequence stay where they are.)"""
        free = set(self.free_pages)
        used = self.max_pages - len(free)
        owned = {p for seq in self.sequences.values() for p in seq["page_table"] if p >= 0}
        src = sorted(p for p in owned if p >= used)
        dst = sorted(p for p in free if p < used)[:len(src)]
        src = src[len(src) - len(dst):]
        if src:
            self._copy(src, dst)
            to = dict(zip(src, dst))
            for seq in self.sequences.values():
                seq["page_table"][:] = [to.get(p, p) for p in seq["page_table"]]
            self._owners = {to.get(p, p): n for p, n in self._owners.items()}
            free = (free - set(dst)) | set(src)
        self.free_pages[:] = sorted(free)
        return len(src)
