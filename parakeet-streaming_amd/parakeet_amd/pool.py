"""Page pools: FIFO free-page queue and per-slot page rings, on the host (C++ side)
or in device memory.

Replaces the reference's slot pool / dense shift buffers
(parakeet/engine/scheduler.py:68-104, parakeet/modules/cache.py:8-63): a slot
owns a ring of ``max_pages`` page ids; each step frees the pages that slid out
of its window and allocates pages for the new frames.  :class:`PagePool` does that
on the host, a step's rows are uploaded; :class:`DevicePagePool` does it in launches
(one up to 64 streams, two to 3500, four past them), so a step needs no host work and can be
recorded in a graph, and its streams may append fewer frames than a whole chunk.
"""

from __future__ import annotations

import ctypes
from ctypes import POINTER, c_int32, c_int64, c_void_p

import numpy as np
import torch

from . import ops
from ._lib import PAGE_STEP_MAX_SLOTS, check, lib


def pages_per_slot(left: int, chunk: int, page_size: int) -> int:
    """Ring entries a slot needs: a window of left+chunk frames touches at most
    (window + page_size - 2) // page_size + 1 pages."""
    window = left + chunk
    return (window + page_size - 2) // page_size + 1


def _i32p(a: np.ndarray):
    return a.ctypes.data_as(POINTER(c_int32))


class PagePool:
    """Thread-safe page allocator; every call goes to ``pk_pool_*``."""

    def __init__(
        self,
        num_slots: int,
        page_size: int,
        left: int,
        chunk: int,
        num_pages: int | None = None,
        page_order=None,
    ):
        self.num_slots = int(num_slots)
        self.page_size = int(page_size)
        self.left = int(left)
        self.chunk = int(chunk)
        self.max_pages = pages_per_slot(self.left, self.chunk, self.page_size)
        if num_pages is None:
            num_pages = self.num_slots * self.max_pages
        self.num_pages = int(num_pages)
        self.rows_stride = 1 + self.max_pages
        order_ptr = None
        if page_order is not None:
            order = np.ascontiguousarray(np.asarray(page_order, dtype=np.int32))
            if order.shape != (self.num_pages,):
                raise ValueError(f"page_order must have {self.num_pages} entries, got {order.shape}")
            self._order = order
            order_ptr = _i32p(order)
        handle = c_void_p()
        check(
            lib().pk_pool_create(
                self.num_pages,
                self.num_slots,
                self.page_size,
                self.left,
                self.chunk,
                order_ptr,
                ctypes.byref(handle),
            ),
            "pk_pool_create",
        )
        self._h = handle
        got = lib().pk_pool_max_pages(self._h)
        if got != self.max_pages:
            raise RuntimeError(f"pk_pool_max_pages {got} != {self.max_pages}")

    # -- lifetime
    def close(self) -> None:
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            lib().pk_pool_destroy(h)
            self._h = c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # -- stepping
    def advance(self, slots: np.ndarray, out: np.ndarray | None = None) -> np.ndarray:
        """Opens one step for ``slots`` (in order): evicts, allocates, returns
        int32 rows [n, 1 + max_pages] = {A, ring...} and advances each A by chunk."""
        slots = np.ascontiguousarray(slots, dtype=np.int32)
        n = int(slots.shape[0])
        if out is None:
            out = np.empty((n, self.rows_stride), dtype=np.int32)
        if out.dtype != np.int32 or not out.flags.c_contiguous or out.shape[0] < n or out.shape[1] != self.rows_stride:
            raise ValueError("advance: out must be C-contiguous int32 [n, 1 + max_pages]")
        check(lib().pk_pool_advance(self._h, n, _i32p(slots), _i32p(out), self.rows_stride), "pk_pool_advance")
        return out[:n]

    def reset_slot(self, slot: int) -> None:
        check(lib().pk_pool_reset_slot(self._h, int(slot)), "pk_pool_reset_slot")

    def reset_all(self) -> None:
        check(lib().pk_pool_reset_all(self._h), "pk_pool_reset_all")

    # -- inspection
    def free_pages(self) -> int:
        return check(lib().pk_pool_free_pages(self._h), "pk_pool_free_pages")

    def free_list(self) -> np.ndarray:
        n = self.free_pages()
        out = np.empty(max(n, 1), dtype=np.int32)
        got = check(lib().pk_pool_free_list(self._h, _i32p(out), out.shape[0]), "pk_pool_free_list")
        return out[:got].copy()

    def slot_info(self, slot: int) -> tuple[int, np.ndarray]:
        appended = c_int64()
        ring = np.empty(self.max_pages, dtype=np.int32)
        check(
            lib().pk_pool_slot_info(self._h, int(slot), ctypes.byref(appended), _i32p(ring)),
            "pk_pool_slot_info",
        )
        return int(appended.value), ring


class DevicePagePool:
    """A page pool in device memory: the rings, rows and FIFO order of
    :class:`PagePool`, advanced by ``ops.page_step`` on torch's current stream.

    The inspection methods (``free_pages``, ``free_list``, ``slot_info``) wait for the
    device; nothing else does.  Steps and resets of one pool run on one stream, or are
    ordered by the caller's events (threads included: there is no lock)."""

    def __init__(
        self,
        num_slots: int,
        page_size: int,
        left: int,
        chunk: int,
        device: torch.device,
        num_pages: int | None = None,
        page_order=None,
    ):
        self.num_slots, self.page_size = int(num_slots), int(page_size)
        self.left, self.chunk = int(left), int(chunk)
        if self.page_size <= 0 or self.page_size & (self.page_size - 1):
            raise ValueError(f"page_size {page_size} is not a power of two")
        if self.left < 0 or self.chunk <= 0 or not 0 < self.num_slots <= PAGE_STEP_MAX_SLOTS:
            raise ValueError(f"need left >= 0, chunk > 0 and 0 < num_slots <= {PAGE_STEP_MAX_SLOTS}")
        self.max_pages = pages_per_slot(self.left, self.chunk, self.page_size)
        self.num_pages = self.num_slots * self.max_pages if num_pages is None else int(num_pages)
        if self.num_pages < self.num_slots * self.max_pages:
            raise ValueError(f"{self.num_pages} pages cannot hold {self.num_slots} slots of {self.max_pages} pages each")
        if self.num_pages * self.page_size >= 1 << 31:
            raise ValueError(f"{self.num_pages} pages of {self.page_size} frames are past a slot map's 2^31 frames")
        order = np.arange(self.num_pages) if page_order is None else np.asarray(page_order)
        if order.shape != (self.num_pages,) or not np.array_equal(np.sort(order), np.arange(self.num_pages)):
            raise ValueError(f"page_order is not a permutation of 0..{self.num_pages - 1}")
        self.device = torch.device(device)
        self.state = ops.PageState(
            torch.from_numpy(order.astype(np.int32)).to(self.device),
            torch.tensor([0, self.num_pages], dtype=torch.int32, device=self.device),
            torch.zeros(self.num_slots, dtype=torch.int64, device=self.device),
            torch.full((self.num_slots, self.max_pages), -1, dtype=torch.int32, device=self.device),
            page_size=self.page_size,
            left=self.left,
            chunk=self.chunk,
        )

    def slots_tensor(self, slots) -> torch.Tensor:
        """Slot numbers checked on the host (distinct, in range) and uploaded; a device
        tensor is taken as it is (``ops.page_step`` leaves its bad entries out)."""
        if isinstance(slots, torch.Tensor) and slots.device.type == "cuda":
            return slots
        s = np.ascontiguousarray(np.asarray(slots, dtype=np.int32).reshape(-1))
        if len(np.unique(s)) != len(s) or (len(s) and (s.min() < 0 or s.max() >= self.num_slots)):
            raise ValueError(f"slots must be distinct and in [0, {self.num_slots})")
        t = torch.from_numpy(s)
        # from pinned memory, without waiting (torch keeps it until the copy has run)
        return t.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else t

    # -- stepping
    def advance(self, slots, lengths: torch.Tensor | None = None, rows=None, slot_map=None, places: bool = True):
        """One step for ``slots`` (in order): ``(rows, slot_map)`` of ``ops.page_step``."""
        return ops.page_step(self.state, self.slots_tensor(slots), lengths, rows=rows, slot_map=slot_map, places=places)

    def reset_slot(self, slot: int) -> None:
        self.reset_slots([int(slot)])

    def reset_slots(self, slots) -> None:
        """Every page of ``slots`` back to the queue, slot after slot."""
        ops.page_reset(self.state, self.slots_tensor(slots))

    def reset_all(self) -> None:
        ops.page_reset(self.state, torch.arange(self.num_slots, dtype=torch.int32, device=self.device))

    # -- inspection
    def free_pages(self) -> int:
        return int(self.state.head[1])

    def free_list(self) -> np.ndarray:
        first, n = self.state.head.tolist()
        return self.state.queue.cpu().numpy()[(first + np.arange(n)) % self.num_pages]

    def slot_info(self, slot: int) -> tuple[int, np.ndarray]:
        if not 0 <= int(slot) < self.num_slots:
            raise ValueError(f"slot {slot} out of range [0, {self.num_slots})")
        return int(self.state.appended[slot]), self.state.ring[slot].cpu().numpy()
