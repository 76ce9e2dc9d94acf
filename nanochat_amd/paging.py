"""The page bookkeeping of a server's slots on the GPU (csrc/paging.hip): the block tables, lengths and free pages that
`attention.qk_norm_rope_append_packed`, `attention.packed_attention`, `attention.decode_step` and their like read, kept
and changed in device memory.

A step: `extend` gives every slot its new tokens' pages and the step's packed rows their positions and cache slots; the
append and the attention read what it returns; `trim` takes back what a slot no longer needs (a finished request: keep 0;
rejected draft tokens: the accepted length). Nothing synchronizes, so a step can be captured into a graph and replayed
with other token counts. (The reference's slots own fixed contiguous caches, model/kernels/decode.cu:740-763.)"""
from typing import NamedTuple

import torch

from .config import PAGE_SIZE
from .kv_cache import _require
from .native import check, device_guard, hip_library, pointer, stream

MAX_SLOTS = 4096
MAX_PAGES = (2 ** 31 - 1) // PAGE_SIZE   # pages of a pool or a table row: 16 times them fit an int32


class StepMaps(NamedTuple):
    """The packed rows of one step, int32 on the device. Slot b's new tokens are rows cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1, in position order; rows past cu_seqlens[-1] hold -1 in positions and slot_map."""
    cu_seqlens: torch.Tensor   # [slots + 1]
    positions: torch.Tensor    # [rows]: the row's position in its sequence
    slot_map: torch.Tensor     # [rows]: the row's cache slot, 16 page + position % 16
    granted: torch.Tensor      # [slots]: the tokens a slot was given, all it asked or 0


class BlockTables:
    """The block tables of `slots` sequences over one pool of `num_pages` pages, at most `max_pages` a sequence.

    table int32 [slots, max_pages] (-1: no page), lengths int32 [slots] (tokens a slot holds, those of the last extend
    included: the seq_lens of the attention calls), free_pages int32 [num_pages] (its first free_count entries are free,
    the last of them is taken next) and free_count int32 [1]. All start empty and free. Calls on one object are ordered by
    their stream; two that overlap on different streams race."""

    def __init__(self, slots: int, max_pages: int, num_pages: int, device):
        if not 0 < slots <= MAX_SLOTS:
            raise ValueError(f"slots must be in [1, {MAX_SLOTS}], got {slots}")
        if not (0 < max_pages <= MAX_PAGES and 0 < num_pages <= MAX_PAGES):
            raise ValueError(f"max_pages and num_pages must be in [1, {MAX_PAGES}], got {max_pages} and {num_pages}")
        self.slots, self.max_pages, self.num_pages = slots, max_pages, num_pages
        self.table = torch.full((slots, max_pages), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(slots, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)
        self._arrived = torch.zeros(1, dtype=torch.int32, device=device)   # zero between launches
        for name in ("table", "lengths", "free_pages", "free_count"):
            _require(getattr(self, name), name, torch.int32)

    def _per_slot(self, t: torch.Tensor, name: str) -> None:
        if (t.get_device() != self.table.get_device() or t.dtype != torch.int32 or t.shape != (self.slots,) or
                not t.is_contiguous()):
            _require(t, name, torch.int32)
            raise ValueError(f"{name} must be [{self.slots}] on {self.table.device}, got {tuple(t.shape)} on {t.device}")

    def extend(self, new_tokens: torch.Tensor, rows: int, maps: StepMaps | None = None) -> StepMaps:
        """Every slot b grows by new_tokens[b] (int32 [slots]; negative: 0), all or nothing, and the step's `rows` packed
        rows get their places. Slots are served in order: pages as long as the pool has them (from the first slot that it
        cannot serve on, those that need a page get nothing), then rows as long as there are any. A slot whose length
        would pass max_pages * 16 gets nothing. maps, when given, is written and returned."""
        self._per_slot(new_tokens, "new_tokens")
        if not 0 < rows < 2 ** 31:
            raise ValueError(f"rows must be in [1, 2^31), got {rows}")
        sizes = (self.slots + 1, rows, rows, self.slots)
        if maps is None:   # one allocation
            maps = StepMaps(*torch.empty(sum(sizes), dtype=torch.int32, device=self.table.device).split(sizes))
        else:
            for (name, t), n in zip(maps._asdict().items(), sizes):
                _require(t, name, torch.int32)
                if t.shape != (n,) or t.device != self.table.device:
                    raise ValueError(f"{name} must be [{n}] on {self.table.device}, got {tuple(t.shape)} on {t.device}")
                if t.data_ptr() < new_tokens.data_ptr() + 4 * self.slots and new_tokens.data_ptr() < t.data_ptr() + 4 * n:
                    raise ValueError(f"{name} must not share memory with new_tokens, which is read while it is written")
        with device_guard(self.table):
            check(hip_library().nc_pages_extend(
                pointer(new_tokens), self.slots, pointer(self.lengths), pointer(self.table), self.max_pages,
                pointer(self.free_pages), pointer(self.free_count), self.num_pages, rows, *(pointer(t) for t in maps),
                pointer(self._arrived), stream()))
        return maps

    def trim(self, keep: torch.Tensor) -> None:
        """Every slot b longer than keep[b] (int32 [slots]) falls back to that length, and the pages past it are free
        again (0 releases the slot); a negative or longer keep[b] leaves it as it is. A trim back to the lengths before an
        extend undoes it, the free list's order included."""
        self._per_slot(keep, "keep")
        with device_guard(self.table):
            check(hip_library().nc_pages_trim(
                pointer(keep), self.slots, pointer(self.lengths), pointer(self.table), self.max_pages,
                pointer(self.free_pages), pointer(self.free_count), self.num_pages, pointer(self._arrived), stream()))
