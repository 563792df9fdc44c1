"""What the beams of a search keep in a cache, as the list of pieces that `ops.beam_reorder` moves between two steps
(csrc/beam_reorder.cu): planes of rows of the newest page, stretches of fixed-size states, page tables."""
from __future__ import annotations

from typing import Sequence

import numpy as np
import torch

from .allocators import CacheError

_PIECE = np.dtype([("base", "<i8"), ("stride", "<i8"), ("table", "<i8"), ("units", "<i8"), ("table_width", "<i4"),
                   ("kind", "<i4"), ("bytes", "<i4"), ("vector", "<i4"), ("first", "<i4"), ("count", "<i4"), ("unused", "<i8")])
_ROWS, _STATE, _TABLE = 0, 1, 2
STATE_PIECE = 8 << 10
"""Bytes of a state that one block moves."""
ROWS_PIECE = 32
"""Rows of a plane that one block moves."""


def _vector(*numbers: int) -> int:
    """Bytes moved at a time: 16 where every address is a multiple of 16, else 4."""
    if all(number % 16 == 0 for number in numbers):
        return 16
    if all(number % 4 == 0 for number in numbers):
        return 4
    raise CacheError("rows of a cache that are no multiple of 4 bytes cannot be moved")


class CacheRows:
    """`pages`: (storage [entries, pages, ...], page table int32 [slots, pages of a slot], kv heads, key size, value size) of
    each group of paged entries; a page holds the rows of its keys, [kv heads, page_size, key size], and behind them those of
    its values (size 0: a page of keys only). `states`: tensors [slots, ...]. The list holds addresses: it is made
    anew when a tensor is."""

    def __init__(self, pages: Sequence[tuple], states: Sequence[torch.Tensor], page_size: int) -> None:
        self.page_size = int(page_size)
        parts: list[np.ndarray] = []
        device = None
        self._keep = [*states]
        for storage, table, kv_heads, key_dim, value_dim in pages:
            per_page = kv_heads * self.page_size * (key_dim + value_dim)
            if not storage.is_contiguous() or not table.is_contiguous() or table.dtype != torch.int32 or table.dim() != 2:
                raise CacheError("paged entries are contiguous, with an int32 table [slots, pages]")
            if storage.dim() < 2 or storage[0, 0].numel() != per_page:
                raise CacheError(f"a page of {kv_heads} heads x {page_size} x ({key_dim} + {value_dim}) has {per_page} values, "
                                 f"the storage's have {storage[0, 0].numel() if storage.dim() > 1 else 0}")
            self._keep += [storage, table]
            device = storage.device
            entries, n_pages, size = storage.shape[0], storage.shape[1], storage.element_size()
            for dim, behind in ((key_dim, 0), (value_dim, kv_heads * self.page_size * key_dim)):
                if dim:
                    first = np.arange(0, self.page_size, ROWS_PIECE, dtype=np.int64)
                    piece = np.zeros((entries, kv_heads, len(first)), _PIECE)
                    piece["base"] = (storage.data_ptr() + size * behind + first[None, None, :] * (dim * size)
                                     + np.arange(entries, dtype=np.int64)[:, None, None] * (n_pages * per_page * size)
                                     + np.arange(kv_heads, dtype=np.int64)[None, :, None] * (self.page_size * dim * size))
                    piece["first"], piece["count"] = first, np.minimum(ROWS_PIECE, self.page_size - first)
                    piece["stride"], piece["units"] = per_page * size, n_pages
                    piece["table"], piece["table_width"] = table.data_ptr(), table.shape[1]
                    piece["kind"], piece["bytes"] = _ROWS, dim * size
                    piece["vector"] = _vector(storage.data_ptr(), size * behind, per_page * size, self.page_size * dim * size,
                                              dim * size)
                    parts.append(piece.reshape(-1))
            piece = np.zeros(1, _PIECE)
            piece["base"], piece["stride"], piece["units"] = table.data_ptr(), 4 * table.shape[1], table.shape[0]
            piece["table_width"], piece["kind"], piece["vector"] = table.shape[1], _TABLE, 4
            parts.append(piece)
        for state in states:
            if not state.is_contiguous():
                raise CacheError("states are contiguous")
            device = state.device
            each = state.numel() // max(1, state.shape[0]) * state.element_size()
            first = np.arange(0, each, STATE_PIECE, dtype=np.int64)
            piece = np.zeros(len(first), _PIECE)
            piece["base"], piece["stride"], piece["units"] = state.data_ptr() + first, each, state.shape[0]
            piece["kind"], piece["bytes"] = _STATE, np.minimum(STATE_PIECE, each - first)
            piece["vector"] = _vector(state.data_ptr(), each)
            parts.append(piece)
        if not parts:
            raise CacheError("a cache without paged entries and without states keeps nothing that beams could take over")
        everything = np.concatenate(parts)
        self.n_pieces = len(everything)
        host = torch.from_numpy(everything.view(np.int64).reshape(self.n_pieces, 8))
        self.pieces = host.to(device) if device.type == "cuda" else host
