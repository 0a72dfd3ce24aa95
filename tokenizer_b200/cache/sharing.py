"""Which of a step's rows have the beginnings of their caches in common: sets of rows whose block tables begin with the same
pages, as `ops.shared_prefix_attention` reads them (once a set).  Host side alone."""
from __future__ import annotations

from typing import List, Sequence, Tuple

import numpy as np


def common_beginnings(table: np.ndarray, usable: Sequence[int], least: int = 1) -> List[Tuple[List[int], int]]:
    """[(rows, pages)] of disjoint sets of at least two rows whose first `pages` table entries are the same.  `table` is
    [rows, pages], of row r the first usable[r] entries may be shared (none from a hole, -1, on).  Where a set's parts have more in common than the
    whole, it is taken whole or in parts by how many page reads that saves: (rows - 1) * pages.  Sets with fewer than
    `least` pages are left out."""
    holes = np.concatenate([np.asarray(table) < 0, np.ones((len(table), 1), dtype=bool)], axis=1)
    usable = np.minimum(np.asarray(usable, dtype=np.int64), holes.argmax(axis=1)) if len(table) else np.zeros(0, dtype=np.int64)

    def split(rows, at):
        """`rows` by their entry at place `at`, those that have one."""
        rows = rows[usable[rows] > at]
        if len(rows) < 2:
            return []
        entries = table[rows, at]
        if (entries == entries[0]).all():
            return [rows]
        return [part for value in np.unique(entries) if len(part := rows[entries == value]) > 1]

    def best(rows, at):
        """(page reads saved, sets) of rows that agree on their first `at` entries."""
        end = int(usable[rows].min())
        differs = (table[rows, at:end] != table[rows[0], at:end]).any(axis=0)
        pages = at + int(differs.argmax()) if differs.any() else end
        whole = (len(rows) - 1) * pages if pages >= least else 0
        found = [best(part, pages) for part in split(rows, pages)]
        if sum(saved for saved, _ in found) > whole:
            return sum(saved for saved, _ in found), [s for _, sets in found for s in sets]
        return whole, [(rows.tolist(), pages)] if whole else []

    if len(usable) == 0 or table.shape[1] == 0:
        return []
    return [s for part in split(np.arange(len(usable)), 0) for s in best(part, 0)[1]]


def plan(table: np.ndarray, usable: Sequence[int], page_size: int, tile_members: int, least: int = 1):
    """(shared [rows], members, tiles [n, 4]) as `ops.shared_prefix_attention` takes them, int32 on the host: the sets of
    `common_beginnings` cut into tiles of at most `tile_members` rows."""
    if tile_members < 1:
        raise ValueError("a tile has at least one member")
    shared = np.zeros(len(usable), dtype=np.int32)
    members: List[int] = []
    tiles = []
    for rows, pages in common_beginnings(table, usable, least):
        shared[rows] = pages * page_size
        for at in range(0, len(rows), tile_members):
            part = rows[at:at + tile_members]
            tiles.append((len(members), len(part), pages * page_size, 0))
            members += part
    return shared, np.asarray(members, dtype=np.int32), np.asarray(tiles, dtype=np.int32).reshape(-1, 4)
