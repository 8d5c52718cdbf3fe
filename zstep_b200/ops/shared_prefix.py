"""Attention of rows whose sequences share leading pages of the paged cache.

A ``SharedPrefixPlan`` holds which rows share which page positions.  It changes only with the
batch: while sequences grow, ``update(seq_lens)`` (once a step) and ``attend`` (once a layer)
run on the device alone, so a step can be captured in a CUDA graph.  The pages of a segment are
read once for all its rows instead of once per row.
"""

from __future__ import annotations

import torch

from . import _ext

MAX_GROUP = 64     # q heads per kv head
MAX_SEGS = 1024    # segments of a plan
MAX_PIECES = 4096  # their parts in work units
SLOTS = 128        # query slots (row x head of a GQA group) of a work unit


class SharedPrefixPlan:
    def __init__(self, slots: list[int], segments: list[tuple[list[int], int, int | None]], num_q_heads: int,
                 num_kv_heads: int, device="cuda"):
        """``slots``: page-table row of each query row.  ``segments``: (rows, first page position,
        end page position); the pages [first, end) of those rows' tables are the same, and an end
        of None means up to each row's own length.  The segments of a row must follow one another
        from position 0 to None."""
        rows = len(slots)
        if num_kv_heads < 1 or num_q_heads < 1 or num_q_heads % num_kv_heads or num_q_heads // num_kv_heads > MAX_GROUP:
            raise ValueError(f"need 1..{MAX_GROUP} q heads per kv head, got {num_q_heads} / {num_kv_heads}")
        if any(s < 0 for s in slots):
            raise ValueError("slots must not be negative")
        if len(segments) > MAX_SEGS:
            raise ValueError(f"at most {MAX_SEGS} segments, got {len(segments)}")
        order = sorted(range(len(segments)), key=lambda i: segments[i][1])  # a row's segments by position
        row_entry: list[list[int]] = [[] for _ in range(rows)]
        reach: list[int | None] = [0] * rows
        seg_rows, entry_seg, entry_piece, pieces = [], [], [], []
        room = SLOTS // (num_q_heads // num_kv_heads)   # rows of a work unit
        unit = [0, 0]                                   # first entry and rows of the last one
        units: list[int] = []                           # first piece of each
        for s, i in enumerate(order):
            members, first, end = segments[i]
            if not members:
                raise ValueError("a segment needs rows")
            if end is not None and end <= first:
                raise ValueError(f"segment [{first}, {end}) is empty")
            for r in members:
                if not 0 <= r < rows:
                    raise ValueError(f"row {r} outside the {rows} rows")
                if reach[r] is None or reach[r] != first:
                    raise ValueError(f"the segments of row {r} must follow one another from position 0")
                reach[r] = end
                row_entry[r].append(len(seg_rows))
                seg_rows.append(r)
                entry_seg.append(s)
            # Units: a segment that does not fit behind the others of the last unit starts one.
            done = len(seg_rows) - len(members)
            while done < len(seg_rows):
                left = len(seg_rows) - done
                start = not pieces or unit[1] + min(left, room) > room
                if start:
                    unit = [done, 0]
                take = min(left, room - unit[1])
                if start:
                    units.append(len(pieces))
                pieces.append((s, unit, len(units) - 1, unit[1] << 16 | unit[1] + take, first, -1 if end is None else end))
                unit[1] += take
                entry_piece += [len(pieces) - 1] * take
                done += take
        if len(pieces) > MAX_PIECES:
            raise ValueError(f"at most {MAX_PIECES} pieces of segments, got {len(pieces)}")
        if any(x is not None for x in reach):
            raise ValueError("the last segment of every row must end at None")
        self.C = _ext.load()
        self.rows, self.num_q_heads, self.num_kv_heads = rows, num_q_heads, num_kv_heads
        self.device = torch.device(device)
        self.slot_list = list(slots)
        self.max_slot = max(slots, default=0)
        self.levels = max((len(e) for e in row_entry), default=1)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        self.slots = i32(slots)
        self._num_segs = len(order)
        ends = units + [len(pieces)]
        self._segs = [i32(seg_rows), i32(entry_seg), i32(entry_piece),
                      i32([x for e in row_entry for x in e + [-1] * (self.levels - len(e))]),
                      i32([x for s, u, k, r, p0, p1 in pieces for x in (s, u[0], u[1], ends[k], ends[k + 1], r, p0, p1)])]
        self.err = torch.zeros(1, dtype=torch.int32, device=device)
        ints, floats = self.C.shared_attn_sizes(len(pieces), len(seg_rows), num_q_heads, num_kv_heads)
        self._work = torch.zeros(ints, dtype=torch.int32, device=device)
        self._partial = torch.empty(floats, dtype=torch.float32, device=device)
        self._planned = False

    @classmethod
    def from_prefixes(cls, slots: list[int], prefixes: list[tuple[list[int], int]], num_q_heads: int, num_kv_heads: int,
                      device="cuda") -> "SharedPrefixPlan":
        """Plan of rows in groups with a common prompt: (rows, whole pages that they share).  Behind
        its prefix every sequence (rows of one slot) has pages of its own; rows in no group share
        nothing."""
        first = {}
        segments: list[tuple[list[int], int, int | None]] = []
        for members, pages in prefixes:
            for r in members:
                if r in first:
                    raise ValueError(f"row {r} is in two groups")
                first[r] = pages
            if pages > 0 and members:
                segments.append((list(members), 0, pages))
        own: dict[tuple[int, int], list[int]] = {}
        for r, s in enumerate(slots):
            own.setdefault((s, first.get(r, 0)), []).append(r)
        segments += [(members, pages, None) for (_, pages), members in own.items()]
        return cls(slots, segments, num_q_heads, num_kv_heads, device)

    def update(self, seq_lens: torch.Tensor) -> None:
        """Divide a step's keys over the GPU: ``seq_lens`` [rows] int32, the keys each row sees."""
        self.C.shared_attn_plan(self.num_q_heads, self.num_kv_heads, self.slots, seq_lens, self.levels, self._num_segs, self._segs,
                                self._work, self.err)
        self._planned = True

    def attend(self, q: torch.Tensor, gate: torch.Tensor | None, k_cache: torch.Tensor, v_cache: torch.Tensor,
               page_table: torch.Tensor, seq_lens: torch.Tensor, sm_scale: float, out: torch.Tensor | None = None,
               out_q: torch.Tensor | None = None, out_sf: torch.Tensor | None = None) -> torch.Tensor | None:
        """sigmoid(gate) * attention of ``q`` [rows, heads, 256] (bf16) over its sequences' pages;
        ``gate`` None: no gate.  The result goes to ``out`` (bf16 [rows, heads * 256], allocated
        unless the MXFP8 pair ``out_q``, ``out_sf`` is given alone).  ``seq_lens`` must be what the
        last ``update`` got; a row of length 0 gives 0."""
        if q.dim() != 3 or q.shape[0] != self.rows or q.shape[1] != self.num_q_heads:
            raise ValueError(f"q must be [{self.rows}, {self.num_q_heads}, 256], got {tuple(q.shape)}")
        if not self._planned:
            raise RuntimeError("attend needs an update first")
        if page_table.dim() != 2 or page_table.shape[0] <= self.max_slot:
            raise ValueError(f"page_table must have more than {self.max_slot} rows")
        if out is None and out_q is None:
            out = torch.empty(self.rows, self.num_q_heads * 256, dtype=torch.bfloat16, device=q.device)
        self.C.shared_attn(q, gate, self.num_kv_heads, k_cache, v_cache, page_table, self.slots, seq_lens, self.levels,
                           self._num_segs, self._segs, self._work, self._partial, sm_scale, out, out_q, out_sf, self.err)
        return out

    def check(self) -> None:
        """Raise if a call since the last check met a page or length outside the cache (reads the error word)."""
        code = int(self.err.item())
        if code:
            self.err.zero_()
            raise RuntimeError(f"shared-prefix attention: kernel error status {code}")
