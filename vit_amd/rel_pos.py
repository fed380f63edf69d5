"""Where the tokens of a relative position bias are and which bucket each pair of them has (``vit_rel_pos`` of
include/vit_amd.h): the plan that ``ops.attention_rel_bias`` and its gradient take beside the learned table.

Tokens are ``prefix`` tokens without a place (CLS, registers), then a ``grid_h x grid_w`` grid in row order; a sequence is
a grid of one row. Without ``bucket_of`` every (row, column) offset has a bucket of its own, in the order
``(dy + grid_h - 1) * (2 grid_w - 1) + dx + grid_w - 1`` with ``(dy, dx) = place of the query - place of the key``, and three
more follow if there is a prefix: prefix query on a grid key, grid query on a prefix key, prefix on prefix.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib


class RelPosBuckets:
    """Buckets of a ``grid = (grid_h, grid_w)`` with ``prefix`` tokens in front.

    ``bucket_of``: the bucket of every offset index (and, with a prefix, of the three indices behind them), integers in
    ``[0, num_buckets)``; ``None``: the index itself."""

    def __init__(self, grid: Tuple[int, int], prefix: int = 0, bucket_of: Union[None, Sequence[int], torch.Tensor] = None,
                 num_buckets: Optional[int] = None, device="cuda"):
        self.grid_h, self.grid_w = (int(v) for v in grid)
        self.prefix = int(prefix)
        if self.grid_h < 1 or self.grid_w < 1 or self.grid_h * self.grid_w > 16384:
            raise ValueError(f"RelPosBuckets: bad grid {self.grid_h} x {self.grid_w}")
        if not 0 <= self.prefix <= 32:
            raise ValueError(f"RelPosBuckets: prefix must be in [0, 32], got {self.prefix}")
        self.device = torch.device(device)
        self.seq = self.prefix + self.grid_h * self.grid_w
        self.offsets = (2 * self.grid_h - 1) * (2 * self.grid_w - 1)
        self.indices = self.offsets + (3 if self.prefix else 0)
        self.bucket_of = self.by_bucket = self.bucket_start = None
        if bucket_of is None:
            self.num_buckets = self.indices if num_buckets is None else int(num_buckets)
            if self.num_buckets < self.indices:
                raise ValueError(f"RelPosBuckets: {self.num_buckets} buckets without a map for {self.indices} offset indices")
        else:
            m = torch.as_tensor(bucket_of).detach()
            if m.is_floating_point() or m.is_complex() or m.dtype == torch.bool:
                raise TypeError(f"RelPosBuckets: bucket_of holds integers, got {m.dtype}")
            if m.shape != (self.indices,):
                raise ValueError(f"RelPosBuckets: bucket_of has shape {tuple(m.shape)}, expected ({self.indices},)")
            m = m.to(self.device, torch.int64)
            # the indices sorted by bucket: the order in which the gradient adds a bucket's offsets
            by = torch.sort(m, stable=True)
            self.bucket_of, self.by_bucket = m.to(torch.int32), by.indices.to(torch.int32)
            self.num_buckets = int(by.values[-1]) + 1 if num_buckets is None else int(num_buckets)
            self.bucket_start = torch.searchsorted(by.values, torch.arange(max(self.num_buckets, 0) + 1, device=self.device), out_int32=True)
            ends = by.values[::max(self.indices - 1, 1)].tolist()  # (waits for all of it: the plan may be used on any stream)
            low, high = int(ends[0]), int(ends[-1])
            if low < 0 or high >= self.num_buckets:
                raise ValueError(f"RelPosBuckets: buckets {low}..{high} outside [0, {self.num_buckets})")

    @classmethod
    def sequence(cls, n: int, num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True, device="cuda") -> "RelPosBuckets":
        """A sequence of ``n`` tokens with logarithmic buckets: distances below half of a direction's buckets have one each,
        the rest share the others up to ``max_distance`` and everything behind it the last. ``bidirectional``: half of the
        buckets for keys before the query, half for keys behind it; otherwise all keys behind it have bucket 0."""
        return cls((1, n), bucket_of=cls.log_buckets(n, num_buckets, max_distance, bidirectional), num_buckets=num_buckets, device=device)

    @staticmethod
    def log_buckets(n: int, num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True) -> list:
        """Bucket of every offset ``query - key`` from ``-(n - 1)`` to ``n - 1``."""
        per = num_buckets // 2 if bidirectional else num_buckets
        exact = per // 2
        if exact < 1 or max_distance <= exact:
            raise ValueError(f"log_buckets: {num_buckets} buckets, max_distance {max_distance}")
        out = []
        for d in range(-(n - 1), n):
            a = abs(d) if bidirectional else max(d, 0)
            if a < exact:
                b = a
            else:
                # (the small addend keeps distances on a bucket's border, whose logarithms are a rounding short, in it)
                b = min(exact + int(math.log(a / exact) / math.log(max_distance / exact) * (per - exact) + 1e-9), per - 1)
            out.append(b + (per if bidirectional and d < 0 else 0))
        return out

    def index(self) -> torch.Tensor:
        """int64 [seq, seq] on the CPU: the bucket of every (query, key)."""
        g = torch.arange(self.grid_h * self.grid_w)
        y, x = g // self.grid_w, g % self.grid_w
        at = (y[:, None] - y + self.grid_h - 1) * (2 * self.grid_w - 1) + x[:, None] - x + self.grid_w - 1
        full = torch.full((self.seq, self.seq), self.offsets + 2)
        full[:self.prefix, self.prefix:] = self.offsets
        full[self.prefix:, :self.prefix] = self.offsets + 1
        full[self.prefix:, self.prefix:] = at
        return full if self.bucket_of is None else self.bucket_of.cpu().long()[full]

    def _c(self) -> "_lib.vit_rel_pos":
        if self.bucket_of is None:
            return _lib.vit_rel_pos(self.prefix, self.grid_h, self.grid_w, self.num_buckets)
        return _lib.vit_rel_pos(self.prefix, self.grid_h, self.grid_w, self.num_buckets, self.bucket_of.data_ptr(),
                                self.by_bucket.data_ptr(), self.bucket_start.data_ptr())
