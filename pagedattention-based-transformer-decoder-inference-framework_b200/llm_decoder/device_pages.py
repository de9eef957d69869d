"""Pages handed out on the GPU, for steps whose lengths only the GPU knows (an accepted path, a replayed graph).

    pages = kv.pages_on_device()                    # from now on its table changes on the GPU alone
    new = pages.take(ctx, tree.node_start, tree.rows)       # room behind the context; where the rows go
    kv.append(k, v, new.positions, new.row_seq)     # or kv.append(k, v, slots=new.slots)
    ...
    pages.release(done.ctx_lens)                    # what the accepted rows do not need goes back
    pages.check()                                   # now and then: synchronises, raises where pages ran out
    pages.to_host()                                 # back to register_tile and the others"""
import collections

import numpy as np
import torch

from . import _cabi
from .host_stage import to_device

NewRows = collections.namedtuple("NewRows", "row_seq positions slots")
MOST_SEQS = 16384


class DevicePages:
    """The pages of a PageTable, of a pool of total_pages with tile_size tokens each.  Every table row has pages for its first tiles, of every
    head alike (else ValueError); `free`: the pages that are not in the table, in the order in which they are handed out from its end (default: all of
    them, the lowest first).  The table's host side (assign, lookup, KVTileCache.register_tile, ...) raises until to_host.

    All calls go to the stream that is current; calls of one object come one after the other (capture and replay included)."""

    def __init__(self, page_table, total_pages, tile_size, free=None):
        pt = page_table
        if pt.d_table_ is None:
            raise ValueError("DevicePages: a page table with dimensions")
        total_pages, tile_size = int(total_pages), int(tile_size)
        if total_pages <= 0 or tile_size <= 0 or total_pages * tile_size >= 2 ** 31:
            raise ValueError("DevicePages: pages of some tokens, fewer than 2^31 tokens in all")
        pt.on_host("DevicePages")
        pt.flush()
        table = pt.host_table_.reshape(pt.num_beams_, pt.num_heads_, pt.num_tiles_)
        mapped = table >= 0
        held = mapped[:, 0].sum(1)
        if not (mapped == (np.arange(pt.num_tiles_) < held[:, None])[:, None]).all():
            raise ValueError("DevicePages: a row's first tiles have pages, of every head alike")
        used = table[mapped]
        taken = np.zeros(total_pages, dtype=bool)           # marks, not a sort: pools have many pages
        if len(used) and used.max() < total_pages:
            taken[used] = True
        if np.count_nonzero(taken) != len(used):
            raise ValueError("DevicePages: pages of the pool, none of them twice")
        if free is None:
            free = np.flatnonzero(~taken)[::-1]
        else:
            free = np.asarray(free.cpu() if isinstance(free, torch.Tensor) else free)
            if len(free) and 0 <= free.min() <= free.max() < total_pages:
                taken[free] = True
            if np.count_nonzero(taken) != len(used) + len(free):
                raise ValueError("DevicePages: free pages are pages of the pool, none of them twice or in the table")
        self.table, self.total_pages, self.tile_size = pt, total_pages, tile_size
        self.device, self._cache = pt.d_table_.device, None
        B = pt.num_beams_
        host = np.zeros(4 + B + total_pages, dtype=np.int32)
        host[0], host[4:4 + B], host[4 + B:4 + B + len(free)] = len(free), held, free
        self._state, self._held, self._free = to_device(torch.from_numpy(host), self.device).clone().split_with_sizes([4, B, total_pages])
        pt.device_pages_ = self
        self._common = (pt.d_table_.data_ptr(), B, pt.num_heads_, pt.num_tiles_, tile_size, total_pages, self._free.data_ptr(), self._held.data_ptr(),
                        self._state.data_ptr())
        self._most, self._take, self._release = min(B, MOST_SEQS), _cabi.lib().pa_take_pages, _cabi.lib().pa_release_pages

    def _mine(self, what):
        if self.table.device_pages_ is not self:
            raise RuntimeError(f"DevicePages.{what}: the table is the host's again")

    def _vector(self, x, n, what):
        if not isinstance(x, torch.Tensor):
            if _cabi.capturing(_cabi.stream_on(self.device)):       # (a replay would copy what the staging buffer holds by then)
                raise RuntimeError(f"{what}: a tensor on {self.device} while a graph is captured")
            x = to_device(torch.as_tensor(np.asarray(x), dtype=torch.int32), self.device)
        if x.dtype is not torch.int32 or x.dim() != 1 or (n is not None and x.numel() != n) or x.device != self.device or not x.is_contiguous():
            raise ValueError(f"{what}: a contiguous int32 vector{'' if n is None else f' of {n}'} on {self.device}")
        return x

    def _sizes(self, lengths, what):
        lengths = self._vector(lengths, None, "lengths")
        if lengths.numel() > self._most:
            raise ValueError(f"DevicePages.{what}: at most {self._most} sequences")
        return lengths

    def take(self, lengths, start, rows):
        """Room for new rows start[b] .. start[b + 1] - 1 (`rows` of them in all) behind the first lengths[b] tokens of table row b, for all b below
        len(lengths): tiles that they need and that have no page get one (pa_take_pages).  lengths, start: int32 device tensors, or
        sequences of ints (not while a graph is captured).  NewRows(row_seq [rows], positions [rows], slots [rows, heads]); a slot is a row of the
        pool, or -1 where there is no page: too few pages, or more tokens than the table has tiles for, and the call hands out none (`check`)."""
        self._mine("take")
        lengths = self._sizes(lengths, "take")
        B, rows, H = lengths.numel(), int(rows), self.table.num_heads_
        start = self._vector(start, B + 1, "start")
        if rows < 0 or (rows and not B):
            raise ValueError("DevicePages.take: rows of the sequences")
        with _cabi.on_device(self.device):
            row_seq, positions, slots = torch.empty(rows * (H + 2), dtype=torch.int32, device=self.device).split_with_sizes((rows, rows, rows * H))
            _cabi.check(self._take(*self._common, lengths.data_ptr(), start.data_ptr(), B, rows, row_seq.data_ptr(),
                                                  positions.data_ptr(), slots.data_ptr(), _cabi.stream_on(self.device)), "pa_take_pages")
        return NewRows(row_seq, positions, slots.view(rows, H))

    def release(self, lengths):
        """Table row b keeps the tiles of its first lengths[b] tokens, for all b below len(lengths); the pages of the others go back
        (pa_release_pages), so that releasing what was just taken undoes it."""
        self._mine("release")
        lengths = self._sizes(lengths, "release")
        with _cabi.on_device(self.device):
            _cabi.check(self._release(*self._common, lengths.data_ptr(), lengths.numel(), _cabi.stream_on(self.device)),
                        "pa_release_pages")

    def free_pages(self):
        """Pages that can still be taken.  Synchronises."""
        return int(self._state[0])

    def check(self):
        """Raises where calls of take found too few pages since the last check.  Synchronises."""
        refused = int(self._state[1])
        if refused:
            self._state[1] = 0
            raise RuntimeError(f"DevicePages: {refused} steps found too few pages (or tiles), their rows have no place")

    def forget(self):
        """Calls that found too few pages so far count no longer."""
        self._state[1:2].zero_()

    def to_host(self):
        """The table and the free pages are the host's again.  Synchronises."""
        self._mine("to_host")
        pt, cache = self.table, self._cache
        pt.host_table_[:] = pt.d_table_.cpu().numpy()
        pt.device_pages_ = None
        free = self._free[:int(self._state[0])].tolist()
        if cache is not None:
            cache.pages_of_host(free)
        return free
