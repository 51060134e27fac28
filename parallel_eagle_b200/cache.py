"""The drafter's key/value cache for a batch of requests.

The reference runs the drafter over a request's whole context for every draft
(``src/pe/drafter.py:195-236``).  A real slot only sees real slots before it, so its keys
and values never change: :class:`DraftCache` keeps them in pages, and
:meth:`ParallelDrafter.draft_logits_cached` runs the new tokens and the prediction slots
only, for all requests together.  Requests forked from one prompt share its pages
(:meth:`DraftCache.set_prefix`).
"""

from __future__ import annotations

import torch

from . import _lib as L
from . import ops


class DraftCache:
    """Paged keys and values of ``requests`` requests (numbered from 0) of one drafter.

    ``pages`` pages of ``page`` keys (a multiple of 16) serve all requests and layers;
    ``max_len`` bounds a request's length, its prediction slots included (default: what the
    pages hold).  The host knows every length and the number of free pages, so running out
    raises :class:`PeError` before anything is launched; which pages a request holds is
    planned on the device.  A step plans twice (its rows, then without its prediction slots),
    each time from lengths that the host sends, so it cannot be captured; the operators can."""

    def __init__(self, drafter, requests: int, pages: int, page: int = 64,
                 max_len: int | None = None):
        if requests < 1 or pages < 1 or page < 16 or page % 16:
            raise ValueError(f"{requests} requests, {pages} pages of {page} keys: at least one "
                             "of each, pages a multiple of 16 keys")
        if max_len is None:
            max_len = pages * page
        if max_len < 1:
            raise ValueError(f"max_len must be positive, got {max_len}")
        dev, dtype = drafter.device, drafter.param_dtype
        if dev.type != "cuda":
            raise L.PeError("the draft cache is on CUDA only; move the drafter to a CUDA device")
        shape = (len(drafter.layers), pages, drafter.n_kv_heads, page, drafter.head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=dev)
        self.v = torch.zeros(shape, dtype=dtype, device=dev)
        self.page, self.pages = page, pages
        width = -(-max_len // page)
        self.table = torch.zeros(requests, width, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=dev)
        self._free = torch.arange(pages, dtype=torch.int32, device=dev)
        self._ring = torch.tensor([0, pages, 0], device=dev)
        #: keys of each request, shared ones included
        self.lengths = [0] * requests
        #: keys all requests share
        self.shared = 0
        self.free_pages = pages

    @property
    def requests(self) -> int:
        return len(self.lengths)

    def _own_pages(self, length: int) -> int:
        return max(0, -(-length // self.page) - self.shared // self.page)

    def resize(self, lengths: list[int]):
        """Take every request to its entry of ``lengths``, taking and giving back pages.
        Returns the new rows' ``(cu, slots, pos)`` (:func:`ops.cache_plan`)."""
        if len(lengths) != self.requests:
            raise ValueError(f"{len(lengths)} lengths for {self.requests} requests")
        most = self.table.shape[1] * self.page
        need = back = 0
        for b, (have, want) in enumerate(zip(self.lengths, lengths)):
            if not self.shared <= want <= most:
                raise L.PeError(f"request {b}: length {want}, expected {self.shared} to {most}")
            d = self._own_pages(want) - self._own_pages(have)
            need += max(d, 0)
            back += max(-d, 0)
        if need > self.free_pages:
            raise L.PeError(f"the draft cache has {self.free_pages} free pages, {need} are needed")
        rows = sum(max(0, w - h) for h, w in zip(self.lengths, lengths))
        want = torch.tensor(lengths, dtype=torch.int32).to(self.lens.device)
        with torch.cuda.device(self.lens.device):
            lens, ring = self.lens, self._ring
            self.lens, cu, slots, pos, self._ring = ops.cache_plan(
                lens, want, self.table, self._free, ring, self.page, rows, shared=self.shared)
            # they may be another stream's memory (the one the cache was used on before), which
            # must not give them to others while this stream still reads them
            stream = torch.cuda.current_stream()
            lens.record_stream(stream)
            ring.record_stream(stream)
        self.lengths = list(lengths)
        self.free_pages += back - need
        return cu, slots, pos

    def truncate(self, request: int, length: int) -> None:
        """Forget the keys of ``request`` behind ``length`` (tokens taken back)."""
        if not self.shared <= length <= self.lengths[request]:
            raise ValueError(f"request {request} holds {self.lengths[request]} keys "
                             f"({self.shared} shared), cannot keep {length}")
        self.resize([length if b == request else n for b, n in enumerate(self.lengths)])

    def finish(self, request: int) -> None:
        """Give the pages of ``request`` back, all but a shared prefix's; the number can be used
        for a new request."""
        self.truncate(request, self.shared)

    def set_prefix(self, drafter, ids: torch.Tensor, features: torch.Tensor) -> int:
        """Compute the whole pages of a prompt once, for all requests: every request then
        starts behind them.  Returns how many of its tokens they hold; the rest of the
        prompt is each request's own.  The cache has to be empty (:meth:`drop_prefix` gives
        an earlier prefix back)."""
        if any(self.lengths) or self.shared:
            raise ValueError("the shared prefix is set on an empty cache")
        n = ids.shape[0] // self.page * self.page
        if n:
            drafter.forward_cached(self, ids[:n], features[:n], [n] + [0] * (self.requests - 1), 1)
            own = self.table[0, : n // self.page].clone()
            self.table[:, : n // self.page] = own
            self.lens.fill_(n)
            self.lengths = [n] * self.requests
            self.shared = n
        return n

    def drop_prefix(self) -> None:
        """Give the shared prefix's pages back, for another one or none; every request has to
        be finished."""
        if not self.shared:
            return
        if any(n != self.shared for n in self.lengths):
            raise ValueError(f"the shared prefix of {self.shared} keys is dropped once every "
                             f"request is finished, not at lengths {self.lengths}")
        # its pages become request 0's own, which gives them back once
        self.lens[1:].zero_()
        self.lengths[1:] = [0] * (self.requests - 1)
        self.shared = 0
        self.resize([0] * self.requests)
