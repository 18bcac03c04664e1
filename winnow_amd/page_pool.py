"""Paged KV pool of the packed decode path: one set of page tensors for every layer,
per-request leases, generation-checked page references and fenced recycling.

The API and its exceptions are those of ``turboquant_kv/page_pool.py:30-175``
(``PoolExhausted``, ``StalePage``, ``PageRef``, ``default_fence``, ``PagePool`` with
``bytes``, ``bytes_per_token``, ``stats``, ``held``, ``pages_for``, ``ensure``,
``release``, ``reclaim``, ``validate``). The page tensors have the reference's shapes
and byte format (page_pool.py:73-78), so packed codes compare byte for byte:

    k_pages, v_pages   (layers, P, Hkv, S, NB) uint8   (dense pools: (layers, P, Hkv, S, D)
    k_norms, v_norms   (layers, P, Hkv, S)     fp16     of dense_dtype, and no norms)

Page id ``p`` addresses ``k_pages[layer, p]`` in every layer, so a request takes pages
once per token span, not once per layer. On MI355X the tensors sit in HBM: one
32k-token Llama-3-8B layer at 4 bits is 264 MiB with norms, and a full 32-layer pool
for 16 such sequences is 16.5 GiB of the 288 GB.

Bookkeeping:

* Page state is two numpy arrays indexed by page id: the holder (the integer id of a
  lease, -1 while the page is free or waits for its fence) and the generation. A
  lease is validated with one vectorised comparison.
* Free pages are a bitmap. A grant takes the lowest-numbered free pages, so a fresh
  pool gives each request a contiguous run of pages (a contiguous page-table row).
* ``release`` revokes a lease at once (generation + 1, holder -1), so any launch
  still holding its refs fails ``validate``. Its pages wait as one retirement batch
  behind one fence, recorded after the last launch that read them, and return to the
  bitmap when that fence has completed. Refusing (``PoolExhausted``) replaces
  eviction; one request is capped at ``max_pages_per_request``.
* ``batch_table`` turns the leases of a forward's sequences into the
  ``(B, width)`` int32 page table (-1 past a sequence's pages), the start positions
  and the lengths after the forward, in one pass, and ``PageTable.to`` uploads all
  three with a single host-to-device copy. The host copies stay beside the device
  ones, so metadata range checks never read device memory.
"""
from __future__ import annotations

import threading
from dataclasses import dataclass
from functools import partial

import numpy as np
import torch


class PoolExhausted(RuntimeError):
    """Not enough free pages; the caller should refuse or queue the request."""


class StalePage(RuntimeError):
    """A launch referenced a page its caller no longer owns."""


@dataclass(frozen=True)
class PageRef:
    """A page id and the generation it had when granted."""

    page: int
    generation: int


class _Done:
    """Fence of work that has already finished (pools on the host)."""

    def query(self) -> bool:
        return True

    def synchronize(self) -> None:
        pass


def default_fence(device):
    """A HIP event recorded on the device's current stream; a completed fence on the host."""
    device = torch.device(device)
    if device.type != "cuda":
        return _Done()
    ev = torch.cuda.Event()
    ev.record(torch.cuda.current_stream(device))
    return ev


class _Lease:
    """The pages one owner holds, in grant order, with their generations at grant time."""

    __slots__ = ("lid", "pages", "gens")

    def __init__(self, lid: int):
        self.lid = lid
        self.pages = np.empty(0, np.int64)
        self.gens = np.empty(0, np.int64)

    def refs(self) -> list[PageRef]:
        return [PageRef(int(p), int(g)) for p, g in zip(self.pages, self.gens)]


@dataclass
class PageTable:
    """Page metadata of one forward over B sequences appending ``n_new`` tokens each.

    ``table_host`` (B, width) int32 (-1 padded), ``start_host`` (B,) the tokens stored
    before the forward, ``seq_host`` (B,) the lengths after it; ``table``, ``start``
    and ``seq`` are the device copies once ``to`` has run (the host ones until then).
    ``gens`` (B, width) are the generations of the table's pages when it was made (None for
    a table that the pool did not make).
    """

    table_host: torch.Tensor
    start_host: torch.Tensor
    seq_host: torch.Tensor
    n_new: int
    table: torch.Tensor | None = None
    start: torch.Tensor | None = None
    seq: torch.Tensor | None = None
    gens: np.ndarray | None = None

    def to(self, device) -> "PageTable":
        """Upload the three tensors with one copy (they are views of one int32 buffer)."""
        B, W = self.table_host.shape
        flat = torch.cat([self.table_host.reshape(-1), self.start_host, self.seq_host])
        if torch.device(device).type == "cuda":
            # a fresh pinned buffer that nothing writes again: the copy need not block
            dev = flat.pin_memory().to(device, non_blocking=True)
        else:
            dev = flat.to(device)
        self.table = dev[:B * W].view(B, W)
        self.start = dev[B * W:B * W + B]
        self.seq = dev[B * W + B:]
        return self


class PagePool:
    def __init__(self, *, num_layers: int, num_pages: int, num_kv_heads: int,
                 page_size: int, nb_k: int, nb_v: int, device="cpu",
                 max_pages_per_request: int | None = None, fence_factory=None,
                 dense_dtype: torch.dtype | None = None):
        """Packed pools hold uint8 rows of ``nb_k`` / ``nb_v`` bytes plus fp16 norms;
        with ``dense_dtype`` they hold unquantized rows of ``nb`` elements and no norms."""
        if min(num_layers, num_pages, num_kv_heads, page_size, nb_k, nb_v) <= 0:
            raise ValueError("pool dimensions must be positive")
        self.device = torch.device(device)
        self.num_layers, self.num_pages = num_layers, num_pages
        self.num_kv_heads, self.page_size = num_kv_heads, page_size
        self.dense = dense_dtype is not None
        lead = (num_layers, num_pages, num_kv_heads, page_size)
        elem = dense_dtype if self.dense else torch.uint8
        self.k_pages = torch.zeros(lead + (nb_k,), dtype=elem, device=self.device)
        self.v_pages = torch.zeros(lead + (nb_v,), dtype=elem, device=self.device)
        if self.dense:
            self.k_norms = self.v_norms = None
        else:
            self.k_norms = torch.zeros(lead, dtype=torch.float16, device=self.device)
            self.v_norms = torch.zeros(lead, dtype=torch.float16, device=self.device)
        self.max_pages_per_request = int(max_pages_per_request or num_pages)
        self._make_fence = fence_factory or partial(default_fence, self.device)
        self._holder = np.full(num_pages, -1, np.int64)
        self._gen = np.zeros(num_pages, np.int64)
        self._free = np.ones(num_pages, bool)
        self._retired: list[tuple[np.ndarray, object]] = []   # (pages, fence) per release
        self._leases: dict[str, _Lease] = {}
        self._next_lid = 0
        self._mu = threading.Lock()

    # -- accounting -------------------------------------------------------
    def bytes(self) -> int:
        tensors = (self.k_pages, self.v_pages, self.k_norms, self.v_norms)
        return sum(t.nelement() * t.element_size() for t in tensors if t is not None)

    def bytes_per_token(self) -> int:
        """Resident KV bytes one token costs across all layers."""
        return self.bytes() // (self.num_pages * self.page_size)

    def stats(self) -> dict:
        """Page counts by state, and the owners the pool has seen since their last release."""
        with self._mu:
            return {"free": int(self._free.sum()),
                    "pending": sum(len(p) for p, _ in self._retired),
                    "owned": int((self._holder >= 0).sum()),
                    "requests": len(self._leases), "total": self.num_pages}

    def held(self, owner: str) -> list[PageRef]:
        with self._mu:
            lease = self._leases.get(owner)
            return lease.refs() if lease is not None else []

    # -- lifecycle --------------------------------------------------------
    def pages_for(self, tokens: int) -> int:
        return -(-int(tokens) // self.page_size)

    def _lease(self, owner: str) -> _Lease:
        lease = self._leases.get(owner)
        if lease is None:
            lease = self._leases[owner] = _Lease(self._next_lid)
            self._next_lid += 1
        return lease

    def ensure(self, owner: str, tokens: int) -> list[PageRef]:
        """Grow ``owner``'s lease to cover ``tokens`` tokens, all or nothing.

        The owner is registered even when the grant is refused, so that a queued
        request can retry under the same lease; ``release`` forgets it."""
        with self._mu:
            lease = self._lease(owner)
            want = self.pages_for(tokens)
            extra = want - len(lease.pages)
            if extra > 0:
                if want > self.max_pages_per_request:
                    raise PoolExhausted(f"{owner} needs {want} pages > per-request cap "
                                        f"{self.max_pages_per_request}")
                self._reclaim_locked()
                free = np.flatnonzero(self._free)
                if free.size < extra:
                    waiting = sum(len(p) for p, _ in self._retired)
                    raise PoolExhausted(f"{owner} needs {extra} more pages, {free.size} free, "
                                        f"{waiting} awaiting fences")
                grant = free[:extra]
                self._free[grant] = False
                self._holder[grant] = lease.lid
                lease.pages = np.concatenate([lease.pages, grant])
                lease.gens = np.concatenate([lease.gens, self._gen[grant]])
            return lease.refs()

    def release(self, owner: str, fence=None) -> int:
        """Revoke ``owner``'s pages now; they return to the pool once ``fence`` completes.

        ``fence`` must complete after the last launch that read the pages; by default
        an event is recorded on the current stream here."""
        fence = self._make_fence() if fence is None else fence
        with self._mu:
            lease = self._leases.pop(owner, None)
            if lease is None or lease.pages.size == 0:
                return 0
            self._revoke(lease.pages)
            self._retired.append((lease.pages, fence))
            self._reclaim_locked()
            return int(lease.pages.size)

    def _revoke(self, pages: np.ndarray) -> None:
        """Invalidate every outstanding ref of ``pages`` (holder cleared, generation + 1)."""
        self._gen[pages] += 1
        self._holder[pages] = -1

    def reclaim(self) -> int:
        with self._mu:
            return self._reclaim_locked()

    def _fence_done(self, fence) -> bool:
        return bool(fence.query())

    def _reclaim_locked(self) -> int:
        back = 0
        waiting = []
        for pages, fence in self._retired:
            if self._fence_done(fence):
                self._free[pages] = True
                back += int(pages.size)
            else:
                waiting.append((pages, fence))
        self._retired = waiting
        return back

    def _holder_name(self, lid: int):
        return next((o for o, lease in self._leases.items() if lease.lid == lid), None)

    def validate(self, owner: str, refs) -> None:
        """Raise ``StalePage`` unless every ref is held by ``owner`` at its generation."""
        refs = list(refs)
        if not refs:
            return
        pages = np.array([r.page for r in refs], np.int64)
        gens = np.array([r.generation for r in refs], np.int64)
        if pages.min() < 0 or pages.max() >= self.num_pages:
            raise StalePage(f"{owner} referenced a page outside [0, {self.num_pages})")
        with self._mu:
            lease = self._leases.get(owner)
            lid = lease.lid if lease is not None else -2
            bad = np.flatnonzero((self._holder[pages] != lid) | (self._gen[pages] != gens))
            if bad.size:
                p, g = int(pages[bad[0]]), int(gens[bad[0]])
                raise StalePage(f"{owner} referenced page {p} gen {g}; current owner "
                                f"{self._holder_name(int(self._holder[p]))!r} gen {int(self._gen[p])}")

    # -- per-forward metadata ---------------------------------------------
    def batch_table(self, owners, lengths, n_new: int) -> PageTable:
        """The page table of a forward appending ``n_new`` tokens to each owner's sequence.

        Every owner must hold pages for ``length + n_new`` tokens; a released or
        short lease raises ``StalePage``. Never grants pages: a forward racing a
        release must fail rather than take pages for a request that has ended."""
        lengths = [int(L) for L in lengths]
        with self._mu:
            leases = []
            for o, L in zip(owners, lengths):
                lease = self._leases.get(o)
                have = 0 if lease is None else int(lease.pages.size)
                need = self.pages_for(L + n_new)
                if need > have:
                    raise StalePage(f"{o} holds {have} pages, needs {need}")
                leases.append(lease)
            width = max([1] + [int(lz.pages.size) for lz in leases if lz is not None])
            table = np.full((len(leases), width), -1, np.int32)
            gens = np.full(table.shape, -1, np.int64)
            for b, lz in enumerate(leases):
                if lz is not None:
                    table[b, :lz.pages.size] = lz.pages
                    gens[b, :lz.pages.size] = lz.gens
        start = torch.tensor(lengths, dtype=torch.int32)
        return PageTable(torch.from_numpy(table), start, start + n_new, int(n_new), gens=gens)

    def still_held(self, owners, meta: PageTable, rows) -> None:
        """Raise ``StalePage`` unless each of the batch's ``rows`` still holds, under its owner and at
        the generations of ``meta``, the pages that the forward over ``meta`` appended to."""
        for b in rows:
            lo, hi = int(meta.start_host[b]), int(meta.seq_host[b])
            at = slice(lo // self.page_size, self.pages_for(hi))
            self.validate(owners[b], [PageRef(int(p), int(g)) for p, g in zip(meta.table_host[b, at], meta.gens[b, at])])
