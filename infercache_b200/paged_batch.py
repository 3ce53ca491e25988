"""PagedBatch: a server's sessions of growing length over one 8-bit PagePool,
with their lengths, block tables and free pages on the device.

``SessionBatch`` keeps a fixed budget of tokens per session and
``MultiSessionCache`` keeps whole sessions with host bookkeeping and 16-bit
gathers; this keeps whole sessions and attends over their pages in place, with
no host round trip in a tick, so a tick can be captured in a CUDA graph:

    plan = batch.extend(counts)                   # this tick's tokens per session
    for layer in range(n_layers):
        batch.append(layer, k, v)                 # [N, Hkv, D], session after session
        out = batch.attend(layer, q)              # [N, Hq, D]
    logits = process_logits(logits, ...)
    batch.release([0 if done else -1 for done in finished])

The reference has no counterpart (its paged sessions are gathered into
16-bit tensors for every step, paged_cache.py:365-378).
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .paged_cache import PAGE_SIZE, PagePool
from .paged_ops import PagePlan, page_plan, page_release, page_write, paged_attention

Counts = Union[Sequence[int], torch.Tensor]


class PagedBatch:
    """``max_sessions`` rows of sessions over ``pool``.

    ``pages``: the page ids the batch may hand out (default all of the pool's;
    pages leased from a ``KVAllocator`` keep it apart from other users of the
    pool); the last one is handed out first, as KVAllocator does.  A call's
    tensors belong to the current stream; one batch's calls run on one stream,
    or in an order the caller makes.
    """

    def __init__(self, pool: PagePool, max_sessions: int, max_pages_per_session: Optional[int] = None,
                 pages: Optional[Sequence[int]] = None) -> None:
        if not pool.quantised:
            raise ValueError(f"PagedBatch needs an 8-bit pool (float8_e4m3fn or int8), got {pool.cfg.dtype}")
        width = pool.cfg.max_pages_per_session if max_pages_per_session is None else int(max_pages_per_session)
        if not 1 <= max_sessions <= 4096 or width < 1:  # paged_attention's limit
            raise ValueError("max_sessions must be in [1, 4096] and max_pages_per_session positive")
        ids = list(range(pool.cfg.n_pages)) if pages is None else [int(p) for p in pages]
        if len(set(ids)) != len(ids) or any(not 0 <= p < pool.cfg.n_pages for p in ids):
            raise ValueError(f"pages must be distinct ids in [0, {pool.cfg.n_pages})")
        dev = pool.device
        self.pool, self.device, self.max_sessions, self.width = pool, dev, int(max_sessions), width
        self.lens = torch.zeros(self.max_sessions, dtype=torch.int32, device=dev)
        self.block_table = torch.full((self.max_sessions, width), -1, dtype=torch.int32, device=dev)
        self.free_pages = torch.tensor(ids, dtype=torch.int32, device=dev)
        self.free_count = torch.tensor([len(ids)], dtype=torch.int32, device=dev)
        self.dev_status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.plan: Optional[PagePlan] = None
        # one layer's views, so that a call does not slice
        self._k, self._v = list(pool.K.unbind(0)), list(pool.V.unbind(0))
        self._ks, self._vs = list(pool.k_scale.unbind(0)), list(pool.v_scale.unbind(0))

    def _ints(self, name: str, x: Counts) -> torch.Tensor:
        if isinstance(x, torch.Tensor):
            if x.shape != (self.max_sessions,) or x.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"{name} must be an int32 or int64 [{self.max_sessions}] tensor")
            if x.dtype == torch.int64:  # more than 32 bits hold is more than any session holds
                x = x.clamp(-2 ** 31, 2 ** 31 - 1)
            return x.to(self.device, torch.int32).contiguous()
        if len(x) != self.max_sessions:
            raise ValueError(f"{name} must have {self.max_sessions} entries, got {len(x)}")
        return torch.tensor(list(x), dtype=torch.int32).to(self.device, non_blocking=True)

    def extend(self, counts: Counts, total: Optional[int] = None, max_count: Optional[int] = None,
               commit: bool = True) -> PagePlan:
        """Take ``counts[s]`` (>= 0) new tokens for every session: pages, slots
        and positions (``page_plan``).  Counts on the host give ``total`` and
        ``max_count`` themselves; device counts need ``total``, their sum.
        A session that finds no pages keeps its length, and attend() gives its
        tokens' rows of that tick no meaning (check_device_status reports it).
        Without ``commit`` the lengths stay as they were until ``commit_plan``,
        and the next ``extend`` or ``release`` drops the plan."""
        if not (isinstance(counts, torch.Tensor) and counts.is_cuda):
            host = counts.tolist() if isinstance(counts, torch.Tensor) else [int(c) for c in counts]
            if any(c < 0 for c in host):
                raise ValueError("counts must be >= 0")
            total = sum(host) if total is None else total
            max_count = max(host, default=0) if max_count is None else max_count
        elif total is None:
            raise ValueError("counts on the device need total, their sum")
        self.plan = page_plan(self.lens, self._ints("counts", counts), self.block_table, self.free_pages,
                              self.free_count, total, max_count=max_count, commit=commit, status=self.dev_status)
        return self.plan

    def commit_plan(self) -> None:
        """Make the last ``extend(..., commit=False)`` the batch's state."""
        if self.plan is None:
            raise ValueError("there is no plan to commit")
        self.lens.copy_(self.plan.lens)
        self.free_count.copy_(self.plan.free_count)

    def _layer(self, layer: int) -> Tuple[torch.Tensor, ...]:
        if self.plan is None:
            raise ValueError("extend() comes before append() and attend()")
        if not 0 <= layer < len(self._k):
            raise ValueError(f"layer must be in [0, {len(self._k)}), got {layer}")
        return self._k[layer], self._v[layer], self._ks[layer], self._vs[layer]

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Quantise the plan's tokens' K/V [N, Hkv, D] into ``layer``'s pages."""
        page_write(k, v, *self._layer(layer), self.plan.slots, status=self.dev_status)

    def attend(self, layer: int, q: torch.Tensor, *, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
               return_lse: bool = False):
        """The plan's tokens' queries [N, Hq, D] over their sessions' pages
        (append the same tokens first): out [N, Hq, D]."""
        cache = self._layer(layer)
        p = self.plan
        return paged_attention(q, *cache, self.block_table, p.lens, p.q_start, scale=scale, max_count=p.max_count, out=out,
                               return_lse=return_lse, status=self.dev_status)

    def release(self, keep: Counts) -> None:
        """Session s keeps its first ``keep[s]`` tokens: 0 ends it, a negative
        number leaves it alone, others drop its newest tokens (rejected drafts).
        A dropped token that raised its page's scale leaves the page's kept tokens
        rounded to that scale's unit."""
        page_release(self.lens, self._ints("keep", keep), self.block_table, self.free_pages, self.free_count,
                     status=self.dev_status)
        self.plan = None

    def gather(self, session: int, n_tokens: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """K, V [n_layers, Hkv, n_tokens, D] of a session's first tokens, in the
        pool's value_dtype."""
        if not 0 <= session < self.max_sessions or not 0 <= n_tokens <= self.width * PAGE_SIZE:
            raise ValueError("no such session, or more tokens than a session can hold")
        return self.pool.gather_rows(self.block_table[session], n_tokens, 0, self.pool.cfg.n_layers)

    def check_device_status(self) -> None:
        """Raise for what the device reported since the last check (synchronises):
        sessions that got no pages, page ids outside the pool, infinities or NaN
        written into the pool."""
        flags = int(self.dev_status.item())
        if not flags:
            return
        self.dev_status.zero_()
        what = [text for bit, text in ((_lib.IC_DEVFLAG_NO_PAGES, "a session's tokens found no pages"),
                                       (_lib.IC_DEVFLAG_BAD_ROW, "a page id or length is out of range"),
                                       (_lib.IC_DEVFLAG_NONFINITE, "an infinity or a NaN was written"),
                                       (_lib.IC_DEVFLAG_TIMEOUT, "a device-side wait timed out")) if flags & bit]
        text = "PagedBatch: " + "; ".join(what)
        if flags == _lib.IC_DEVFLAG_NONFINITE:
            raise _lib.InvalidArgument(_lib.IC_ERR_INVALID_ARG, text)
        raise _lib.InferCacheError(_lib.IC_ERR_OUT_OF_PAGES if flags & _lib.IC_DEVFLAG_NO_PAGES else
                                   _lib.IC_ERR_CORRUPT_TABLE if flags & _lib.IC_DEVFLAG_BAD_ROW else
                                   _lib.IC_ERR_DEVICE_TIMEOUT, text)
