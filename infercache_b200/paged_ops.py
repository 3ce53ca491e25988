"""The paged serving tick on plain tensors.

A server that keeps its sessions in 8-bit pages runs, per tick,

* ``page_plan`` — the tick's token counts become pages, slots and positions on
  the device (``page_release`` gives pages back);
* ``page_write`` / ``page_read`` — a layer's new K/V quantised into pages, and
  pages back as fp16 / bf16 / fp32;
* ``paged_attention`` — the new tokens of every session attend over its pages.

``PagedBatch`` (paged_batch) keeps the state of such a server and calls these;
``process_logits`` (logits) ends the tick.  Caches are ``[H, pool_tokens, D]``
(one layer) or ``[L, H, pool_tokens, D]`` tensors of ``float8_e4m3fn`` or
``int8`` codes with float32 scales ``[..., pool_tokens / 16]``: one power of two
per page of 16 tokens and head; a stored value is code * scale.

All tensors are on one sm_100 device; work goes to torch's current stream of
that device, and nothing synchronises.  ``status`` arguments take an int32
tensor of one element into which the kernels OR their IC_DEVFLAG_* bits.  The
reference has no counterpart: its paged cache is host bookkeeping around 16-bit
rows (paged_cache.py:99-288).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib

PAGE_SIZE = 16
HEAD_DIMS = (64, 128, 256)


class PagePlan(NamedTuple):
    """What a tick's tokens became (all on the device; N = total)."""
    q_start: torch.Tensor     # int32 [S + 1]: session s owns tokens q_start[s] .. q_start[s + 1]
    slots: torch.Tensor       # int32 [N]: pool row of each token, -1 where its session was denied
    positions: torch.Tensor   # int64 [N]: position in its session, -1 likewise
    lens: torch.Tensor        # int32 [S]: lengths after the tick
    free_count: torch.Tensor  # int32 [1]: free pages after the tick
    max_count: int            # the most tokens one session may have in this plan


def page_plan(lens: torch.Tensor, counts: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
              free_count: torch.Tensor, total: int, *, max_count: Optional[int] = None, commit: bool = False,
              status: Optional[torch.Tensor] = None) -> PagePlan:
    """Pages, slots and positions of a tick's new tokens (``ic_page_plan``).

    ``lens`` int32 [S] tokens held, ``counts`` int32 [S] tokens to add,
    ``block_table`` int32 [S, width], ``free_pages`` int32 [P] of which the
    first ``free_count`` (int32 [1]) are a stack of free pages; ``total`` is the
    sum of the counts (on the host: it sizes the outputs).  Sessions take their
    pages in order, all or none; one that does not fit (see the header) keeps
    its length, its tokens get slot -1 and ``status`` IC_DEVFLAG_NO_PAGES.
    New pages are entered into ``block_table``; with ``commit`` the new lengths
    and stack height replace ``lens`` and ``free_count``, otherwise they are
    returned alone and the plan can be dropped.
    """
    q_start, slots, positions, after, free = _lib.binding().page_plan(lens, counts, block_table, free_pages, free_count,
                                                                      total, commit, status)
    return PagePlan(q_start, slots, positions, after, free, total if max_count is None else min(max_count, total))


def page_release(lens: torch.Tensor, keep: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 free_count: torch.Tensor, *, status: Optional[torch.Tensor] = None) -> None:
    """Session s keeps its first ``keep[s]`` tokens (0: none; negative, or its
    length and more: all); the pages behind them go back on the stack, in
    place (``ic_page_release``)."""
    _lib.binding().page_release(lens, keep, block_table, free_pages, free_count, status)


def rows16(t: torch.Tensor) -> bool:
    """Whether every row (last dim) of t starts on a 16-byte boundary and is contiguous."""
    e = t.element_size()
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
        s * e % 16 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)


def page_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, slots: torch.Tensor, *, status: Optional[torch.Tensor] = None) -> None:
    """Quantise K/V rows into pages (``ic_page_write_q8``).

    ``k``, ``v`` [N, H, D] into a cache [H, pool_tokens, D], or [L, N, H, D] into
    [L, H, pool_tokens, D]; fp32, fp16 or bf16, any strides (rows that are not
    contiguous and 16-byte aligned are copied first).  Token i goes to pool row
    ``slots[i]``; the tokens of one page stand next to each other and in order (slots
    may be left out), no row occurs twice, and rows outside the pool are skipped
    (not from among a page's tokens).  A page is written
    in order: tokens that begin at its slot 0 start it anew, later ones keep its
    scale or raise it (the page's other codes are then rounded again; the errors sum
    to at most one step of the last unit, see the header).
    Infinities are stored as the largest value and NaN as zero; both set
    IC_DEVFLAG_NONFINITE in ``status``.
    """
    _lib.binding().page_write(k, v, k_cache, v_cache, k_scale, v_scale, slots, status)


def page_read(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
              slots: torch.Tensor, *, dtype: torch.dtype = torch.float16,
              out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """K, V of the pool rows ``slots`` as values (``ic_page_read_q8``): [H, N, D]
    for a cache [H, pool_tokens, D], [L, H, N, D] for [L, H, pool_tokens, D]; rows
    outside the pool give zeros.  ``out``: a pair of contiguous tensors to write
    into instead (``dtype`` is then theirs)."""
    k, v = (None, None) if out is None else out
    return _lib.binding().page_read(k_cache, v_cache, k_scale, v_scale, slots, _lib.dtype_code(dtype), k, v)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, q_start: torch.Tensor, *,
                    scale: Optional[float] = None, max_count: Optional[int] = None, out: Optional[torch.Tensor] = None,
                    return_lse: bool = False, status: Optional[torch.Tensor] = None):
    """Causal attention of every session's newest tokens over its 8-bit pages
    (``ic_paged_attention``).

    ``q`` [N, Hq, D] (fp16 / bf16, D 64, 128 or 256; rows of heads may be
    strided): session s owns tokens ``q_start[s]`` .. ``q_start[s + 1]`` (int32
    [S + 1]), the last ones of its ``lens[s]`` (int32 [S], this tick's tokens
    among them), whose pages are ``block_table[s]`` (int32 [S, width]).  The
    cache is one layer's, [Hkv, pool_tokens, D]; query head h reads KV head
    h // (Hq / Hkv).  ``max_count`` bounds the tokens of one session (default N)
    and only steers the choice of kernel.  Returns out [N, Hq, D] in q's dtype,
    with ``return_lse`` also the float32 [N, Hq] natural-log log-sum-exp.  A
    query with nothing to attend over gets zeros and -inf; rows of ``out`` past
    ``q_start[S]`` are left as they were.  ``out`` is ``q`` or does not overlap it.
    """
    return _lib.binding().paged_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, lens, q_start, scale,
                                          max_count, out, return_lse, status)
