"""The paged serving tick on plain tensors.

A server that keeps its sessions in 8-bit pages runs, per tick,

* ``page_plan`` — the tick's token counts become pages, slots and positions on
  the device (``page_release`` gives pages back);
* ``page_write`` / ``page_read`` — a layer's new K/V quantised into pages, and
  pages back as fp16 / bf16 / fp32;
* ``paged_attention`` — the new tokens of every session attend over its pages.

``PagedBatch`` (paged_cache) keeps the state of such a server and calls these;
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

import ctypes
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


def _on(dev: torch.device, name: str, args) -> None:
    """Call an entry point with `dev` current."""
    if torch.cuda.current_device() == dev.index:
        _lib.call(name, args)
    else:
        with torch.cuda.device(dev):
            _lib.call(name, args)


def _device_of(name: str, t: torch.Tensor) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{name} runs on CUDA tensors only")
    _lib.require_device(t.device)
    return t.device


def _state(name: str, what: str, t: torch.Tensor, dev: torch.device, shape, dtype=torch.int32) -> int:
    """Data pointer of a tensor that the kernels read or write in place."""
    if t.dtype != dtype or t.device != dev or not t.is_contiguous() or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: {what} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {dev}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _status(name: str, status: Optional[torch.Tensor], dev: torch.device) -> int:
    return 0 if status is None else _state(name, "status", status, dev, (1,))


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
    dev = _device_of("page_plan", lens)
    if lens.dim() != 1 or block_table.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("page_plan: lens must be [S], block_table [S, width] and free_pages [P]")
    S, (rows, width), P = lens.shape[0], block_table.shape, free_pages.shape[0]
    total = int(total)
    if total < 0 or total > 0x7fffffff:
        raise ValueError(f"page_plan: total must be in [0, 2^31), got {total}")
    lp, cp = _state("page_plan", "lens", lens, dev, (S,)), _state("page_plan", "counts", counts, dev, (S,))
    tp = _state("page_plan", "block_table", block_table, dev, (S, width))
    fp, np_ = _state("page_plan", "free_pages", free_pages, dev, (P,)), _state("page_plan", "free_count", free_count, dev, (1,))
    # one allocation for the int32 outputs and the workspace: q_start, lens, free_count, workspace
    ints = torch.empty(4 * S + 3, dtype=torch.int32, device=dev)
    slots = torch.empty(total, dtype=torch.int32, device=dev)
    positions = torch.empty(total, dtype=torch.int64, device=dev)
    base = ints.data_ptr()
    if commit:
        lens_after, free_after, lo, fo = lens, free_count, lp, np_
    else:
        lens_after, free_after = ints[S + 1:2 * S + 1], ints[2 * S + 1:2 * S + 2]
        lo, fo = base + 4 * (S + 1), base + 4 * (2 * S + 1)
    a = _lib.ic_page_plan_args(lp, cp, tp, fp, np_, base, slots.data_ptr(), positions.data_ptr(), lo, fo,
                               base + 4 * (2 * S + 2), _status("page_plan", status, dev), S, width, total, P)
    _on(dev, "ic_page_plan", a)
    return PagePlan(ints[:S + 1], slots, positions, lens_after, free_after,
                    total if max_count is None else min(int(max_count), total))


def page_release(lens: torch.Tensor, keep: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 free_count: torch.Tensor, *, status: Optional[torch.Tensor] = None) -> None:
    """Session s keeps its first ``keep[s]`` tokens (0: none; negative, or its
    length and more: all); the pages behind them go back on the stack, in
    place (``ic_page_release``)."""
    dev = _device_of("page_release", lens)
    if lens.dim() != 1 or block_table.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("page_release: lens must be [S], block_table [S, width] and free_pages [P]")
    S, width, P = lens.shape[0], block_table.shape[1], free_pages.shape[0]
    a = _lib.ic_page_release_args(
        _state("page_release", "lens", lens, dev, (S,)), _state("page_release", "keep", keep, dev, (S,)),
        _state("page_release", "block_table", block_table, dev, (S, width)),
        _state("page_release", "free_pages", free_pages, dev, (P,)),
        _state("page_release", "free_count", free_count, dev, (1,)), _status("page_release", status, dev), S, width, P, 0)
    _on(dev, "ic_page_release", a)


def _cache_geometry(name: str, k_cache, v_cache, k_scale, v_scale):
    """(device, L, H, pool tokens, D, code) of an 8-bit cache, checked."""
    dev = _device_of(name, k_cache)
    code = _lib.CODE_DTYPE.get(k_cache.dtype)
    if code is None:
        raise ValueError(f"{name}: the cache must be float8_e4m3fn or int8, got {k_cache.dtype}")
    if k_cache.dim() not in (3, 4):
        raise ValueError(f"{name}: the cache must be [H, pool_tokens, D] or [L, H, pool_tokens, D]")
    shape = k_cache.shape
    L, (H, n, D) = (shape[0] if len(shape) == 4 else 1), shape[-3:]
    if n < PAGE_SIZE or n % PAGE_SIZE:
        raise ValueError(f"{name}: pool_tokens must be a positive multiple of {PAGE_SIZE}, got {n}")
    if v_cache.dtype != k_cache.dtype or v_cache.shape != shape or v_cache.device != dev or \
            not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError(f"{name}: k_cache and v_cache must be contiguous and alike in shape, dtype and device")
    want = shape[:-2] + (n // PAGE_SIZE,)
    for s in (k_scale, v_scale):
        if s.dtype != torch.float32 or s.shape != want or s.device != dev or not s.is_contiguous():
            raise ValueError(f"{name}: scales must be contiguous float32 tensors of shape {tuple(want)} on {dev}")
    return dev, L, H, n, D, code


def _slots(name: str, slots: torch.Tensor, dev: torch.device) -> torch.Tensor:
    if slots.dim() != 1 or slots.dtype not in (torch.int32, torch.int64) or slots.device != dev:
        raise ValueError(f"{name}: slots must be an int32 or int64 [N] tensor on {dev}")
    return slots.to(torch.int32).contiguous()


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
    ``slots[i]``; the tokens of one page stand next to each other and in order, no
    row occurs twice, and rows outside the pool are skipped.  A page is written
    in order: tokens that begin at its slot 0 start it anew, later ones keep its
    scale or raise it (the page's other codes are then rounded again).
    Infinities are stored as the largest value and NaN as zero; both set
    IC_DEVFLAG_NONFINITE in ``status``.
    """
    dev, L, H, n, D, code = _cache_geometry("page_write", k_cache, v_cache, k_scale, v_scale)
    dims = k_cache.dim()
    if k.dim() != dims or v.shape != k.shape or k.shape[-2:] != (H, D) or (dims == 4 and k.shape[0] != L):
        raise ValueError(f"page_write: k and v must be {'[L, N, H, D]' if dims == 4 else '[N, H, D]'} for a cache "
                         f"{tuple(k_cache.shape)}, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != v.dtype or k.device != dev or v.device != dev:
        raise ValueError("page_write: k and v must share the cache's device and a dtype")
    dt = _lib.dtype_code(k.dtype)
    N = k.shape[-3]
    sl = _slots("page_write", slots, dev)
    if sl.shape[0] != N:
        raise ValueError(f"page_write: {N} tokens but {sl.shape[0]} slots")
    if N == 0 or L == 0 or H == 0:
        return
    if k.stride() != v.stride() or not rows16(k) or not rows16(v):
        k, v = k.contiguous(), v.contiguous()
        if not rows16(k) or not rows16(v):  # a contiguous view that begins off a 16-byte boundary
            k, v = k.clone(), v.clone()
    st = k.stride()
    rows = _lib.ic_page_q8_rows(sl.data_ptr(), 0, k.data_ptr(), v.data_ptr(), 0, N, st[0] if dims == 4 else 0, st[-2],
                                st[-3], 0, 0)
    _q8_call("ic_page_write_q8", dev, k_cache, v_cache, k_scale, v_scale, (L, H, n, D, code), rows, dt,
             _status("page_write", status, dev))


def page_read(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
              slots: torch.Tensor, *, dtype: torch.dtype = torch.float16,
              out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """K, V of the pool rows ``slots`` as values (``ic_page_read_q8``): [H, N, D]
    for a cache [H, pool_tokens, D], [L, H, N, D] for [L, H, pool_tokens, D]; rows
    outside the pool give zeros.  ``out``: a pair of contiguous tensors to write
    into instead (``dtype`` is then theirs)."""
    dev, L, H, n, D, code = _cache_geometry("page_read", k_cache, v_cache, k_scale, v_scale)
    sl = _slots("page_read", slots, dev)
    N = sl.shape[0]
    shape = k_cache.shape[:-2] + (N, D)
    if out is None:
        _lib.dtype_code(dtype)
        out = torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev)
    for t in out:
        if t.shape != shape or t.dtype != out[0].dtype or t.device != dev or not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"page_read: out must be two contiguous, 16-byte aligned {tuple(shape)} tensors on {dev}")
    if N and L and H:
        rows = _lib.ic_page_q8_rows(sl.data_ptr(), 0, out[0].data_ptr(), out[1].data_ptr(), 0, N, H * N * D, N * D, D, 0, 0)
        _q8_call("ic_page_read_q8", dev, k_cache, v_cache, k_scale, v_scale, (L, H, n, D, code), rows,
                 _lib.dtype_code(out[0].dtype), 0)
    return out


def _q8_call(name, dev, k_cache, v_cache, k_scale, v_scale, geometry, rows, buf_dtype, status):
    L, H, n, D, code = geometry
    pool = _lib.ic_pool(k_cache.data_ptr(), v_cache.data_ptr(), n, L, H, D, code)
    a = _lib.ic_page_q8_args(pool, k_scale.data_ptr(), v_scale.data_ptr(), ctypes.pointer(rows), status, 1, 0, L, buf_dtype)
    _on(dev, name, a)


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
    ``q_start[S]`` are left as they were.
    """
    dev, _, H, n, D, code = _cache_geometry("paged_attention", k_cache, v_cache, k_scale, v_scale)
    if k_cache.dim() != 3:
        raise ValueError("paged_attention: the cache must be one layer's, [H, pool_tokens, D]")
    if q.dim() != 3 or q.shape[2] != D or H == 0 or q.shape[1] == 0 or q.shape[1] % H:
        raise ValueError(f"paged_attention: q must be [N, Hq, {D}] with Hq a multiple of {H}, got {tuple(q.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16) or q.device != dev:
        raise ValueError(f"paged_attention: q must be float16 or bfloat16 on {dev}, got {q.dtype} on {q.device}")
    if block_table.dim() != 2:
        raise ValueError("paged_attention: block_table must be [S, width]")
    (S, width), (N, Hq, _) = block_table.shape, q.shape
    tp = _state("paged_attention", "block_table", block_table, dev, (S, width))
    lp = _state("paged_attention", "lens", lens, dev, (S,))
    sp = _state("paged_attention", "q_start", q_start, dev, (S + 1,))
    if out is None:
        out = torch.empty((N, Hq, D), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"paged_attention: out must be a contiguous, 16-byte aligned {q.dtype} {tuple(q.shape)} tensor on {dev}")
    lse = torch.empty((N, Hq), dtype=torch.float32, device=dev) if return_lse else None
    if N == 0 or S == 0:
        return (out, lse) if return_lse else out
    if not rows16(q):
        q = q.clone(memory_format=torch.contiguous_format)
    a = _lib.ic_paged_attn_args(q.data_ptr(), out.data_ptr(), _lib.ptr(lse), k_cache.data_ptr(), v_cache.data_ptr(),
                                k_scale.data_ptr(), v_scale.data_ptr(), tp, lp, sp, 0, 0,
                                _status("paged_attention", status, dev), n, q.stride(0), q.stride(1), S, width, N,
                                N if max_count is None else max(0, min(int(max_count), N)), Hq, H, D,
                                _lib.DTYPE_CODE[q.dtype], code, float(D ** -0.5 if scale is None else scale))
    a.workspace_bytes = _lib.load().ic_paged_attention_workspace(ctypes.byref(a))
    if a.workspace_bytes:
        ws = torch.empty(a.workspace_bytes, dtype=torch.uint8, device=dev)
        a.workspace = ws.data_ptr()
    _on(dev, "ic_paged_attention", a)
    return (out, lse) if return_lse else out
