"""The paged serving tick's operators written out in 64 bits, one token, page and
row at a time, for the tests that hold the kernels to them."""
import math

import numpy as np
import torch

PAGE = 16
QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def plan(lens, counts, table, free_pages, free_count, total):
    """page_plan on Python ints; `table` rows are lists of width entries.
    Returns (q_start, slots, positions, lens, free_count, table, denied)."""
    table = [list(r) for r in table]
    width = len(table[0])
    q_start, slots, positions, after, denied = [0], [-1] * total, [-1] * total, [], []
    for c in counts:
        q_start.append(q_start[-1] + max(c, 0))
    top, asked = free_count, 0
    for s, (n, c) in enumerate(zip(lens, counts)):
        fits = c >= 0 and n + c <= width * PAGE and q_start[s + 1] <= total
        need = -(-(n + c) // PAGE) - -(-n // PAGE) if fits else 0
        asked += need
        if not fits or (need and asked > free_count):
            after.append(n)
            denied.append(s)
            continue
        for i in range(need):
            top -= 1
            table[s][-(-n // PAGE) + i] = free_pages[top]
        for i in range(c):
            p = n + i
            slots[q_start[s] + i] = table[s][p // PAGE] * PAGE + p % PAGE
            positions[q_start[s] + i] = p
        after.append(n + c)
    return q_start, slots, positions, after, top, table, denied


def release(lens, keep, table, free_pages, free_count):
    lens, table, free = list(lens), [list(r) for r in table], list(free_pages[:free_count])
    back = []
    for s, k in enumerate(keep):
        if 0 <= k < lens[s]:
            for p in range(-(-k // PAGE), -(-lens[s] // PAGE)):
                back.append(table[s][p])
                table[s][p] = -1
            lens[s] = k
    return lens, table, free + back[::-1]


def round_code(x, dtype):
    """x (float64, in units of the scale) to the nearest code value, ties to even."""
    if dtype == torch.int8:
        return np.clip(np.rint(x), -127, 127)
    mag = np.minimum(np.abs(x), 448.0)
    _, e = np.frexp(np.maximum(mag, 2.0 ** -6))
    step = np.ldexp(1.0, e - 4)
    return np.sign(x) * np.rint(mag / step) * step


def exponent(amax, dtype):
    e = -60
    while e < 60 and amax > QMAX[dtype] * 2.0 ** e:
        e += 1
    return e


def write(values, scales, rows, slots, dtype):
    """Write rows [N, D] (float64) at `slots` into one plane: values [tokens, D]
    (code * scale) and scales [pages], both changed in place."""
    i = 0
    while i < len(slots):
        if slots[i] < 0 or slots[i] >= values.shape[0]:
            i += 1
            continue
        page, n = slots[i] // PAGE, 1
        while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] // PAGE == page:
            n += 1
        x = rows[i:i + n]
        finite = np.isfinite(x)
        e = exponent(np.abs(np.where(finite, x, 0.0)).max(), dtype)
        if slots[i] % PAGE:
            e = max(e, int(round(math.log2(scales[page]))))
            held = values[page * PAGE:(page + 1) * PAGE]
            held[:] = round_code(held / 2.0 ** e, dtype) * 2.0 ** e
        x = np.where(np.isnan(x), 0.0, np.where(finite, x, np.sign(x) * QMAX[dtype] * 2.0 ** e))
        values[slots[i]:slots[i] + n] = round_code(x / 2.0 ** e, dtype) * 2.0 ** e
        scales[page] = 2.0 ** e
        i += n


def cache_values(codes, scales):
    """code * scale in float64, [..., tokens, D]."""
    return codes.double() * scales.double().repeat_interleave(PAGE, dim=-1)[..., None]


def attention(q, k, v, table, lens, q_start, scale):
    """Per session and head in float64 from cache values k, v [H, tokens, D].
    Returns out, lse and the elementwise bounds of a kernel that sums exact
    products in 32 bits and rounds its weights to fp16:

      score       D + 4 roundings of at most sum |q k| scale: ds
      weight      2^-11 (fp16) + 2^-21 (exponential, exponent sums) + 2 ds,
                  and 2^-32 of the largest where fp16 runs out of exponent
      sums        2^-24 for each addition: 2 * n of them at most
      output      half a step of q's type
    """
    N, Hq, D = q.shape
    H = k.shape[0]
    G = Hq // H
    qd = q.double()
    out = torch.zeros(N, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((N, Hq), -math.inf, dtype=torch.float64, device=q.device)
    lse_tol = torch.zeros_like(lse)
    half = torch.finfo(q.dtype).eps / 2
    for s, n in enumerate(lens):
        a, b = q_start[s], q_start[s + 1]
        n = min(n, table.shape[1] * PAGE)
        if a == b or n <= 0:
            continue
        pos = torch.arange(n, device=q.device)
        page = table[s, pos // PAGE].long()
        good = (page >= 0) & (page < k.shape[1] // PAGE)
        at = page.clamp(0, k.shape[1] // PAGE - 1) * PAGE + pos % PAGE
        seen = (pos[None, :] <= torch.arange(n - (b - a), n, device=q.device)[:, None]) & good[None, :]
        for h in range(Hq):
            kk, vv = k[h // G, at], v[h // G, at]
            vv = torch.where(good[:, None], vv, 0.0)
            x = (qd[a:b, h] @ kk.T) * scale
            mag = (qd[a:b, h].abs() @ kk.abs().T) * abs(scale)
            x, mag = x.masked_fill(~seen, -math.inf), mag.masked_fill(~seen, 0.0)
            some = seen.any(dim=1)
            top = torch.where(some, x.amax(dim=1), 0.0)
            w = torch.exp(x - top[:, None])
            total = w.sum(dim=1)
            p = torch.where(some[:, None], w / total[:, None], 0.0)
            out[a:b, h] = p @ vv
            lse[a:b, h] = torch.where(some, top + torch.log(total), -math.inf)
            ds = (D + 4) * 2.0 ** -24 * mag.amax(dim=1, keepdim=True) + 2.0 ** -22 * (1 + top.abs()[:, None])
            rel = 2.0 ** -11 + 2.0 ** -21 + 2 * ds + 2 * n * 2.0 ** -24
            tol[a:b, h] = rel * (p @ vv.abs()) + n * 2.0 ** -32 * vv.abs().amax(dim=0) + half * out[a:b, h].abs() + 1e-30
            lse_tol[a:b, h] = (2 * ds[:, 0] + n * 2.0 ** -24 + 2.0 ** -20 * (1 + lse[a:b, h].abs())).nan_to_num(0, 0, 0)
    return out, lse, tol, lse_tol


def logits(x, tokens, token_lens, prompt_lens, rep, pres, freq, bias, mask):
    """One row at a time; bias: list of dicts, mask: bool [S, V] (allowed) or None."""
    out = x.double().clone()
    S, V = x.shape
    for r in range(S):
        said = {}
        for t in range(token_lens[r]):
            v = int(tokens[r][t])
            if 0 <= v < V:
                said[v] = said.get(v, 0) + (1 if t >= prompt_lens[r] else 0)
        for v, n in said.items():
            y = float(out[r, v])
            y = y / rep[r] if y > 0 else y * rep[r]
            out[r, v] = y - (freq[r] * n + pres[r]) if n else y
        for v, b in bias[r].items():
            if 0 <= v < V:
                out[r, v] += b
    if mask is not None:
        out[~mask] = -math.inf
    return out
