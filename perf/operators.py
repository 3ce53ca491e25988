"""Cases and plain forms of the paged serving tick's operators.

One tick of a server that keeps its sessions in a page pool is, in order:
``page_plan`` (the tick's token counts become pages, slots and positions),
``page_write`` (each layer's new K/V quantised into 8-bit pages with one scale
per page and head; ``page_read`` gives pages back as 16-bit values),
``paged_attention`` (the new tokens attend over the pages) and
``process_logits`` (penalties, biases and the grammar's mask).

``run`` computes each in plain torch (``own`` false) or through
infercache_b200 (``own`` true); ``exact`` computes them again in 64 bits.
"""
import math
import zlib

import torch

own = False

PAGE = 16
QMAX = {"e4m3": 448.0, "int8": 127.0}
DTYPE = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
E_MIN, E_MAX = -60, 60  # range of a page scale's exponent


# ---- cases ----------------------------------------------------------------------
def listed():
    return [
        # one chat session's layer: the shortest wait between two tokens
        dict(name="attend-1x300", kind="attend", sessions=1, len_lo=300, len_hi=300, count_lo=1, count_hi=1,
             heads=2, group=8, dim=128, codes="e4m3", dtype="fp16"),
        # the 16 sessions of the decode benchmark, 2048-token prompts and up to 512 tokens more
        dict(name="attend-16x2k", kind="attend", sessions=16, len_lo=2049, len_hi=2560, count_lo=1, count_hi=1,
             heads=2, group=8, dim=128, codes="int8", dtype="bf16"),
        # the 64 sessions of the 7B-shaped decode, prompts of 1024 to 8192 tokens
        dict(name="attend-64x8k", kind="attend", sessions=64, len_lo=1024, len_hi=8192, count_lo=1, count_hi=1,
             heads=4, group=7, dim=128, codes="e4m3", dtype="bf16"),
        # one long document: a single row of work that has to be split to fill the GPU
        dict(name="attend-1x128k", kind="attend", sessions=1, len_lo=131071, len_hi=131071, count_lo=1, count_hi=1,
             heads=2, group=8, dim=128, codes="int8", dtype="fp16"),
        # verification of drafted tokens: a few query tokens for each session
        dict(name="attend-draft", kind="attend", sessions=24, len_lo=256, len_hi=4096, count_lo=2, count_hi=6,
             heads=2, group=4, dim=64, codes="e4m3", dtype="bf16"),
        # chunked prefill: prompts arriving in chunks on top of what the cache holds
        dict(name="attend-chunk", kind="attend", sessions=4, len_lo=4096, len_hi=8192, count_lo=1500, count_hi=2048,
             heads=2, group=8, dim=128, codes="e4m3", dtype="bf16"),
        # a decode tick's write of one layer: one token in each of 64 sessions' last pages
        dict(name="write-64x1", kind="write", sessions=64, layers=1, len_lo=1024, len_hi=8192, count_lo=1, count_hi=1,
             heads=4, dim=128, codes="e4m3", dtype="bf16"),
        # 16 prompts of 2048 tokens written into all 36 layers and handed back in 16 bits
        dict(name="write-16x2k", kind="write", sessions=16, layers=36, len_lo=2048, len_hi=2048, count_lo=2048,
             count_hi=2048, heads=2, dim=128, codes="int8", dtype="fp16"),
        # a decode tick of 16 sessions
        dict(name="plan-16", kind="plan", sessions=16, len_lo=2048, len_hi=2560, count_lo=1, count_hi=1, width=256,
             spare=1.0),
        # admission of 512 prompts of 256 to 32768 tokens
        dict(name="plan-512", kind="plan", sessions=512, len_lo=0, len_hi=0, count_lo=256, count_hi=32768, width=2048,
             spare=1.1),
        # one session's sampler: a repetition penalty over what it has generated
        dict(name="logits-1", kind="logits", sessions=1, vocab=151936, dtype="fp32", history=256, prompt=0.0,
             bias=0, mask=False),
        # a batch with everything on: penalties over prompt and answer, biases, a grammar's mask
        dict(name="logits-64", kind="logits", sessions=64, vocab=151936, dtype="bf16", history=2048, prompt=0.5,
             bias=64, mask=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "write", "plan", "logits"])
    if kind == "attend":
        heads, group, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), rng.choice([64, 128, 128, 256])
        sessions = _log_int(rng, 1, 96)
        count = rng.choice([1, 1, 1, _log_int(rng, 1, 16), _log_int(rng, 1, 1024)])
        top = 1_500_000 * 128 // (sessions * heads * dim)
        top = min(top, 131072, max(1, 400_000_000 // (sessions * heads * group * count)))
        hi = max(count + 1, _log_int(rng, 2, max(2, top)))
        lo = max(count, _log_int(rng, 1, hi))
        return dict(kind=kind, sessions=sessions, len_lo=lo, len_hi=hi, count_lo=rng.choice([0, 1, count]) if count > 1 else 1,
                    count_hi=count, heads=heads, group=group, dim=dim, codes=rng.choice(["e4m3", "int8"]),
                    dtype=rng.choice(["fp16", "bf16"]))
    if kind == "write":
        heads, dim, layers = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 128, 256]), rng.choice([1, 1, 2, 28, 36])
        sessions = _log_int(rng, 1, 256)
        top = max(1, min(8192, 2_000_000 * 128 // (sessions * heads * dim * layers)))
        count = rng.choice([1, _log_int(rng, 1, top)])
        lo = rng.randint(1, 64)
        return dict(kind=kind, sessions=sessions, layers=layers, len_lo=max(lo, count), len_hi=max(lo, count) + rng.randint(0, 64),
                    count_lo=rng.randint(1, count), count_hi=count, heads=heads, dim=dim,
                    codes=rng.choice(["e4m3", "int8"]), dtype=rng.choice(["fp32", "fp16", "bf16"]))
    if kind == "plan":
        sessions, width = _log_int(rng, 1, 2048), _log_int(rng, 4, 2048)
        count = max(1, min(width * 8, rng.choice([1, _log_int(rng, 1, 16384)]), 8_000_000 // sessions))
        lo = rng.randint(0, width * 4)
        return dict(kind=kind, sessions=sessions, len_lo=lo, len_hi=lo + rng.randint(0, width * 4), count_lo=rng.choice([0, count]),
                    count_hi=count, width=width, spare=rng.choice([1.0, 1.2, 0.6]))
    return dict(kind=kind, sessions=_log_int(rng, 1, 64), vocab=rng.choice([32000, 32001, 50257, 128256, 151936, 151936]),
                dtype=rng.choice(["fp32", "fp16", "bf16"]), history=_log_int(rng, 1, 8192), prompt=rng.choice([0.0, 0.3, 0.9]),
                bias=rng.choice([0, 1, 40, 300]), mask=rng.choice([False, True]))


def _lengths(case, seed):
    """Each session's held tokens (the new ones among them for attend and write) and new tokens.
    The case fixes the lengths, the seed their order."""
    own_seed = zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode())
    g = torch.Generator().manual_seed(own_seed)
    S = case["sessions"]
    lens = torch.randint(case["len_lo"], case["len_hi"] + 1, (S,), generator=g)
    counts = torch.randint(case["count_lo"], case["count_hi"] + 1, (S,), generator=g)
    if case["kind"] != "plan":
        counts = torch.minimum(counts, lens)
    order = torch.randperm(S, generator=torch.Generator().manual_seed(seed * 7919 + 13))
    return lens[order], counts[order]


# ---- inputs ---------------------------------------------------------------------
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _page_table(lens, gen, dev, spare_pages=7):
    """Shuffled pages for sessions of these lengths, as after some churn: [S, width] (-1 past the end), page count."""
    need = (lens + PAGE - 1) // PAGE
    width, total = int(need.max()) + 1, int(need.sum())
    n_pages = total + spare_pages
    perm = torch.randperm(n_pages, generator=gen, device=dev)[:total].to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    cols = torch.arange(width, device=dev)[None, :]
    table[cols < need.to(dev)[:, None]] = perm
    return table, n_pages


def _cache(planes, n_pages, dim, codes, gen, dev):
    """[planes, tokens, dim] codes of normal values with channels of unequal size, and scales [planes, n_pages]."""
    out_c = torch.empty(planes, n_pages * PAGE, dim, dtype=CODES[codes], device=dev)
    out_s = torch.empty(planes, n_pages, dtype=torch.float32, device=dev)
    chan = torch.exp(0.5 * torch.randn(planes, 1, dim, generator=gen, device=dev))
    step = max(1, 50_000_000 // (planes * PAGE * dim))
    for p0 in range(0, n_pages, step):
        n = min(step, n_pages - p0)
        x = torch.randn(planes, n * PAGE, dim, generator=gen, device=dev) * chan
        x = x.view(planes, n, PAGE, dim)
        e = _exponent(x.abs().amax(dim=(-1, -2)), codes)
        scale = torch.exp2(e.float())
        out_c[:, p0 * PAGE:(p0 + n) * PAGE] = _encode(x / scale[..., None, None], codes).view(planes, n * PAGE, dim)
        out_s[:, p0:p0 + n] = scale
    return out_c, out_s


def _stale_tails(cache, table, lens, gen):
    """Bytes of earlier owners behind each session's last token, NaN codes among them."""
    dev, S = cache.device, len(lens)
    raw = cache.view(torch.uint8)
    last = (lens - 1).clamp(min=0).to(dev)
    page = table[torch.arange(S, device=dev), last // PAGE].long()
    off = torch.arange(PAGE, device=dev)
    slot = (page[:, None] * PAGE + off)[off[None, :] > (last % PAGE)[:, None]]
    raw[:, slot] = torch.randint(0, 256, (raw.shape[0], slot.numel(), raw.shape[2]), generator=gen, device=dev).to(torch.uint8)


def _attend_state(case, seed, gen, dev):
    lens, counts = _lengths(case, seed)
    table, n_pages = _page_table(lens, gen, dev)
    H, D = case["heads"], case["dim"]
    k, ks = _cache(H, n_pages, D, case["codes"], gen, dev)
    v, vs = _cache(H, n_pages, D, case["codes"], gen, dev)
    for c in (k, v):
        _stale_tails(c, table, lens, gen)
    N = int(counts.sum())
    q = (1.5 * torch.randn(N, H * case["group"], D, generator=gen, device=dev)).to(DTYPE[case["dtype"]])
    q_start = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32).to(dev)
    return dict(q=q, k=k, v=v, k_scale=ks, v_scale=vs, table=table, lens=lens.to(torch.int32).to(dev), q_start=q_start,
                max_count=int(counts.max()))


def _write_state(case, seed, gen, dev):
    lens, counts = _lengths(case, seed)
    table, n_pages = _page_table(lens, gen, dev)
    L, H, D = case["layers"], case["heads"], case["dim"]
    k, ks = _cache(L * H, n_pages, D, case["codes"], gen, dev)
    v, vs = _cache(L * H, n_pages, D, case["codes"], gen, dev)
    k, v = k.view(L, H, -1, D), v.view(L, H, -1, D)
    ks, vs = ks.view(L, H, -1), vs.view(L, H, -1)
    N = int(counts.sum())
    row = torch.repeat_interleave(torch.arange(len(lens)), counts)
    start = counts.cumsum(0) - counts
    pos = (lens - counts)[row] + torch.arange(N) - start[row]
    # what is read back: every token of the pages that the write touches
    first = (lens - counts) // PAGE * PAGE
    n_read = lens - first
    row_r = torch.repeat_interleave(torch.arange(len(lens)), n_read)
    pos_r = first[row_r] + torch.arange(int(n_read.sum())) - (n_read.cumsum(0) - n_read)[row_r]

    def slots(r, p):
        r, p = r.to(dev), p.to(dev)
        return (table[r, p // PAGE] * PAGE + p % PAGE).to(torch.int32)

    dt = DTYPE[case["dtype"]]
    new = [(1.2 * torch.randn(L, N, H, D, generator=gen, device=dev)).to(dt) for _ in range(2)]
    return dict(new_k=new[0], new_v=new[1], k=k, v=v, k_scale=ks, v_scale=vs, slots=slots(row, pos),
                read=slots(row_r, pos_r), out_dtype=torch.bfloat16 if case["dtype"] == "bf16" else torch.float16)


def _plan_state(case, seed, gen, dev):
    lens, counts = _lengths(case, seed)
    S, W = case["sessions"], case["width"]
    held = (lens + PAGE - 1) // PAGE
    need = (lens + counts + PAGE - 1) // PAGE - held
    n_free = max(1, int(case["spare"] * int(need.sum())))
    perm = torch.randperm(int(held.sum()) + n_free, generator=gen, device=dev).to(torch.int32)
    table = torch.full((S, W), -1, dtype=torch.int32, device=dev)
    table[torch.arange(W, device=dev)[None, :] < held.to(dev)[:, None]] = perm[n_free:]
    return dict(lens=lens.to(torch.int32).to(dev), counts=counts.to(torch.int32).to(dev), table=table,
                free_pages=perm[:n_free].contiguous(), free_count=torch.tensor([n_free], dtype=torch.int32, device=dev),
                total=int(counts.sum()))


def _logits_state(case, seed, gen, dev):
    S, V, T = case["sessions"], case["vocab"], case["history"]
    cpu = torch.Generator().manual_seed(seed * 104729 + 7)
    lens = torch.randint((T + 1) // 2, T + 1, (S,), generator=cpu)
    st = dict(logits=(3.0 * torch.randn(S, V, generator=gen, device=dev)).to(DTYPE[case["dtype"]]))
    # text repeats itself: tokens of a heavy-tailed distribution over the vocabulary
    u = torch.rand(S, T, generator=gen, device=dev)
    st["tokens"] = (torch.pow(float(V), u) - 1).long().clamp(0, V - 1).mul(7919).remainder(V).to(torch.int32)
    st["token_lens"] = lens.to(torch.int32).to(dev)
    st["prompt_lens"] = (lens * case["prompt"]).to(torch.int32).to(dev)
    st["repetition"] = 1.0 + 0.5 * torch.rand(S, generator=gen, device=dev)
    st["presence"] = 0.6 * torch.rand(S, generator=gen, device=dev) if case["prompt"] else None
    st["frequency"] = 0.3 * torch.rand(S, generator=gen, device=dev) if case["prompt"] else None
    st["bias_ids"] = st["bias_values"] = st["mask"] = None
    if case["bias"]:
        ids = torch.randint(0, V, (S, case["bias"]), generator=gen, device=dev)
        st["bias_ids"] = ids.to(torch.int32)
        st["bias_values"] = 2.0 * torch.randn(S, case["bias"], generator=gen, device=dev)
    if case["mask"]:
        words = (V + 31) // 32
        bits = torch.randint(-2 ** 31, 2 ** 31, (S, words), generator=gen, device=dev)
        st["mask"] = bits.to(torch.int32)
    return st


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    make = dict(attend=_attend_state, write=_write_state, plan=_plan_state, logits=_logits_state)[case["kind"]]
    return dict(make(case, seed, gen, dev), kind=case["kind"])


# ---- the operators' plain forms -------------------------------------------------
def _exponent(amax, codes):
    """The smallest e with amax <= QMAX * 2^e, from the 32-bit value's own exponent."""
    top = {"e4m3": 0.875, "int8": 127 / 128}[codes]
    bits = {"e4m3": 9, "int8": 7}[codes]
    m, x = torch.frexp(amax.float())
    e = x.to(torch.int32) - bits + (m > top).to(torch.int32)
    e = torch.where(amax > 0, e, torch.full_like(e, E_MIN))
    return e.clamp(E_MIN, E_MAX)


def _encode(x, codes):
    if codes == "int8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _codes_of(t):
    return "int8" if t.dtype == torch.int8 else "e4m3"


def _plain_attend(s):
    q, table, lens, q_start = s["q"], s["table"], s["lens"].long(), s["q_start"].long()
    dev = q.device
    H, D = s["k"].shape[0], s["k"].shape[2]
    S, G = table.shape[0], q.shape[1] // H
    L, C = int(table.shape[1]) * PAGE, s["max_count"]
    page = table.clamp(min=0).long()
    slot = (page[:, :, None] * PAGE + torch.arange(PAGE, device=dev)).view(S, L)
    valid = torch.arange(L, device=dev)[None, :] < lens[:, None]

    def values(c, scale):
        x = c[:, slot].float() * scale[:, page].repeat_interleave(PAGE, dim=2)[..., None]
        return torch.where(valid[None, :, :, None], x, 0.0)  # [H, S, L, D]

    count = q_start[1:] - q_start[:-1]
    i = torch.arange(C, device=dev)
    here = i[None, :] < count[:, None]
    at = (q_start[:-1, None] + i)[here]
    rows = torch.zeros(S, C, H * G, D, dtype=torch.float32, device=dev)
    rows[here] = q[at].float()
    rows = rows.view(S, C, H, G, D).permute(2, 0, 3, 1, 4).reshape(H, S, G * C, D)
    x = torch.matmul(rows, values(s["k"], s["k_scale"]).transpose(-1, -2)).view(H, S, G, C, L)
    x *= D ** -0.5
    seen = torch.arange(L, device=dev) <= (lens[:, None] - count[:, None] + i)[..., None]  # [S, C, L]
    x.masked_fill_(~seen[None, :, None], float("-inf"))
    top = x.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    x = x.sub_(top).exp_()
    total = x.sum(dim=-1, keepdim=True)
    o = torch.matmul(x.view(H, S, G * C, L), values(s["v"], s["v_scale"])).view(H, S, G, C, D)
    o = torch.where(total > 0, o / total, 0.0)
    lse = (top + torch.log(total))[..., 0]
    out = torch.empty_like(q)
    out[at] = o.permute(1, 3, 0, 2, 4).reshape(S, C, H * G, D)[here].to(q.dtype)
    lse_out = torch.empty(q.shape[0], H * G, dtype=torch.float32, device=dev)
    lse_out[at] = lse.permute(1, 3, 0, 2).reshape(S, C, H * G)[here]
    return out, lse_out


def _plain_write_one(x, cache, scale, slots, codes):
    """x [L, N, H, D] into cache [L, H, tokens, D] at `slots`, the tokens of a page next to each other."""
    L, N, H, D = x.shape
    page, off = (slots // PAGE).long(), (slots % PAGE).long()
    first = torch.ones(N, dtype=torch.bool, device=x.device)
    first[1:] = page[1:] != page[:-1]
    run_of = first.long().cumsum(0) - 1
    pages = page[first]
    R = pages.numel()
    x = x.float()
    amax = torch.zeros(L, R, H, device=x.device)
    amax.scatter_reduce_(1, run_of[None, :, None].expand(L, N, H), x.abs().amax(dim=-1), "amax")
    e = _exponent(amax, codes).permute(0, 2, 1)  # [L, H, R]
    old = torch.frexp(scale[:, :, pages])[1].to(torch.int32) - 1
    fresh = torch.zeros(R, dtype=torch.bool, device=x.device).index_put_((run_of[off == 0],), torch.tensor(True, device=x.device))
    e = torch.where(fresh, e, torch.maximum(e, old))
    shift = torch.where(fresh, torch.zeros_like(e), old - e)
    held = cache.view(L, H, -1, PAGE, D)
    kept = held[:, :, pages].float() * torch.exp2(shift.float())[..., None, None]
    held[:, :, pages] = _encode(kept, codes)
    scale[:, :, pages] = torch.exp2(e.float())
    unit = torch.exp2(-e.float())[:, :, run_of]  # [L, H, N]
    cache[:, :, slots.long()] = _encode(x.permute(0, 2, 1, 3) * unit[..., None], codes)


def _plain_write(s):
    codes = _codes_of(s["k"])
    got = []
    for x, c, sc in ((s["new_k"], s["k"], s["k_scale"]), (s["new_v"], s["v"], s["v_scale"])):
        _plain_write_one(x, c, sc, s["slots"], codes)
        at = s["read"].long()
        got.append((c[:, :, at].float() * sc[:, :, at // PAGE][..., None]).to(s["out_dtype"]))
    return got


def _plain_plan(s):
    lens, counts, table = s["lens"].long(), s["counts"].long(), s["table"]
    dev, (S, W), n_free = lens.device, table.shape, s["free_pages"].numel()
    q_start = torch.zeros(S + 1, dtype=torch.int64, device=dev)
    q_start[1:] = counts.cumsum(0)
    after = lens + counts
    held = (lens + PAGE - 1) // PAGE
    fits = (after <= W * PAGE) & (q_start[1:] <= s["total"])
    need = torch.where(fits, (after + PAGE - 1) // PAGE - held, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= s["free_count"].long()))
    rank = upto - need
    new = torch.where(granted, need, 0)
    table = table.clone()
    col = torch.arange(W, device=dev)[None, :] - held[:, None]
    take = (col >= 0) & (col < new[:, None])
    top = s["free_count"].long()
    table[take] = s["free_pages"][(top - 1 - (rank[:, None] + col)[take])]
    token = torch.arange(s["total"], device=dev)
    row = torch.searchsorted(q_start[1:], token, right=True).clamp(max=S - 1)
    pos = lens[row] + token - q_start[row]
    ok = granted[row]
    slot = table[row, (pos // PAGE).clamp(max=W - 1)] * PAGE + (pos % PAGE).to(torch.int32)
    return dict(q_start=q_start.to(torch.int32), slots=torch.where(ok, slot, -1).to(torch.int32),
                positions=torch.where(ok, pos, -1), lens=torch.where(granted, after, lens).to(torch.int32),
                free_count=(top - new.sum()).to(torch.int32), table=table)


def _plain_logits(s):
    x = s["logits"].float()
    S, V = x.shape
    dev = x.device
    tokens, T = s["tokens"].long(), s["tokens"].shape[1]
    at = torch.arange(T, device=dev)[None, :]
    held = at < s["token_lens"][:, None]
    said = held & (at >= s["prompt_lens"][:, None])
    count = torch.zeros(S, V, dtype=torch.float32, device=dev)
    seen = torch.zeros(S, V, dtype=torch.float32, device=dev).scatter_add_(1, tokens, held.float()) > 0
    count.scatter_add_(1, tokens, said.float())
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    if s["presence"] is not None:
        x = x - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if s["bias_ids"] is not None:
        # an id that is given twice takes its last value
        ids, B = s["bias_ids"].long(), s["bias_ids"].shape[1]
        last = torch.full((S, V), -1, dtype=torch.int64, device=dev)
        last.scatter_reduce_(1, ids, torch.arange(B, device=dev).expand(S, B), "amax")
        x = torch.where(last >= 0, x + s["bias_values"].gather(1, last.clamp(min=0)), x)
    if s["mask"] is not None:
        bit = (s["mask"][:, :, None] >> torch.arange(32, device=dev, dtype=torch.int32)) & 1
        x = x.masked_fill(bit.view(S, -1)[:, :V] == 0, float("-inf"))
    return x


# ---- the framework's calls ------------------------------------------------------
def _own_attend(s):
    from infercache_b200.paged_ops import paged_attention
    return paged_attention(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["lens"], s["q_start"],
                           max_count=s["max_count"], return_lse=True)


def _own_write(s):
    from infercache_b200.paged_ops import page_read, page_write
    page_write(s["new_k"], s["new_v"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["slots"])
    return page_read(s["k"], s["v"], s["k_scale"], s["v_scale"], s["read"], dtype=s["out_dtype"])


def _own_plan(s):
    from infercache_b200.paged_ops import page_plan
    p = page_plan(s["lens"], s["counts"], s["table"], s["free_pages"], s["free_count"], s["total"])
    return dict(q_start=p.q_start, slots=p.slots, positions=p.positions, lens=p.lens, free_count=p.free_count,
                table=s["table"])


def _own_logits(s):
    from infercache_b200.logits import process_logits
    return process_logits(s["logits"], tokens=s["tokens"], token_lens=s["token_lens"], prompt_lens=s["prompt_lens"],
                          repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                          bias_ids=s["bias_ids"], bias_values=s["bias_values"], mask=s["mask"])


def run(state):
    if own:
        ops = dict(attend=_own_attend, write=_own_write, plan=_own_plan, logits=_own_logits)
    else:
        ops = dict(attend=_plain_attend, write=_plain_write, plan=_plain_plan, logits=_plain_logits)
    return ops[state["kind"]](state)


# ---- what a pass cannot do without ----------------------------------------------
def work(case):
    mid = lambda lo, hi: (case[lo] + case[hi]) / 2  # noqa: E731
    S = case["sessions"]
    if case["kind"] == "attend":
        H, G, D = case["heads"], case["group"], case["dim"]
        length, count = mid("len_lo", "len_hi"), mid("count_lo", "count_hi")
        cache = S * H * (length * 2 * D + length / PAGE * 8) + S * length / PAGE * 4
        rows = S * count * H * G
        return dict(bytes=int(cache + rows * (4 * D + 4)), flops=int(4 * D * rows * (length - (count - 1) / 2)))
    if case["kind"] == "write":
        size = 4 if case["dtype"] == "fp32" else 2
        new = S * mid("count_lo", "count_hi") * case["layers"] * case["heads"] * case["dim"] * 2
        return dict(bytes=int(new * (size + 1) + new * (1 + 2)), flops=int(4 * new))
    if case["kind"] == "plan":
        tokens = S * mid("count_lo", "count_hi")
        return dict(bytes=int(tokens * 12 + tokens / PAGE * 8 + S * 20), flops=int(8 * tokens))
    size = 4 if case["dtype"] == "fp32" else 2
    V = case["vocab"]
    return dict(bytes=int(S * (V * (size + 4) + case["history"] * 3 + case["bias"] * 8 + (V // 8 if case["mask"] else 0))),
                flops=int(4 * S * V))


# ---- the definitions in 64 bits --------------------------------------------------
def _exact_attend(s):
    q, k, v, table = s["q"], s["k"], s["v"], s["table"].tolist()
    lens, q_start = s["lens"].tolist(), s["q_start"].tolist()
    H, D, G = k.shape[0], k.shape[2], q.shape[1] // k.shape[0]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for r, n in enumerate(lens):
        a, b = q_start[r], q_start[r + 1]
        if a == b:
            continue
        pages = torch.tensor(table[r][:(n + PAGE - 1) // PAGE], device=q.device)
        at = (pages[:, None] * PAGE + torch.arange(PAGE, device=q.device)).reshape(-1)[:n]
        mask = torch.arange(n, device=q.device)[None, :] > torch.arange(n - (b - a), n, device=q.device)[:, None]
        for h in range(H):
            kk = k[h, at].double() * s["k_scale"][h, at // PAGE].double()[:, None]
            vv = v[h, at].double() * s["v_scale"][h, at // PAGE].double()[:, None]
            for g in range(G):
                x = q[a:b, h * G + g].double() @ kk.T / math.sqrt(D)
                x = x.masked_fill(mask, -math.inf)
                lse[a:b, h * G + g] = torch.logsumexp(x, dim=1)
                out[a:b, h * G + g] = torch.softmax(x, dim=1) @ vv
    return out, lse


def _two_to(e):
    return torch.exp2(e.float()).double()  # whole exponents: exact in 32 bits


def _exact_round(x, codes):
    """x to the nearest representable value, ties to the even one."""
    if codes == "int8":
        return torch.round(x).clamp(-127, 127)
    mag = x.abs().clamp(max=448)
    step = _two_to(torch.frexp(mag.clamp(min=2.0 ** -6))[1] - 4)
    return torch.sign(x) * torch.round(mag / step) * step


def _exact_write_one(x, cache, scale, slots, read, codes):
    """The pages' values after the write, from the values that stood there and the new ones."""
    top = QMAX[codes]
    where = slots.long()
    vals = cache.double() * scale.double().repeat_interleave(PAGE, dim=2)[..., None]
    x = x.double().permute(0, 2, 1, 3)
    touched = torch.unique(where // PAGE)
    is_new = torch.zeros(cache.shape[2], dtype=torch.bool, device=x.device)
    is_new[where] = True
    pick = (touched[:, None] * PAGE + torch.arange(PAGE, device=x.device)).reshape(-1)
    vals[:, :, where] = x
    L, H, D = vals.shape[0], vals.shape[1], vals.shape[3]
    page = vals[:, :, pick].view(L, H, -1, PAGE, D)
    new = is_new[pick].view(1, 1, -1, PAGE, 1)
    amax = torch.where(new, page, torch.zeros_like(page)).abs().amax(dim=(-1, -2))
    part, need = torch.frexp((amax / top).clamp(min=2.0 ** E_MIN))
    need = _two_to((need - (part == 0.5).int()).clamp(E_MIN, E_MAX))
    starts = is_new[touched * PAGE]
    unit = torch.where(starts, need, torch.maximum(need, scale[:, :, touched].double()))[..., None, None]
    vals[:, :, pick] = (_exact_round(page / unit, codes) * unit).reshape(L, H, -1, D)
    return vals[:, :, read.long()]


def _exact_write(s):
    if s["new_k"].numel() * 8 * 6 > 40e9:
        return None
    codes = _codes_of(s["k"])
    return [_exact_write_one(s["new_" + n], s[n], s[n + "_scale"], s["slots"], s["read"], codes) for n in ("k", "v")]


def _exact_logits(s):
    rows = []
    for r in range(s["logits"].shape[0]):
        x = s["logits"][r].double().clone()
        n, p = int(s["token_lens"][r]), int(s["prompt_lens"][r])
        said = torch.bincount(s["tokens"][r, p:n].long(), minlength=x.numel()).double()
        seen = torch.unique(s["tokens"][r, :n].long())
        rep = float(s["repetition"][r])
        x[seen] = torch.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
        if s["presence"] is not None:
            x = x - float(s["frequency"][r]) * said - float(s["presence"][r]) * (said > 0).double()
        if s["bias_ids"] is not None:
            given = dict(zip(s["bias_ids"][r].tolist(), s["bias_values"][r].double().tolist()))
            x[torch.tensor(list(given), device=x.device)] += torch.tensor(list(given.values()), dtype=torch.float64, device=x.device)
        if s["mask"] is not None:
            words = s["mask"][r].long().remainder(2 ** 32)
            v = torch.arange(x.numel(), device=x.device)
            x[torch.bitwise_right_shift(words[v // 32], v % 32) % 2 == 0] = -math.inf
        rows.append(x)
    return torch.stack(rows)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "plan":  # whole numbers: nothing is rounded
        return None
    return dict(attend=_exact_attend, write=_exact_write, logits=_exact_logits)[case["kind"]](s)
