"""Edges of the paged serving tick on a B200: factors that vanish, indices wider
than 32 bits, and the paths that only long rows reach.  References and bounds
are those of paged_reference.py and test_paged_serving_gpu.py."""
import math

import numpy as np
import pytest
import torch

import paged_reference as ref
from test_paged_serving_gpu import CODES, attention_inputs, check_attention, check_plan, empty_cache, gen, held, i32

pytestmark = pytest.mark.gpu
BIG = 2 ** 32
I64 = torch.iinfo(torch.int64)


def i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


# ---- factors that vanish -----------------------------------------------------------
LENS, COUNTS = [300, 200, 40], [300, 150, 3]  # 453 x 16 heads: the tile kernel's, for 64, 128 and 256 dims


def prompt_inputs(codes, dtype, D, seed=7):
    x = attention_inputs(seed, LENS, COUNTS, 2, 8, D, codes, dtype)
    assert x[0].shape[0] * x[0].shape[1] > 6144
    return x


def check_both(x, **kw):
    """Through the tile kernel, and with few tokens announced through the streaming kernel."""
    for max_count in (None, 1):
        assert check_attention(x, max_count=max_count, **kw)[2] == 0


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_zero_queries_over_zero_keys(codes, dtype, D):
    """A warm-up's or a zeroed head's inputs: the first session's K and queries are
    zero, and some queries of the others; right is the mean of the V rows seen."""
    from infercache_b200.paged_ops import page_write
    x = prompt_inputs(codes, dtype, D)
    q, k, v, ks, vs, table = x[:6]
    pages = table[0, :-(-LENS[0] // 16)].long()
    slots = (pages[:, None] * 16 + torch.arange(16, device="cuda")).reshape(-1)[:LENS[0]]
    keep = v.clone(), vs.clone()
    zeros = torch.zeros(LENS[0], 2, D, device="cuda", dtype=dtype)
    page_write(zeros, zeros, k, v, ks, vs, slots)
    assert bool((ks[:, pages] == 2.0 ** -60).all())
    v.view(torch.uint8).copy_(keep[0].view(torch.uint8))
    vs.copy_(keep[1])
    q[:LENS[0]] = 0
    q[310:330, 3:7] = 0
    check_both(x)
    check_both(x, scale=1e-30)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scales_that_leave_no_score(codes, dtype, D):
    x = prompt_inputs(codes, dtype, D)
    check_both(x, scale=0.0)
    check_both(((x[0] * 1e-30).to(dtype),) + x[1:], scale=1e-30)
    tiny = x[3] * 2.0 ** -50
    check_both(((x[0] * 1e-30).to(dtype), x[1], x[2], tiny) + x[4:], scale=-1e-20)


# ---- indices wider than 32 bits ------------------------------------------------------
OUTSIDE = [BIG, BIG + 5, -BIG + 5, I64.min, I64.max, I64.min + 3, 2 ** 31, -2 ** 31 - 1]


@pytest.mark.parametrize("codes", CODES)
def test_slots_beyond_32_bits_are_outside_the_pool(codes):
    from infercache_b200.paged_ops import page_read, page_write
    cache = [t[0] for t in empty_cache(1, 2, 3, 64, codes)]
    x = torch.randn(1 + len(OUTSIDE), 2, 64, generator=gen(2), device="cuda").half()
    before = [t.clone() for t in cache]
    page_write(x[1:], x[1:], *cache, i64(OUTSIDE))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))
    page_write(x, x, *cache, i64([16] + OUTSIDE))
    want = [t.clone() for t in before]
    page_write(x[:1], x[:1], *want, i32([16]))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, want))
    k, v = page_read(*cache, i64([16] + OUTSIDE))
    assert bool(k[:, 0].any()) and bool(v[:, 0].any()) and not k[:, 1:].any() and not v[:, 1:].any()


def test_ids_beyond_32_bits_are_outside_the_vocabulary():
    from infercache_b200.logits import process_logits
    x = torch.randn(1, 200, generator=gen(3), device="cuda")
    outside, vals = i64([OUTSIDE]), torch.ones(1, len(OUTSIDE), device="cuda")
    got = process_logits(x, tokens=outside, repetition=3.0, presence=1.0, frequency=0.5, bias_ids=outside, bias_values=vals)
    assert torch.equal(got, x)
    # and lengths beyond them are all of the row
    tok, ids = i64([[1, 2, 3, 4]]), i64([[7, 8]])
    whole = dict(tokens=tok, repetition=3.0, frequency=1.0, bias_ids=ids, bias_values=vals[:, :2])
    assert torch.equal(process_logits(x, **whole, token_lens=i64([BIG]), bias_lens=i64([BIG])), process_logits(x, **whole))
    assert torch.equal(process_logits(x, **whole, prompt_lens=i64([BIG])), process_logits(x, **whole, prompt_lens=i64([4])))
    assert torch.equal(process_logits(x, **whole, token_lens=i64([-BIG + 2])), process_logits(x, bias_ids=ids, bias_values=vals[:, :2]))


def test_batch_counts_and_keeps_beyond_32_bits():
    from infercache_b200 import PagedBatch
    from test_paged_serving_gpu import make_pool
    b = PagedBatch(make_pool(torch.int8), 4)
    b.extend([20, 5, 1, 0])
    b.release(i64([BIG, I64.max, I64.min, BIG + 1]))  # more than they hold, or negative: all of them
    assert b.lens.tolist() == [20, 5, 1, 0]
    b.extend(i64([BIG + 1, 0, -BIG + 1, 1]), total=2)  # two that cannot be had, one of them negative
    assert b.lens.tolist()[:3] == [20, 5, 1]
    with pytest.raises(RuntimeError):
        b.check_device_status()


# ---- pages whose tokens leave slots out ------------------------------------------------
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("pages,H", [(60, 2), (500, 4), (1400, 8)])
def test_write_leaves_slots_out(codes, pages, H):
    """A page's tokens in order but not in consecutive slots are one warp's, run
    after run: the scale covers them all.  Sizes at which a warp looks after 1, 4
    and 16 tokens."""
    from infercache_b200.paged_ops import page_write
    rng = np.random.default_rng(pages)
    slots = []
    for page in rng.permutation(pages + 20)[:pages].tolist():
        slots += [page * 16 + j for j in range(16) if rng.random() < 0.45]
    n = len(slots) * H
    assert n <= 8192 if pages == 60 else 8192 < n <= 65536 if pages == 500 else n > 65536
    cache = [t[0] for t in empty_cache(1, H, pages + 20, 64, codes, 1)]
    planes = [(c, s, np.nan_to_num(held(c, s)), s.cpu().double().numpy().copy()) for c, s in zip(cache[:2], cache[2:])]
    g, known = gen(2), set()
    for piece, scale in ((slots, 1.0), ([5, 7, 9, 15], 6.0), ([48, 50], 0.5), ([20, 22, 23, 31], 40.0)):
        new = [(torch.randn(len(piece), H, 64, generator=g, device="cuda") * scale).bfloat16() for _ in range(2)]
        page_write(*new, *cache, i32(piece))
        anew = {x // 16 for x in piece if x % 16 == 0}  # what stood in these pages is gone
        known = {x for x in known if x // 16 not in anew} | set(piece)
        at, held_pages = sorted(known), sorted({x // 16 for x in known})
        for x, (c, s, want, wscale) in zip(new, planes):
            rows = x.double().cpu().numpy()
            for h in range(H):
                ref.write(want[h], wscale[h], rows[:, h], piece, codes)
            assert np.array_equal(held(c, s)[:, at], want[:, at])
            assert np.array_equal(s.cpu().double().numpy()[:, held_pages], wscale[:, held_pages])


# ---- one long prompt in one call -----------------------------------------------------
def test_long_prompt_with_a_wide_table():
    """65.3k tokens x 8 KV heads of 4 under a table for 128k tokens: the tile
    kernel's, whose work the table's width does not bound."""
    from infercache_b200.paged_ops import paged_attention
    n, H, G, D, width = 65_300, 8, 4, 64, 8192
    x = list(attention_inputs(5, [n], [n], H, G, D, torch.int8, torch.float16))
    wide = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    wide[:, :x[5].shape[1]] = x[5]
    x[5] = wide
    out, lse = paged_attention(*x, return_lse=True)
    at = [0, 1, 15, 16, 127, 128, 129, 5000, 33_333, 65_298, 65_299]
    q, k, v, ks, vs = x[:5]
    # a query's row is that of a session that ends with it
    want, wlse, tol, ltol = ref.attention(q[at], ref.cache_values(k, ks), ref.cache_values(v, vs), wide.expand(len(at), width),
                                          [i + 1 for i in at], list(range(len(at) + 1)), D ** -0.5)
    assert float(((out[at].double() - want).abs() - tol).max()) <= 0
    assert float(((lse[at].double() - wlse).abs() - ltol).max()) <= 0


# ---- page ids no pool has --------------------------------------------------------------
@pytest.mark.parametrize("S,count", [(3, 40), (40, 2000)])
def test_plan_gives_no_slot_for_page_ids_past_32_bit_rows(S, count):
    """Ids from 2^27 on, whose rows would not fit 32 bits, are no pool's: slot -1, as
    for negative ones, through the one-kernel plan and the two-kernel one."""
    from infercache_b200.paged_ops import page_plan
    need = -(-count // 16)
    ids = list(range(S * need))
    for i, bad in ((1, 2 ** 27), (4, 2 ** 31 - 1), (7, -5), (2 * need + 1, 2 ** 28 + 3)):
        ids[i] = bad
    ids[0] = 2 ** 27 - 1  # the last that fits
    table = i32([[-1] * need] * S)
    p = page_plan(i32([0] * S), i32([count] * S), table, i32(ids), i32([len(ids)]), S * count, max_count=count)
    want = []
    for s in range(S):
        for t in range(count):
            page = ids[len(ids) - 1 - s * need - t // 16]
            want.append(page * 16 + t % 16 if 0 <= page < 2 ** 27 else -1)
    assert p.slots.tolist() == want


# ---- logits rows longer than the kernel's first reach ----------------------------------
def check_long_logits(V, S, T, B, dtype, spread, seed, in_place):
    from infercache_b200.logits import process_logits
    rng = np.random.default_rng(seed)
    x = torch.randn(S, V, generator=gen(seed), device="cuda").mul(3).to(dtype)
    kw, lens, prompt, bias = {}, [0] * S, [0] * S, [{}] * S
    tokens = np.zeros((S, max(T, 1)), np.int64)
    rep, pres, freq = [1.3, 0.7][:S], [0.5, -0.25][:S], [0.001, 0.003][:S]
    if T:
        tokens = rng.integers(0, spread, (S, T))
        tokens[:, ::11] = rng.integers(-3, V + 3, tokens[:, ::11].shape)
        lens, prompt = [T, T - 7][:S], [T // 3, 5][:S]
        kw.update(tokens=torch.from_numpy(tokens).cuda().int(), token_lens=i32(lens), prompt_lens=i32(prompt),
                  repetition=torch.tensor(rep, device="cuda"), presence=torch.tensor(pres, device="cuda"),
                  frequency=torch.tensor(freq, device="cuda"))
    if B:
        ids, vals = rng.integers(-3, V + 3, (S, B)), rng.normal(size=(S, B)).astype(np.float32)
        ids[:, B // 2:B // 2 + 20] = ids[:, :20]  # given twice: the last value counts
        blens = [B, B - 3][:S]
        bias = [dict(zip(ids[r, :blens[r]].tolist(), vals[r, :blens[r]].tolist())) for r in range(S)]
        kw.update(bias_ids=i32(ids), bias_values=torch.from_numpy(vals).cuda(), bias_lens=i32(blens))
    f32 = lambda v: [float(np.float32(a)) for a in v]  # noqa: E731
    want = ref.logits(x.cpu(), tokens, lens, prompt, f32(rep), f32(pres), f32(freq), bias, None)
    # the penalty's product (two roundings), the term of count and presence (two), a
    # difference and a sum: each at most half a step of the largest intermediate
    n = max(np.bincount(np.clip(tokens[r], 0, V)).max() for r in range(S)) if T else 0
    tol = 6 * 2.0 ** -24 * (2 * x.cpu().double().abs() + float(n) * 0.003 + 1 + 6)
    got = process_logits(x, **kw, **(dict(out=x) if in_place else {})).cpu().double()
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("V", [8192, 32001])
@pytest.mark.parametrize("T,B", [(5000, 0), (5000, 40), (2049, 3000), (0, 5000), (70000, 0), (70000, 40), (50, 33000), (0, 33000),
                                 (70000, 33000)])
def test_logits_long_rows(V, T, B, in_place):
    """Past 2048 tokens, past the list of 2048 named ids, past 65535 tokens and 32766
    biases, each with and without the other part."""
    check_long_logits(V, 2, T, B, torch.float32, V, T + B, in_place)


@pytest.mark.parametrize("T,B,spread", [(5000, 0, 6000), (5000, 300, 8192), (70000, 0, 8000), (70000, 33000, 8192)])
def test_logits_long_rows_in_one_large_chunk(T, B, spread):
    """A batch large enough for chunks of 8192 ids, most of whose first chunk is named."""
    check_long_logits(8192 * 700, 1, T, B, torch.bfloat16, spread, 3, False)


# ---- calls the documentation allows ------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("max_count", [1, None])
def test_attention_writes_over_its_queries(D, max_count):
    """out may be q: a row is read by those alone that write it, before they do;
    one long session in shares, and many rows in tiles."""
    from infercache_b200.paged_ops import paged_attention
    for lens, counts in (([20000, 90], [2, 1]), (LENS, COUNTS)):
        x = attention_inputs(D, lens, counts, 2, 8, D, CODES[0], torch.float16)
        want = paged_attention(*x, max_count=max_count)
        q = x[0].clone()
        got = paged_attention(q, *x[1:], max_count=max_count, out=q)
        assert got is q and torch.equal(q, want)


@pytest.mark.parametrize("max_count", [1, None])
def test_attention_rows_before_the_first_session(max_count):
    from infercache_b200.paged_ops import paged_attention
    x = attention_inputs(4, LENS, COUNTS, 2, 8, 128, CODES[1], torch.bfloat16)
    want, wlse = paged_attention(*x, max_count=max_count, return_lse=True)
    q = torch.cat([torch.full((5, 16, 128), math.nan, device="cuda").bfloat16(), x[0]])
    out = torch.full_like(q, 9.0)
    got, lse = paged_attention(q, *x[1:7], x[7] + 5, max_count=max_count, out=out, return_lse=True)
    assert bool((out[:5] == 9).all()) and torch.equal(out[5:], want) and torch.equal(lse[5:], wlse)


@pytest.mark.parametrize("S", [31, 32, 33, 127, 128, 129])
def test_attention_numbers_of_sessions(S):
    """Around the counts where the kernels look sessions up in another way, alone and
    with one session's prompt beside them."""
    rng = np.random.default_rng(S)
    lens = rng.integers(0, 200, S).tolist()
    counts = [min(n, int(c)) for n, c in zip(lens, rng.integers(0, 3, S))]
    lens[-1] = counts[-1] = 1
    check_attention(attention_inputs(S, lens, counts, 2, 4, 64, CODES[S % 2], torch.float16), max_count=2)
    lens[S // 2], counts[S // 2] = 900, 850
    x = attention_inputs(S, lens, counts, 2, 4, 64, CODES[S % 2], torch.float16)
    assert x[0].shape[0] * x[0].shape[1] > 6144
    check_attention(x)


# ---- roundings of the repetition penalty --------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_own_repetition_penalty_rounds_once(dtype):
    """x / r as 32 bits give it, bit for bit, where r is the row's; NaN, infinities
    and zeros as the comparison sends them."""
    from infercache_b200.logits import process_logits
    x = (torch.randn(6, 20000, generator=gen(8), device="cuda") * 5).to(dtype)
    x[:, :5] = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0], device="cuda").to(dtype)
    r = torch.tensor([1.1, 1.3, 0.9, 3.0, 1.7, 1e-3], device="cuda")
    said = torch.arange(0, 20000, device="cuda", dtype=torch.int32).expand(6, -1)
    f = x.float()
    want = torch.where(f > 0, f / r[:, None], f * r[:, None])
    assert torch.equal(process_logits(x, tokens=said, repetition=r).view(torch.int32), want.view(torch.int32))


# ---- a page filled token by token -----------------------------------------------------
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("growth", [1.0, 1.3, 2.0, 5.0])
def test_error_of_a_page_filled_token_by_token(codes, growth):
    """Each token may raise the page's scale and round the older codes once more.
    Units only grow, by a factor of two or more each time, so the halves of all
    units that a value was rounded to sum to at most the last unit: |stored - x|
    <= unit (int8); an e4m3 code that stays normal is not rounded again, and a
    subnormal one to multiples of 2^-9 of the unit: 2^-4 |x| + 2^-9 unit."""
    from infercache_b200.paged_ops import page_read, page_write
    cache = [t[0] for t in empty_cache(1, 3, 2, 64, codes)]
    x = torch.randn(2, 16, 3, 64, generator=gen(9), device="cuda") * torch.logspace(0, 15, 16, base=growth, device="cuda")[:, None, None]
    for t in range(16):
        page_write(x[0, t:t + 1], x[1, t:t + 1], *cache, i32([16 + t]))
    got = page_read(*cache, i32(list(range(16, 32))), dtype=torch.float32)
    for g, w, s in zip(got, x, cache[2:]):
        w, unit = w.transpose(0, 1).double(), s[:, 1].double()[:, None, None]
        bound = unit if codes == torch.int8 else w.abs() * 2.0 ** -4 + unit * 2.0 ** -9
        assert bool(((g.double() - w).abs() <= bound).all())


@pytest.mark.parametrize("codes", CODES)
def test_rejected_drafts_leave_the_page_its_unit(codes):
    """A dropped token that raised its page's scale has rounded the kept ones to the
    larger unit: within that unit's error, and unchanged by the release."""
    from infercache_b200 import PagedBatch
    from test_paged_serving_gpu import make_pool
    pool = make_pool(codes, L=1, value=torch.float32)
    b = PagedBatch(pool, 1)
    x = torch.randn(6, 2, 64, generator=gen(2), device="cuda")
    x[4:] *= 100
    b.extend([4])
    b.append(0, x[:4], x[:4])
    b.extend([2])
    b.append(0, x[4:], x[4:])
    page = int(b.block_table[0, 0])
    unit = pool.k_scale[0, :, page].clone()
    before = b.gather(0, 4)[0]
    b.release([4])
    assert torch.equal(pool.k_scale[0, :, page], unit) and torch.equal(b.gather(0, 4)[0], before)
    w = x[:4].transpose(0, 1).double()
    bound = unit.double()[:, None, None] * (1.0 if codes == torch.int8 else 2.0 ** -9) + (0 if codes == torch.int8 else w.abs() * 2.0 ** -4)
    assert bool(((before[0].double() - w).abs() <= bound).all())


# ---- outputs over inputs ---------------------------------------------------------------------
def test_overlaps_that_would_race_are_refused():
    from infercache_b200.logits import process_logits
    from infercache_b200.paged_ops import page_read, page_write, paged_attention
    k, v, ks, vs = [t[0] for t in empty_cache(1, 2, 3, 64, torch.int8)]
    rows, slots = torch.randn(2, 2, 64, device="cuda").half(), i32([16, 17])
    for bad in ((k, k, ks, vs), (k, v, ks, ks)):
        with pytest.raises(ValueError):
            page_write(rows, rows, *bad, slots)
    out = torch.empty(2, 2, 64, device="cuda").half()
    with pytest.raises(ValueError):
        page_read(k, v, ks, vs, slots, out=(out, out))
    x = attention_inputs(1, [40], [3], 2, 2, 64, torch.int8, torch.float16)
    buf = torch.zeros(4 * 4 * 64 + 64, device="cuda").half()
    buf[:3 * 256].copy_(x[0].reshape(-1))
    for q, o in ((buf[:768].view(3, 4, 64), buf[64:832].view(3, 4, 64)),
                 (buf[:960].as_strided((3, 4, 64), (320, 64, 1)), buf[:768].view(3, 4, 64))):
        with pytest.raises(ValueError):
            paged_attention(q, *x[1:], out=o)
    wide = torch.randn(5, 300, device="cuda")[:4]
    for a, o in ((wide[:, :100], wide[:, 50:150]), (wide[:, :100], wide[:, 250:300].as_strided((4, 100), (300, 1))),
                 (wide[:, :100], wide.view(-1)[:400].view(4, 100)), (wide[:3], wide[1:4]),
                 (wide.view(torch.float16)[:, :100], wide[:, :100])):
        with pytest.raises(ValueError):
            process_logits(a, out=o)
    tok = i32([[1, 2], [3, 4], [5, 6], [7, 99]])
    want = process_logits(wide[:, :100].clone(), tokens=tok, repetition=1.5)
    got = process_logits(wide[:, :100], tokens=tok, repetition=1.5, out=wide[:, 100:200])  # side by side
    assert torch.equal(got, want)
    got = process_logits(wide[:, 200:], tokens=tok, repetition=1.5, out=wide[:, :100])
    assert torch.equal(got, process_logits(wide[:, 200:].clone(), tokens=tok, repetition=1.5))
    got = process_logits(wide[:1, :100], out=wide[:1, 100:200])
    assert torch.equal(got, wide[:1, :100])
