"""The paged serving tick (paged_ops, logits) on a B200 against the 64-bit
reference in paged_reference.py.  Plans, page codes and scales are compared
exactly; attention within the bounds that reference derives per element;
logits within three fp32 roundings of their largest intermediate."""
import math

import numpy as np
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu
CODES = [torch.float8_e4m3fn, torch.int8]
NO_PAGES, NONFINITE, BAD_ROW = 4, 8, 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- page_plan / page_release -------------------------------------------------------
def plan_inputs(seed, S, width, max_len, max_count, free):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, max_len + 1, S).tolist()
    counts = rng.integers(0, max_count + 1, S).tolist()
    held = [-(-n // 16) for n in lens]
    ids = rng.permutation(sum(held) + free).tolist()
    table, k = [], 0
    for h in held:
        table.append(ids[k:k + h] + [-1] * (width - h))
        k += h
    return lens, counts, table, ids[k:]


def check_plan(lens, counts, table, free, total, commit=False):
    from infercache_b200.paged_ops import page_plan
    tl, tc, tt, tf, tn = i32(lens), i32(counts), i32(table), i32(free), i32([len(free)])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = page_plan(tl, tc, tt, tf, tn, total, commit=commit, status=status)
    want = ref.plan(lens, counts, table, free, len(free), total)
    assert p.q_start.tolist() == want[0]
    assert p.slots.tolist() == want[1]
    assert p.positions.tolist() == want[2]
    assert p.lens.tolist() == want[3]
    assert p.free_count.tolist() == [want[4]]
    assert tt.tolist() == want[5]
    assert int(status) == (NO_PAGES if want[6] else 0)
    assert (tl.tolist(), tn.tolist()) == ((want[3], [want[4]]) if commit else (lens, [len(free)]))
    return want


@pytest.mark.parametrize("S,width,max_len,max_count,free", [
    (1, 1, 0, 16, 1), (1, 4, 40, 1, 2), (7, 5, 40, 30, 40), (33, 8, 100, 28, 12), (1500, 6, 60, 36, 4000),
    (300, 40, 200, 400, 9000), (2, 4096, 20, 60000, 8000)])
def test_plan(S, width, max_len, max_count, free):
    lens, counts, table, fr = plan_inputs(S + free, S, width, max_len, max_count, free)
    check_plan(lens, counts, table, fr, sum(counts))
    check_plan(lens, counts, table, fr, sum(counts), commit=True)


@pytest.mark.parametrize("S,total_free", [(1000, 700), (1025, 5000), (3000, 2000), (8192, 9000)])
@pytest.mark.parametrize("top", [1, 3])
def test_plan_many_sessions_of_few_tokens(S, total_free, top):
    """Most sessions bring nothing or one token: a warp's tokens are many
    sessions', with runs of empty ones between them."""
    lens, counts, table, fr = plan_inputs(S + top, S, 4, 40, top, total_free)
    counts = [c if i % 7 else 0 for i, c in enumerate(counts)]
    counts[3:200] = [0] * 197
    counts[300] = 24 if lens[300] <= 40 else 0
    check_plan(lens, counts, table, fr, sum(counts))
    check_plan(lens, counts, table, fr, sum(counts) + 5)


def test_plan_edges():
    # exactly full table rows and pages, nothing to add, an empty total
    check_plan([16, 0, 31], [16, 32, 1], [[3, -1], [-1, -1], [1, 0]], [9, 8, 7], 49)
    check_plan([5, 0], [0, 0], [[2], [-1]], [1], 0)
    # past the table row; a negative count; past `total`; the stack runs out for the
    # third session, the fourth needs no page, the fifth does
    check_plan([30, 4], [3, 5], [[0, 1], [2, -1]], [5, 6], 8)
    check_plan([4, 4], [-1, 5], [[0, -1], [2, -1]], [5, 6], 5)
    check_plan([4, 4], [5, 5], [[0, -1], [2, -1]], [5, 6], 9)
    want = check_plan([0, 0, 0, 3, 16], [16, 16, 40, 2, 1], [[-1] * 3, [-1] * 3, [-1] * 3, [9, -1, -1], [8, -1, -1]],
                      [4, 5, 6], 75)
    assert want[6] == [2, 4]


def test_release_and_reuse():
    from infercache_b200.paged_ops import page_plan, page_release
    lens, counts, table, free = plan_inputs(5, 40, 12, 150, 0, 30)
    rng = np.random.default_rng(3)
    keep = [int(rng.choice([-1, 0, n, n + 5, max(0, n - 1), n // 2])) for n in lens]
    cap = free + [-7] * 600
    tl, tt, tf, tn = i32(lens), i32(table), i32(cap), i32([len(free)])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    page_release(tl, i32(keep), tt, tf, tn, status=status)
    wl, wt, wf = ref.release(lens, keep, table, free, len(free))
    assert tl.tolist() == wl and tt.tolist() == wt and tn.tolist() == [len(wf)] and tf[:len(wf)].tolist() == wf
    assert tf[len(wf):].tolist() == cap[len(wf):] and int(status) == 0
    # what was given back is handed out again in that order
    more = i32([16] * 40)
    got = page_plan(tl, more, tt, tf, tn, 640, commit=True)
    want = ref.plan(wl, [16] * 40, wt, wf, len(wf), 640)
    assert got.slots.tolist() == want[1]


def test_release_refuses_overflow_whole():
    from infercache_b200.paged_ops import page_release
    lens, tt, tf, tn = i32([16, 40]), i32([[0, -1, -1], [1, 2, 3]]), i32([8, -1, -1]), i32([1])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    page_release(lens, i32([0, 0]), tt, tf, tn, status=status)
    assert int(status) == BAD_ROW and lens.tolist() == [16, 40] and tn.tolist() == [1] and tf.tolist() == [8, -1, -1]
    assert tt.tolist() == [[0, -1, -1], [1, 2, 3]]


# ---- page_write / page_read ---------------------------------------------------------
def empty_cache(L, H, pages, D, dtype, seed=0, spill=True):
    """A cache with stale bytes everywhere and stale scales."""
    shape = (L, H, pages * 16, D)
    g = gen(seed)
    k, v = (torch.randint(0, 256, shape, generator=g, device="cuda").to(torch.uint8).view(dtype) for _ in range(2))
    ks, vs = (torch.exp2(torch.randint(-20, 20, (L, H, pages), generator=g, device="cuda").float()) for _ in range(2))
    return k, v, ks, vs


def held(codes, scales):
    return ref.cache_values(codes, scales).cpu().numpy()


def check_write(L, H, D, dtype, src, pieces, pages, seed=1, scale_of=lambda i: 1.0):
    """Write `pieces` (lists of slots) one after another and compare with the reference after each."""
    from infercache_b200.paged_ops import page_read, page_write
    k, v, ks, vs = empty_cache(L, H, pages, D, dtype, seed)
    want = [[np.nan_to_num(held(c, s)) for c in (t,)][0] for t, s in ((k, ks), (v, vs))]
    wscale = [ks.cpu().double().numpy().copy(), vs.cpu().double().numpy().copy()]
    g = gen(seed + 1)
    known = set()
    for i, slots in enumerate(pieces):
        new = [(torch.randn(L, len(slots), H, D, generator=g, device="cuda") * scale_of(i)).to(src) for _ in range(2)]
        page_write(new[0], new[1], k, v, ks, vs, i32(slots))
        known |= {s for s in slots if 0 <= s < pages * 16}
        for t in range(2):
            x = new[t].double().cpu().numpy()
            for l in range(L):
                for h in range(H):
                    ref.write(want[t][l, h], wscale[t][l, h], x[l, :, h], slots, dtype)
        at = sorted(known)
        for (c, s), w, ws in zip(((k, ks), (v, vs)), want, wscale):
            assert np.array_equal(held(c, s)[:, :, at], w[:, :, at])
            assert np.array_equal(s.cpu().double().numpy()[:, :, sorted({x // 16 for x in at})],
                                  ws[:, :, sorted({x // 16 for x in at})])
        for out in (torch.float32, torch.bfloat16, torch.float16):
            got = page_read(k, v, ks, vs, i32(at + [-1, pages * 16]), dtype=out)
            for t in range(2):
                w = torch.from_numpy(want[t][:, :, at]).to(out)
                assert torch.equal(got[t][:, :, :len(at)].cpu(), w)
                assert not got[t][:, :, len(at):].any()


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("src", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_write_and_read(dtype, src, D):
    # a page from its start, a prompt over three pages that ends in one, its
    # continuation, single tokens; pages out of order; rows outside the pool
    check_write(2, 3, D, dtype, src, [
        list(range(32, 48)), list(range(64, 96)) + list(range(16, 23)), list(range(23, 31)), [31, 0], [1], [2], [-1, 3, 400]],
        7, scale_of=lambda i: [1.0, 0.5, 4.0, 1.0, 8.0, 0.01, 100.0][i])


@pytest.mark.parametrize("dtype", CODES)
def test_write_token_by_token_growing(dtype):
    """Every later token larger than all before it: each write rounds the page again."""
    check_write(1, 2, 64, dtype, torch.float32, [[48 + i] for i in range(16)] + [[0], [1]], 5,
                scale_of=lambda i: 1.7 ** i)


@pytest.mark.parametrize("n_pieces", [1, 3])
def test_write_many_tokens(n_pieces):
    """Past the size where a warp looks after 16 tokens' runs, with runs of every
    length at every alignment."""
    rng = np.random.default_rng(n_pieces)
    pages = rng.permutation(3000)[:1300].tolist()
    fill = [0] * 1300
    pieces = []
    for _ in range(n_pieces):
        slots = []
        for i in rng.permutation(1300).tolist():
            n = int(rng.integers(0, 17 - fill[i]))
            slots += [pages[i] * 16 + fill[i] + j for j in range(n)]
            fill[i] += n
        pieces.append(slots)
    assert len(pieces[0]) * 4 > 16384
    check_write(1, 4, 64, torch.int8, torch.bfloat16, pieces, 3000)


def test_write_nonfinite_and_extremes():
    from infercache_b200.paged_ops import page_write
    for dtype in CODES:
        k, v, ks, vs = empty_cache(1, 1, 2, 64, dtype)
        x = torch.zeros(3, 1, 64, device="cuda")
        x[0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
        x[1, 0, 0] = 1e30     # past 2^60 steps: saturates
        x[2, 0, 0] = 1e-30    # under 2^-60 steps: zero
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        zeros = torch.zeros(1, 1, 64, device="cuda")
        page_write(zeros, zeros, k[0], v[0], ks[0], vs[0], i32([0]), status=status)
        assert int(status) == 0 and float(ks[0, 0, 0]) == 2.0 ** -60 and not held(k, ks)[0, 0, 0].any()
        page_write(x[:1], x[:1], k[0], v[0], ks[0], vs[0], i32([16]), status=status)
        e = ref.exponent(3.0, dtype)
        assert int(status) == NONFINITE
        assert held(k, ks)[0, 0, 16, :4].tolist() == [ref.QMAX[dtype] * 2.0 ** e, -ref.QMAX[dtype] * 2.0 ** e, 0.0, 3.0]
        page_write(x[1:], x[1:], k[0], v[0], ks[0], vs[0], i32([0, 1]))
        assert held(v, vs)[0, 0, 0, 0] == ref.QMAX[dtype] * 2.0 ** 60 and held(v, vs)[0, 0, 1, 0] == 0.0


def test_write_strided_and_misaligned():
    """Slices of a fused projection, a transposed layout and rows off a 16-byte
    boundary give what their contiguous copies give."""
    from infercache_b200.paged_ops import page_write
    g = gen(9)
    fused = torch.randn(40, 2 * 3 * 64 + 8, generator=g, device="cuda").half()
    base = torch.randn(3, 40, 64, generator=g, device="cuda").bfloat16()
    odd = torch.randn(40 * 3 * 64 + 1, generator=g, device="cuda").half()[1:].view(40, 3, 64)
    slots = i32(list(range(40)))
    for k, v in ((fused[:, :192].view(40, 3, 64), fused[:, 192:384].view(40, 3, 64)),
                 (base.transpose(0, 1), (2 * base).transpose(0, 1)), (odd, odd * 2),
                 (base.transpose(0, 1), (2 * base).transpose(0, 1).contiguous())):
        a, b = (empty_cache(1, 3, 4, 64, torch.int8, 4) for _ in range(2))
        page_write(k, v, *(t[0] for t in a), slots)
        page_write(k.contiguous().clone(), v.contiguous().clone(), *(t[0] for t in b), slots.long())
        for x, y in zip(a, b):
            assert torch.equal(x[:, :, :2 if x.dim() == 3 else 40].view(torch.uint8), y[:, :, :2 if y.dim() == 3 else 40].view(torch.uint8))


# ---- paged_attention ------------------------------------------------------------------
def attention_inputs(seed, lens, counts, H, G, D, codes, dtype, extra_pages=3, k_spread=2, v_spread=2):
    """Shuffled pages whose scales spread over many powers of two, stale bytes
    (NaN codes among them) behind each session's last token and in free pages."""
    g = gen(seed)
    need = [-(-n // 16) for n in lens]
    n_pages = sum(need) + extra_pages
    k, v, _, _ = empty_cache(1, H, n_pages, D, codes, seed)
    k, v = k[0], v[0]
    ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(need + [1]) + 1
    table, at, i = [], [], 0
    for n, m in zip(lens, need):
        pages = ids[i:i + m]
        i += m
        table.append(pages + [-1] * (width - m))
        at += [pages[t // 16] * 16 + t % 16 for t in range(n)]
    at = torch.tensor(at, dtype=torch.long, device="cuda")
    ks, vs = (torch.exp2(torch.randint(-s, s + 1, (H, n_pages), generator=g, device="cuda").float()) / 64
              for s in (k_spread, v_spread))
    for c in (k, v):
        if codes == torch.int8:
            c[:, at] = torch.randint(-127, 128, (H, len(at), D), generator=g, device="cuda").to(torch.int8)
        else:
            c.view(torch.uint8)[:, at] = (torch.randn(H, len(at), D, generator=g, device="cuda") * 60).clamp(-448, 448) \
                .to(codes).view(torch.uint8)
    q = (torch.randn(sum(counts), H * G, D, generator=g, device="cuda") * 0.5).to(dtype)
    q_start = [0]
    for c in counts:
        q_start.append(q_start[-1] + c)
    return q, k, v, ks, vs, i32(table), i32(lens), i32(q_start)


def check_attention(inputs, **kw):
    from infercache_b200.paged_ops import paged_attention
    q, k, v, ks, vs, table, lens, q_start = inputs
    scale = kw.get("scale", q.shape[-1] ** -0.5)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = paged_attention(*inputs, return_lse=True, status=status, **kw)
    want, wlse, tol, ltol = ref.attention(q, ref.cache_values(k, ks), ref.cache_values(v, vs), table, lens.tolist(),
                                          q_start.tolist(), scale)
    n = int(q_start[-1])
    assert out.dtype == q.dtype and not torch.isnan(out[:n]).any()
    over = ((out.double() - want).abs() - tol)[:n]
    assert float(over.max()) <= 0, (float(over.max()), over.argmax())
    none = torch.isinf(wlse[:n])
    assert torch.equal(torch.isinf(lse[:n]), none) and not out[:n][none].any()
    assert float(((lse.double() - wlse).abs() - ltol)[:n][~none].max() if (~none).any() else 0) <= 0
    return out, lse, int(status)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G,D", [(2, 8, 128), (1, 1, 64), (3, 7, 64), (2, 12, 128), (1, 16, 256), (2, 3, 256), (1, 40, 64)])
def test_attention_one_token(codes, dtype, H, G, D):
    lens = [1, 15, 16, 17, 700, 33, 0, 128, 129]
    out, _, status = check_attention(attention_inputs(H * G + D, lens, [1] * len(lens), H, G, D, codes, dtype), max_count=1)
    assert status == 0


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G,D", [(2, 4, 64), (1, 7, 128), (2, 2, 256)])
def test_attention_several_tokens(codes, dtype, H, G, D):
    """Drafts and short prompts: causal among the new tokens, sessions without
    any, queries from nothing but themselves, more tokens than are held."""
    lens, counts = [5, 40, 16, 300, 17, 64, 2, 90], [5, 3, 16, 7, 1, 0, 4, 90]
    check_attention(attention_inputs(G + D, lens, counts, H, G, D, codes, dtype))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("S,top", [(1, 20000), (2, 9000), (300, 90)])
def test_attention_shares(codes, S, top):
    """One long session over every CTA, and many short ones in one."""
    rng = np.random.default_rng(S)
    lens = [top - 3] if S == 1 else rng.integers(0, top, S).tolist()
    check_attention(attention_inputs(S, lens, [1] * S, 2, 8, 128, codes, torch.bfloat16), max_count=1)
    check_attention(attention_inputs(S, lens, [min(2, n) for n in lens], 2, 5, 64, codes, torch.float16))


@pytest.mark.parametrize("S", [1, 5, 40, 70])
@pytest.mark.parametrize("G,D", [(8, 128), (5, 64), (1, 256)])
def test_attention_whatever_the_table_holds(S, G, D):
    """Narrow tables give every group a cluster of CTAs (of 8, 4, 2), wide ones equal
    shares of all pages: the same sessions through both, and with sessions
    that have nothing to ask or to attend over."""
    rng = np.random.default_rng(S)
    lens = rng.integers(0, 1500, S).tolist()
    lens[0] = 1500
    counts = [1 if n else int(rng.integers(0, 2)) for n in lens]
    counts[-1] = 1
    x = attention_inputs(S + G, lens, counts, 2, G, D, torch.float8_e4m3fn, torch.float16)
    check_attention(x, max_count=1)
    wide = torch.full((S, 2000), -1, dtype=torch.int32, device="cuda")
    wide[:, :x[5].shape[1]] = x[5]
    check_attention(x[:5] + (wide,) + x[6:], max_count=1)
    # fewer tokens announced than some session has
    lens, counts = [n + 20 for n in lens], [c * 9 for c in counts]
    check_attention(attention_inputs(S + G + 1, lens, counts, 2, G, D, torch.int8, torch.bfloat16), max_count=1)


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("S,G,D", [(5, 1, 64), (40, 5, 128), (40, 12, 128), (24, 3, 256), (150, 16, 64), (9, 16, 256)])
def test_attention_wide_tables_share_the_line(seed, S, G, D):
    """Tables too wide for a cluster per group: shares of one line that begin and
    end anywhere, in a group's pages and in what it costs besides."""
    g = torch.Generator().manual_seed(seed)
    lens = [[0, 1, 16, 17, 300, 700, 2500, 4100][i] for i in torch.randint(0, 8, (S,), generator=g).tolist()]
    counts = [min(n, c) for n, c in zip(lens, torch.randint(0, 4 if G < 12 else 2, (S,), generator=g).tolist())]
    if not sum(counts):
        lens[0] = counts[0] = 1
    q, k, v, ks, vs, table, n, start = attention_inputs(seed, lens, counts, 2, G, D, CODES[seed % 2],
                                                        [torch.float16, torch.bfloat16][seed % 2])
    wide = torch.full((S, 900), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    out, lse, status = check_attention((q, k, v, ks, vs, wide, n, start), max_count=max(counts))
    assert status == 0


def test_flags_that_have_no_truth_are_refused():
    from infercache_b200.paged_ops import page_plan, paged_attention
    two = torch.ones(2, device="cuda")
    with pytest.raises(RuntimeError):
        page_plan(i32([0]), i32([1]), i32([[-1]]), i32([0]), i32([1]), 1, commit=two)
    with pytest.raises(RuntimeError):
        paged_attention(*attention_inputs(1, [3], [1], 1, 1, 64, torch.int8, torch.float16), return_lse=two)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [2, 9])
@pytest.mark.parametrize("width", [0, 1200])
def test_attention_of_4096_sessions(D, G, width):
    """The most sessions a call takes, most of them without a token this tick."""
    lens = [(7 * i) % 45 for i in range(4096)]
    counts = [1 if i % 31 == 5 and n else 0 for i, n in enumerate(lens)]
    q, k, v, ks, vs, table, n, start = attention_inputs(D + G, lens, counts, 1, G, D, CODES[G % 2], torch.float16)
    if width:
        wide = torch.full((4096, width), -1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        table = wide
    assert check_attention((q, k, v, ks, vs, table, n, start), max_count=1)[2] == 0
    from infercache_b200._lib import Unsupported
    from infercache_b200.paged_ops import paged_attention
    more = [torch.cat([x, x[:1]]) for x in (table, n)]
    with pytest.raises(Unsupported):
        paged_attention(q, k, v, ks, vs, *more, torch.cat([start, start[-1:]]))


def test_two_calls_at_once_keep_apart():
    """Calls on two streams, whose workspaces and outputs are their own."""
    from infercache_b200.paged_ops import paged_attention
    calls = []
    for seed in (1, 2):
        q, k, v, ks, vs, table, n, start = attention_inputs(seed, [30000, 5000, 17], [2, 1, 1], 2, 4, 128, torch.int8, torch.float16)
        calls.append((q, k, v, ks, vs, table, n, start))
    want = [paged_attention(*c, max_count=2) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(paged_attention(*calls[i], max_count=2))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


@pytest.mark.parametrize("codes", CODES)
def test_attention_scales_far_apart(codes):
    """Page scales over 2^+-20 for V, scores of hundreds, q at bf16's extremes."""
    x = attention_inputs(3, [500, 90], [1, 2], 2, 4, 128, codes, torch.bfloat16, k_spread=6, v_spread=20)
    check_attention(x)
    q = x[0].clone()
    q[0] *= 1e30
    q[1] *= 1e-30
    check_attention((q,) + x[1:], scale=1e-30)
    check_attention(x, scale=-0.3)
    zero = x[4].clone()
    zero[:, ::2] = 0.0  # a zero V scale: those pages weigh in the softmax and add nothing
    check_attention(x[:4] + (zero,) + x[5:])


TILE_LENS, TILE_COUNTS = [700, 90, 40, 33, 513, 2000, 0, 160], [300, 1, 40, 0, 129, 260, 3, 160]


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G,D", [(2, 8, 128), (1, 7, 128), (2, 5, 64), (4, 3, 128), (1, 16, 64)])
def test_attention_prompts(codes, dtype, H, G, D):
    """Enough query rows for the tile kernel, beside sessions that are not: chunks
    on top of held tokens, whole prompts, ranges that end inside tiles and
    pages, more tokens than are held."""
    x = attention_inputs(H * G + D, TILE_LENS, TILE_COUNTS, H, G, D, codes, dtype)
    assert x[0].shape[0] * x[0].shape[1] > 4096
    _, _, status = check_attention(x, max_count=300)
    assert status == 0
    check_attention(x)


@pytest.mark.parametrize("codes", CODES)
def test_attention_prompts_hard_cases(codes):
    from infercache_b200.paged_ops import paged_attention
    x = attention_inputs(3, TILE_LENS, TILE_COUNTS, 2, 4, 128, codes, torch.bfloat16, k_spread=6, v_spread=20)
    check_attention(x)
    check_attention((x[0] * 1e30,) + x[1:], scale=1e-30)
    check_attention(x, scale=-0.3)
    zero = x[4].clone()
    zero[:, ::2] = 0.0
    check_attention(x[:4] + (zero,) + x[5:])
    t = x[5].clone()
    t[0, 2], t[5, 9] = -1, 10 ** 9
    assert check_attention(x[:5] + (t,) + x[6:])[2] == BAD_ROW
    # strided queries, rows behind the last session, a NaN that stays in its row
    n = x[0].shape[0]
    wide = torch.zeros(n + 9, 8 * 128 + 64, dtype=torch.bfloat16, device="cuda")
    wide[:n, :1024] = x[0].reshape(n, 1024)
    view, out = wide[:, :1024].view(n + 9, 8, 128), torch.full((n + 9, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    paged_attention(view, *x[1:], out=out)
    want = paged_attention(*x)
    assert torch.equal(out[:n], want) and bool((out[n:] == 3).all())
    q = x[0].clone()
    q[17, 3, 40] = math.nan
    got = paged_attention(q, *x[1:])
    assert bool(torch.isnan(got[17, 3]).all())
    got[17, 3] = want[17, 3]
    assert torch.equal(got, want)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G", [(1, 8), (2, 5), (3, 1), (1, 16)])
def test_attention_prompts_of_256_dims(codes, dtype, H, G):
    """One query tile per CTA, a ring of two key tiles."""
    x = attention_inputs(H * G, [n * 3 for n in TILE_LENS], [c * 3 for c in TILE_COUNTS], H, G, 256, codes, dtype)
    assert x[0].shape[0] * x[0].shape[1] > 4096 or H * G < 4
    assert check_attention(x)[2] == 0


def test_attention_prompts_of_256_dims_hard_cases():
    x = attention_inputs(3, TILE_LENS, TILE_COUNTS, 2, 4, 256, CODES[0], torch.bfloat16, k_spread=6, v_spread=20)
    assert x[0].shape[0] * x[0].shape[1] > 4096
    out, _, _ = check_attention(x)
    check_attention((x[0] * 1e30,) + x[1:], scale=-1e-30)
    q = x[0].clone()
    q[17, 3, 200] = math.nan
    from infercache_b200.paged_ops import paged_attention
    got = paged_attention(q, *x[1:])
    assert bool(torch.isnan(got[17, 3]).all())
    got[17, 3] = out[17, 3]
    assert torch.equal(got, out)
    t = x[5].clone()
    t[0, 2], t[5, 9] = -1, 10 ** 9
    assert check_attention(x[:5] + (t,) + x[6:])[2] == BAD_ROW


def test_attention_many_sessions_of_prompts():
    """More sessions than one pass of a CTA's threads looks through."""
    rng = np.random.default_rng(1)
    lens = rng.integers(1, 60, 700).tolist()
    counts = [min(n, int(c)) for n, c in zip(lens, rng.integers(0, 40, 700))]
    check_attention(attention_inputs(2, lens, counts, 1, 4, 64, torch.int8, torch.float16))


def test_attention_strides_padding_and_out():
    from infercache_b200.paged_ops import paged_attention
    q, k, v, ks, vs, table, lens, q_start = attention_inputs(8, [70, 20], [2, 1], 2, 4, 64, torch.int8, torch.float16)
    wide = torch.randn(7, 8 * 64 + 256, device="cuda").half()
    wide[:3, :512] = q.reshape(3, 512)
    view = wide[:, :512].view(7, 8, 64)   # a fused projection's queries and four rows behind the last session
    out = torch.full((7, 8, 64), 7.0, device="cuda").half()
    got, lse, _ = check_attention((view, k, v, ks, vs, table, lens, q_start), out=out)
    assert got is out and bool((out[3:] == 7).all())
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    a = paged_attention(swapped, k, v, ks, vs, table, lens, q_start)
    assert torch.equal(a, out[:3])
    odd = torch.empty(3 * 512 + 1, device="cuda").half()[1:].view(3, 8, 64)
    odd.copy_(q)
    assert torch.equal(paged_attention(odd, k, v, ks, vs, table, lens, q_start), a)


def test_attention_bad_pages_and_lengths():
    x = list(attention_inputs(4, [100, 40], [1, 1], 2, 8, 128, torch.float8_e4m3fn, torch.bfloat16))
    for bad in (-1, -5, 10 ** 9, x[1].shape[1] // 16):
        t = x[5].clone()
        t[0, 2] = bad
        _, _, status = check_attention(tuple(x[:5]) + (t,) + tuple(x[6:]), max_count=1)
        assert status == BAD_ROW
    # lengths past the table row are clipped to it, negative ones are empty; q_start past q is clipped
    t = x[5][:, :3].contiguous()
    t[1, 2] = t[1, 1]
    check_attention(tuple(x[:5]) + (t, i32([10 ** 6, -4]), x[7]), max_count=1)
    from infercache_b200.paged_ops import paged_attention
    a = paged_attention(*x[:7], i32([0, 1, 50]))
    assert torch.equal(a, paged_attention(*x))


def test_attention_nan_query_stays_in_its_row():
    q, *rest = attention_inputs(6, [50, 60], [2, 1], 1, 4, 64, torch.int8, torch.float16)
    from infercache_b200.paged_ops import paged_attention
    clean = paged_attention(q, *rest)
    q = q.clone()
    q[1, 2, 5] = math.nan
    got = paged_attention(q, *rest)
    assert bool(torch.isnan(got[1, 2]).all())
    got[1, 2] = clean[1, 2]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("codes", CODES)
def test_attention_offsets_past_32_bits(codes):
    """A pool whose second head's codes lie past 2^32 bytes."""
    from infercache_b200.paged_ops import page_write, paged_attention
    tokens, D = 36_000_000 // 16 * 16, 128
    k, v = (torch.zeros(2, tokens, D, dtype=torch.uint8, device="cuda").view(codes) for _ in range(2))
    ks, vs = (torch.ones(2, tokens // 16, device="cuda") for _ in range(2))
    last = tokens // 16 - 1
    x = torch.randn(2, 20, 2, D, generator=gen(1), device="cuda").half()
    slots = [(last - t // 16) * 16 + t % 16 for t in range(20)]
    page_write(x[0], x[1], k, v, ks, vs, i32(slots))
    q = torch.randn(1, 8, D, generator=gen(2), device="cuda").half()
    args = i32([[last, last - 1]]), i32([20]), i32([0, 1])
    got = paged_attention(q, k, v, ks, vs, *args, max_count=1)
    small = [t[:, -32:].contiguous() for t in (k, v)] + [t[:, -2:].contiguous() for t in (ks, vs)]
    want = paged_attention(q, *small, i32([[1, 0]]), *args[1:], max_count=1)
    assert torch.equal(got, want) and bool(got.any())


# ---- process_logits -------------------------------------------------------------------
@pytest.mark.parametrize("V", [1, 33, 1000, 32001, 151936])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("parts", ["all", "penalties", "bias", "mask", "none"])
def test_logits(V, dtype, parts):
    from infercache_b200.logits import process_logits
    S, T, B = 3, 50, 9
    rng = np.random.default_rng(V)
    x = torch.randn(S, V, generator=gen(V), device="cuda").mul(3).to(dtype)
    tokens = rng.integers(0, max(2, min(V, 40)), (S, T))
    tokens[:, ::7] = rng.integers(0, V, tokens[:, ::7].shape)
    tokens[0, :3] = [-1, V, 2 ** 31 - 1]
    lens, prompt = [T, 20, 0], [10, 30, 0]
    rep, pres, freq = [1.3, 0.7, 2.0], [0.5, -0.25, 1.0], [0.1, 0.3, 0.2]
    ids = rng.integers(-2, V + 2, (S, B))
    ids[0, 1] = ids[0, 0]
    vals = rng.normal(size=(S, B)).astype(np.float32)
    blens = [B, 4, 0]
    bits = rng.integers(0, 2, (S, -(-V // 32) * 32)).astype(bool)
    words = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
    kw, on = {}, {k: parts in ("all", k) for k in ("penalties", "bias", "mask")}
    if on["penalties"]:
        kw.update(tokens=torch.from_numpy(tokens).cuda(), token_lens=i32(lens), prompt_lens=i32(prompt),
                  repetition=torch.tensor(rep, device="cuda"), presence=torch.tensor(pres, device="cuda"),
                  frequency=torch.tensor(freq, device="cuda"))
    if on["bias"]:
        kw.update(bias_ids=i32(ids), bias_values=torch.from_numpy(vals).cuda(), bias_lens=i32(blens))
    if on["mask"]:
        kw.update(mask=torch.from_numpy(words.copy()).cuda())
    got = process_logits(x, **kw)
    f32 = lambda v: [float(np.float32(a)) for a in v]  # noqa: E731
    bias = [dict(zip(ids[r, :blens[r]].tolist(), vals[r, :blens[r]].tolist())) if on["bias"] else {} for r in range(S)]
    want = ref.logits(x.cpu(), tokens, lens if on["penalties"] else [0] * S, prompt, f32(rep), f32(pres), f32(freq), bias,
                      torch.from_numpy(bits[:, :V]) if on["mask"] else None)
    assert got.dtype == torch.float32 and got.shape == (S, V)
    got = got.cpu().double()
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    # two roundings of the penalty product, one of each term and sum: intermediates up to 2 |x| + 50 f + p + |b|
    tol = 5 * 2.0 ** -24 * (2 * x.cpu().double().abs() + 50 * 0.3 + 1 + 5)
    assert bool(((got - want).abs().nan_to_num(0, 0, 0) <= tol).all())
    if parts == "none":
        assert torch.equal(got, x.cpu().double())


def test_logits_in_place_scalars_strides_and_nan():
    from infercache_b200.logits import process_logits
    wide = torch.randn(4, 5000, generator=gen(1), device="cuda")
    tok = torch.randint(0, 900, (4, 30), generator=gen(2), device="cuda")
    view = wide[:, 100:1100]
    want = process_logits(view.clone(), tokens=tok, repetition=1.5, presence=0.5)
    before = wide.clone()
    got = process_logits(view, tokens=tok, repetition=1.5, presence=0.5, out=view)
    assert got is view and torch.equal(view, want)
    assert torch.equal(wide[:, :100], before[:, :100]) and torch.equal(wide[:, 1100:], before[:, 1100:])
    x = torch.full((1, 64), math.nan, device="cuda")
    x[0, 1:3] = torch.tensor([math.inf, -math.inf])
    y = process_logits(x, tokens=torch.arange(64, device="cuda")[None], repetition=2.0)
    assert math.isnan(float(y[0, 0])) and y[0, 1:3].tolist() == [math.inf, -math.inf]
    assert process_logits(torch.empty(0, 7, device="cuda")).shape == (0, 7)


def test_logits_matches_the_samplers_loop_bit_for_bit():
    """The loop the sampler ran before: tensor / number on the GPU multiplies by the
    reciprocal, as the kernel does."""
    from infercache_b200.logits import process_logits
    x = torch.randn(151936, generator=gen(5), device="cuda") * 4
    said = torch.randint(0, 151936, (200,), generator=gen(6), device="cuda").tolist()
    for r in (1.1, 1.3, 0.9, 2.0):
        want = x.clone()
        for t in set(said):
            want[t] = want[t] / r if want[t] > 0 else want[t] * r
        got = process_logits(x[None], tokens=torch.tensor([said], device="cuda"), repetition=r)
        assert torch.equal(got[0], want)


# ---- 8-bit pools behind the paged cache's own verbs -------------------------------------
def make_pool(dtype, pages=80, L=2, H=2, D=64, cap=40, value=torch.float16):
    from infercache_b200 import PagedCacheConfig, PagePool
    return PagePool(PagedCacheConfig(n_pages=pages, n_layers=L, n_heads=H, head_dim=D, dtype=dtype,
                                     max_pages_per_session=cap, value_dtype=value))


class Shadow:
    """One session's stored values by the reference: tokens written in order into pages of their own."""

    def __init__(self, L, H, D, dtype, tokens=640):
        self.v = np.zeros((L, H, tokens, D))
        self.s = np.zeros((L, H, tokens // 16))
        self.n, self.dtype = 0, dtype

    def push(self, x):  # [L, H, T, D]
        x = x.double().cpu().numpy()
        slots = list(range(self.n, self.n + x.shape[2]))
        for l in range(x.shape[0]):
            for h in range(x.shape[1]):
                ref.write(self.v[l, h], self.s[l, h], x[l, h], slots, self.dtype)
        self.n += x.shape[2]

    def values(self, dtype):
        return torch.from_numpy(self.v[:, :, :self.n]).to(dtype).cuda()


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("value", [torch.float16, torch.float32])
def test_multi_session_cache_over_an_8_bit_pool(dtype, value):
    from infercache_b200 import MultiSessionCache
    pool = make_pool(dtype, value=value)
    assert pool.K.dtype == dtype and abs(pool.cfg.gpu_memory_mb() - 2 * 4 * (80 * 16 * 64 + 80 * 4) / 2 ** 20) < 1e-9
    cache = MultiSessionCache(pool)
    g, shadow = gen(1), {}

    def rows(T, dt):
        return [torch.randn(2, 2, T, 64, generator=g, device="cuda").mul(1 + T % 3).to(dt) for _ in range(2)]

    for sid, T, dt in (("a", 37, torch.float16), ("b", 5, torch.bfloat16), ("a", 1, torch.float32), ("a", 20, torch.float16)):
        k, v = rows(T, dt)
        cache.get_or_create(sid).push(k, v, [], [])
        for i, x in enumerate((k, v)):
            shadow.setdefault((sid, i), Shadow(2, 2, 64, dtype)).push(x)
    ks, vs = zip(*[rows(T, dt) for T, dt in ((3, torch.float16), (18, torch.float32), (1, torch.float16))])
    assert cache.push_many(["a", "b", "c"], ks, vs) == [None] * 3
    for sid, k, v in zip("abc", ks, vs):
        for i, x in enumerate((k, v)):
            shadow.setdefault((sid, i), Shadow(2, 2, 64, dtype)).push(x)
    for sid in "abc":
        K, V = cache.get_or_create(sid).gather_all()
        assert K.dtype == value
        assert torch.equal(K, shadow[sid, 0].values(value)) and torch.equal(V, shadow[sid, 1].values(value))
        k1, v1 = cache.get_or_create(sid).gather(1)
        assert torch.equal(k1, K[1]) and torch.equal(v1, V[1])
    for (K, V), sid in zip(cache.gather_many(list("abc")), "abc"):
        assert torch.equal(K, shadow[sid, 0].values(value)) and torch.equal(V, shadow[sid, 1].values(value))
    # a released session's pages start anew for the next one, whatever their scales were
    cache.reset("a")
    k, v = rows(50, torch.float16)
    cache.get_or_create("d").push(k * 1e-3, v * 1e-3, [], [])
    s = Shadow(2, 2, 64, dtype)
    s.push(k * 1e-3)
    assert torch.equal(cache.get_or_create("d").gather_all()[0], s.values(value))
    pool.check_device_status()
    k[0, 0, 0, 0] = math.inf
    cache.get_or_create("e").push(k, v, [], [])
    with pytest.raises(ValueError):
        pool.check_device_status()


def test_pool_refusals():
    from infercache_b200 import PagedBatch
    with pytest.raises(ValueError):
        make_pool(torch.int8, D=96)
    with pytest.raises(ValueError):
        make_pool(torch.int8, value=torch.float64)
    with pytest.raises(ValueError):
        PagedBatch(make_pool(torch.float16), 4)
    pool = make_pool(torch.int8)
    for kw in (dict(pages=[1, 1]), dict(pages=[80]), dict(pages=[-1]), dict(max_pages_per_session=0)):
        with pytest.raises(ValueError):
            PagedBatch(pool, 4, **kw)
    with pytest.raises(ValueError):
        PagedBatch(pool, 0)
    b = PagedBatch(pool, 3)
    x = torch.zeros(1, 2, 64, device="cuda").half()
    for call in (lambda: b.append(0, x, x), lambda: b.attend(0, x), b.commit_plan, lambda: b.extend([1, 2]),
                 lambda: b.extend([1, -1, 0]), lambda: b.extend(i32([1, 1, 1])), lambda: b.release([0])):
        with pytest.raises(ValueError):
            call()
    b.extend([1, 0, 0])
    for call in (lambda: b.append(2, x, x), lambda: b.append(-1, x, x), lambda: b.append(0, x[:, :1], x[:, :1]),
                 lambda: b.append(0, x.repeat(2, 1, 1), x.repeat(2, 1, 1)), lambda: b.append(0, x, x.float()),
                 lambda: b.append(0, x.double(), x.double()), lambda: b.attend(0, x.float()),
                 lambda: b.attend(0, x.repeat(1, 2, 1)[:, :3]), lambda: b.attend(0, x[..., :32]),
                 lambda: b.attend(0, x.cpu()), lambda: b.attend(0, x, out=x.float()), lambda: b.gather(3, 1)):
        with pytest.raises(ValueError):
            call()


def test_pool_refuses_rows_of_another_shape():
    """Rows that the pool does not have would be read past their end."""
    pool = make_pool(torch.int8)
    good = torch.zeros(2, 2, 5, 64, device="cuda").half()
    for bad in (good[:, :1], good[..., :32], good[0]):
        with pytest.raises(ValueError):
            pool.write_rows([3], 0, bad, bad)
    with pytest.raises(ValueError):
        pool.write_rows([3], 0, good, good[:, :, :4])
    with pytest.raises(ValueError):
        pool.write_rows_many([([3], 0, good[:1], good[:1])])
    with pytest.raises(_lib_error()):
        pool.write_rows([3], 0, good, good, layer_begin=1)
    with pytest.raises(_lib_error()):
        pool.write_rows([3], 12, good, good)
    from infercache_b200 import PagedBatch
    with pytest.raises(ValueError):
        PagedBatch(pool, 4097)


def _lib_error():
    from infercache_b200 import _lib
    return _lib.InferCacheError


# ---- a run of them together ---------------------------------------------------------------
def tick_inputs(g, n, H, G, D, dtype, L):
    return [[torch.randn(n, h, D, generator=g, device="cuda").to(dtype) for h in (H, H, H * G)] for _ in range(L)]


@pytest.mark.parametrize("dtype", CODES)
def test_serving_ticks(dtype):
    """Admission, prompts in one piece and in chunks, decode, drafts of which some
    are rejected, ends and reuse: every attention call of every layer against
    the reference over the reference's own stored values."""
    from infercache_b200 import PagedBatch
    L, H, G, D, S = 2, 2, 4, 64, 4
    pool = make_pool(dtype, pages=60, L=L, H=H, D=D)
    b = PagedBatch(pool, S, max_pages_per_session=20, pages=range(2, 58))
    g = gen(11)
    vals = {(l, t): np.zeros((H, 960, D)) for l in range(L) for t in range(2)}
    scales = {(l, t): np.zeros((H, 60)) for l in range(L) for t in range(2)}
    lens = [0] * S
    ticks = [[40, 0, 7, 0], [1, 100, 1, 0], [1, 30, 1, 16], [4, 1, 3, 1], [-3, 0, -1, 0], [1, 1, 1, 1],
             [-10 ** 6, 0, -10 ** 6, 0], [17, 1, 0, 1], [1, 1, 1, 1]]
    for counts in ticks:
        if min(counts) < 0:
            keep = [max(0, n + c) if c < 0 else -1 for n, c in zip(lens, counts)]
            b.release(keep)
            lens = [n if k < 0 else k for n, k in zip(lens, keep)]
            assert b.lens.tolist() == lens
            continue
        plan = b.extend(counts)
        lens = [n + c for n, c in zip(lens, counts)]
        assert plan.lens.tolist() == lens and plan.max_count == max(counts)
        slots = plan.slots.tolist()
        assert min(slots) >= 32 and max(slots) < 58 * 16
        for l, (k, v, q) in enumerate(tick_inputs(g, sum(counts), H, G, D, torch.bfloat16, L)):
            b.append(l, k, v)
            out, lse = b.attend(l, q, return_lse=True)
            for t, x in enumerate((k, v)):
                x = x.double().cpu().numpy()
                for h in range(H):
                    ref.write(vals[l, t][h], scales[l, t][h], x[:, h], slots, dtype)
            want, wlse, tol, ltol = ref.attention(q, torch.from_numpy(vals[l, 0]).cuda(), torch.from_numpy(vals[l, 1]).cuda(),
                                                  b.block_table, lens, plan.q_start.tolist(), D ** -0.5)
            assert float(((out.double() - want).abs() - tol).max()) <= 0
            assert float(((lse.double() - wlse).abs() - ltol).max()) <= 0
    row = b.block_table[1].tolist()
    at = [row[t // 16] * 16 + t % 16 for t in range(lens[1])]
    for t, x in enumerate(b.gather(1, lens[1])):
        assert torch.equal(x.cpu(), torch.from_numpy(np.stack([vals[l, t][:, at] for l in range(L)])).half())
    b.check_device_status()
    b.extend([320, 0, 0, 0])
    with pytest.raises(RuntimeError):
        b.check_device_status()
    b.check_device_status()


def test_serving_tick_in_a_graph_matches_eager():
    """A captured tick (counts, K/V, queries in static buffers) replayed, against the
    same ticks run eagerly; two graphs over two batches replayed side by side."""
    from infercache_b200 import PagedBatch, process_logits
    S, H, G, D, n = 5, 2, 4, 128, 12
    V = 1000
    g = gen(4)
    ticks = [(torch.randn(S, H, D, generator=g, device="cuda").half(), torch.randn(S, H, D, generator=g, device="cuda").half(),
              torch.randn(S, H * G, D, generator=g, device="cuda").half()) for _ in range(2 * n)]
    tokens = torch.randint(0, V, (S, 64), generator=g, device="cuda").to(torch.int32)
    proj = torch.randn(H * G * D, V, generator=g, device="cuda").half() * 0.02

    def tick(b, k, v, q, counts):
        p = b.extend(counts, total=S, max_count=1)
        b.append(0, k, v)
        o = b.attend(0, q)
        return process_logits((o.view(S, -1) @ proj).float(), tokens=tokens, token_lens=p.lens, repetition=1.2, frequency=0.1)

    def batch():
        return PagedBatch(make_pool(torch.int8, pages=S * 3, L=1, H=H, D=D), S, max_pages_per_session=3)

    ones = torch.ones(S, dtype=torch.int32, device="cuda")
    want = []
    for half in range(2):
        b = batch()
        want.append([tick(b, *ticks[half * n + i], ones).clone() for i in range(n)])
    graphs = []
    for half in range(2):
        b, bufs = batch(), [t.clone() for t in ticks[0]]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            tick(b, *bufs, ones)
            b.release([0] * S)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = tick(b, *bufs, ones)
        torch.cuda.synchronize()
        graphs.append((b, bufs, stream, graph, out))
    for i in range(n):
        for half, (b, bufs, stream, graph, out) in enumerate(graphs):
            with torch.cuda.stream(stream):
                for dst, src in zip(bufs, ticks[half * n + i]):
                    dst.copy_(src)
                graph.replay()
        torch.cuda.synchronize()
        for half, (b, _, _, _, out) in enumerate(graphs):
            assert torch.equal(out, want[half][i]), (half, i)
            b.check_device_status()


def test_uncommitted_plan_leaves_the_batch_as_it_was():
    from infercache_b200 import PagedBatch
    b = PagedBatch(make_pool(torch.int8, L=1), 3)
    b.extend([20, 3, 0])
    lens, free = b.lens.clone(), b.free_count.clone()
    a = b.extend([30, 1, 5], commit=False)
    assert torch.equal(b.lens, lens) and torch.equal(b.free_count, free)
    c = b.extend([30, 1, 5], commit=False)
    assert all(torch.equal(x, y) for x, y in zip(a[:5], c[:5]))
    b.commit_plan()
    assert b.lens.tolist() == [50, 4, 5] and torch.equal(b.free_count, c.free_count)


def test_sampler_penalty_runs_on_the_gpu_as_the_loop_did():
    from infercache_b200 import TwoPassConfig, TwoPassEngine
    eng = TwoPassEngine.__new__(TwoPassEngine)
    x = torch.randn(5000, generator=gen(3), device="cuda") * 2
    said = torch.randint(0, 5000, (300,), generator=gen(4), device="cuda").tolist()
    for r in (1.3, 0.8, 4.0):
        eng.cfg = TwoPassConfig(temperature=0.0, repetition_penalty=r)
        want = x.clone()
        for t in set(said):
            want[t] = want[t] / r if want[t] > 0 else want[t] * r
        assert eng._sample(x, said) == int(want.argmax())
    y = torch.tensor([1.0, 3.0, 2.0], device="cuda")
    eng.cfg = TwoPassConfig(temperature=0.0, repetition_penalty=4.0)
    assert eng._sample(y, [1]) == 2 and y.tolist() == [1.0, 3.0, 2.0]
