"""GPU: the paged-cache operators against plain 64-bit forms, at the sizes, strides and masks where they can go wrong.

Tolerances. An output is rounded once to its type (half a step, eps / 2 of it). Attention also has, relative to
A = sum p |v|: f32 scores (128 products: 128 * 2^-24 of scale * sum |q k|, about 7 for normal values, so 5.5e-5 of every
weight and as much of their sum), sums over up to 2,500 keys in f32 chains of at most 1,250 (7.5e-5), and the hardware's
exp2 (2^-22): 3e-4 A covers them. Prefill rounds the weights to the type: eps / 2 of A more. The norm and rotation
are a dozen f32 operations on values below the head's norm: 1e-5 of max |y| covers them."""
import math

import pytest
import torch

import paged_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = float("nan")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def make_cache(g, lens, page, hkv, dim, dtype, layout="heads_first", spare=3, width=None):
    """Pages in random order for requests of ``lens`` tokens; everything that no request holds is NaN."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    width = width or max(need + [1])
    table = [[-1] * width for _ in lens]
    at = 0
    for r, n in enumerate(need):
        table[r][:n] = order[at:at + n]
        at += n
    shape = (pages, hkv, page, dim) if layout == "heads_first" else (pages, page, hkv, dim)
    k, v = (torch.full(shape, NAN, dtype=dtype, device=DEV) for _ in range(2))
    if layout != "heads_first":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    for r, n in enumerate(lens):
        for i in range(need[r]):
            m = min(page, n - i * page)
            for c in (k, v):
                c[table[r][i], :, :m] = torch.randn(hkv, m, dim, generator=g, device=DEV).to(dtype)
    return k, v, table


def check(out, ref, mag, dtype, p_rounded):
    h = half(dtype)
    tol = h * ref.abs() * 1.01 + (3e-4 + (h if p_rounded else 0.0)) * mag + 1e-30
    assert torch.isfinite(out).all()
    off = (out.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


# ---- plan and release ----------------------------------------------------------------------------


def run_plan(pkg, new, lengths, table, free, count, page, total, in_place):
    t, ln, c = ints(table), ints(lengths), ints([count])
    f = ints(free) if free else torch.empty(0, dtype=torch.int32, device=DEV)
    lo, co = (None, None) if in_place else (torch.empty_like(ln), torch.empty_like(c))
    p = pkg.paged_plan(ints(new), ln, t, f, c, page, total, lengths_out=lo, free_count_out=co)
    if not in_place:
        assert ln.tolist() == lengths and c.tolist() == [count]
        ln, c = lo, co
    return dict(slots=p.slots.tolist(), positions=p.positions.tolist(), cu=p.cu_tokens.tolist(), kv=p.kv_lens.tolist(),
                status=p.status.tolist(), held=ln.tolist(), count=c.tolist()[0]), t.tolist()


def plan_case(n, longest, page, width, pool, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda hi: int(torch.randint(0, hi + 1, (1,), generator=g))   # noqa: E731
    lengths = [r(width * page) for _ in range(n)]
    new = [r(longest) if r(3) else 1 for _ in range(n)]
    table, at = [[-1] * width for _ in range(n)], 0
    for b, a in enumerate(lengths):
        for i in range(-(-a // page)):
            table[b][i] = at
            at += 1
    free = list(range(at, at + pool))
    return new, lengths, table, free


@pytest.mark.parametrize("n,longest,page,width,pool,total", [
    (1, 1, 16, 4, 3, 1), (3, 0, 64, 2, 5, 0), (64, 1, 64, 20, 80, 64), (5, 40, 1, 50, 300, 300), (7, 200, 16, 9, 30, 2000),
    (400, 30, 16, 12, 5000, 9000), (1100, 3, 32, 6, 2000, 5000), (2500, 5, 16, 3, 700, 20000), (40, 700, 128, 8, 900, 30000),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(pkg, n, longest, page, width, pool, total, in_place):
    new, lengths, table, free = plan_case(n, longest, page, width, pool, n + page)
    got, got_table = run_plan(pkg, new, lengths, table, free, len(free), page, total, in_place)
    ref = oracle.plan(new, lengths, table, free, len(free), page, total)
    for key in ref:
        assert got[key] == ref[key], key
    assert got_table == table


def test_plan_refusals_and_padding(pkg):
    """Too few pages (nothing overtakes, requests that need none go on), a full table row, tokens past the arrays, counts
    and lengths below 0, an empty pool, padding behind the last token."""
    cases = [([1, 20, 1, 5], [0, 0, 16, 3], 2, 4, 40), ([1, 1, 200, 1], [15, 16, 0, 1], 9, 3, 300), ([4, 4, 4], [0, 0, 0], 9, 3, 7),
             ([-3, 2], [-1, 4], 4, 2, 5), ([1, 1], [0, 5], 0, 2, 2)]
    for new, lengths, pool, width, total in cases:
        table = [[100 + 10 * b + i if i * 16 < a else -1 for i in range(width)] for b, a in enumerate(lengths)]
        free = list(range(pool))
        got, got_table = run_plan(pkg, new, lengths, table, free, pool, 16, total, True)
        ref = oracle.plan(new, [max(a, 0) for a in lengths], table, free, pool, 16, total)
        assert got == ref and got_table == table, (new, lengths)


def test_release_gives_pages_back(pkg):
    page, width, n = 16, 5, 1500
    new, lengths, table, _ = plan_case(n, 1, page, width, 0, 5)
    pages = sum(-(-a // page) for a in lengths)
    free = [7000, 7001] + [0] * pages
    flags = [int(b % 3 != 1) for b in range(n)]
    t, ln, f, c = ints(table), ints(lengths), ints(free), ints([2])
    pkg.paged_release(ints(flags), ln, t, f, c, page)
    back = [p for b in range(n) if flags[b] for p in table[b] if p >= 0]
    assert c.item() == 2 + len(back) and f.tolist()[:2 + len(back)] == [7000, 7001] + back
    assert ln.tolist() == [0 if flags[b] else lengths[b] for b in range(n)]
    assert t.tolist() == [[-1] * width if flags[b] else table[b] for b in range(n)]
    pkg.paged_release(ints(flags), ln, t, f, c, page)                 # a second release gives nothing
    assert c.item() == 2 + len(back)
    got, _ = run_plan(pkg, [page], [0], [[-1]], f.tolist(), c.item(), page, page, True)
    assert got["slots"][0] == back[-1] * page and got["count"] == 1 + len(back)


def test_release_passes_over_empty_entries(pkg):
    t, ln, f, c = ints([[3, -1, 5, 9]]), ints([40]), ints([0] * 4), ints([0])
    pkg.paged_release(ints([1]), ln, t, f, c, 16)
    assert c.item() == 2 and f.tolist()[:2] == [3, 5] and t.tolist() == [[-1, -1, -1, 9]]


# ---- norms, rotation, store ----------------------------------------------------------------------


@pytest.mark.parametrize("tokens,hq,hkv,dim,page,dtype,mrope,fused,f32,norm", [
    (1, 16, 8, 128, 64, torch.bfloat16, False, True, False, True), (5, 16, 8, 128, 16, torch.bfloat16, True, True, False, True),
    (67, 16, 8, 128, 32, torch.bfloat16, True, False, True, True), (4100, 16, 8, 128, 64, torch.bfloat16, False, True, False, True),
    (33, 3, 1, 64, 16, torch.float16, False, False, True, True), (259, 20, 4, 64, 128, torch.float16, True, True, False, False),
    (4099, 5, 5, 64, 16, torch.bfloat16, False, False, False, True), (18, 1, 1, 128, 16, torch.float16, False, True, True, False),
])
def test_store(pkg, tokens, hq, hkv, dim, page, dtype, mrope, fused, f32, norm):
    g = gen(tokens)
    rows = 500
    angle = torch.rand(rows, dim // 2, generator=g, device=DEV, dtype=torch.float64) * 6.28
    tt = torch.float32 if f32 else dtype
    cos, sin = (torch.cat((f(angle), f(angle)), -1).to(tt) for f in (torch.cos, torch.sin))
    if fused:
        q, k, v = torch.randn(tokens, (hq + 2 * hkv) * dim, generator=g, device=DEV).to(dtype).split([hq * dim, hkv * dim, hkv * dim], 1)
        q, k, v = q.view(tokens, hq, dim), k.view(tokens, hkv, dim), v.view(tokens, hkv, dim)
    else:                                          # heads before tokens
        q, k, v = (torch.randn(h, tokens, dim, generator=g, device=DEV).to(dtype).transpose(0, 1) for h in (hq, hkv, hkv))
    wq, wk = (((1 + 0.2 * torch.randn(dim, generator=g, device=DEV)).to(dtype) if norm else None) for _ in range(2))
    pos = torch.randint(-3, rows + 5, (3, tokens), generator=g, device=DEV, dtype=torch.int32)   # clamped into the tables
    section = (24, 20, 20) if dim == 128 else (12, 10, 10)
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:tokens].to(torch.int32)
    if tokens > 4:                                 # tokens without a place: nothing of them is written
        slots[2], slots[4] = -1, pages * page
    kc, vc = (torch.randn(pages, hkv, page, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    want_k, want_v = kc.double(), vc.double()
    out = torch.full((tokens, hq, dim), 7.0, dtype=dtype, device=DEV)
    got = pkg.qk_norm_rope_store(q, k, v, wq, wk, cos, sin, pos if mrope else pos[0].contiguous(), slots, kc, vc, eps=1e-5,
                                 mrope_section=section, out=out)
    assert got.data_ptr() == out.data_ptr()
    p = pos.long().clamp(0, rows - 1)
    d = torch.arange(dim // 2, device=DEV)
    sec = torch.where((d % 3 == 1) & (d < 3 * section[1]), 1, torch.where((d % 3 == 2) & (d < 3 * section[2]), 2, 0)) if mrope else 0 * d
    c, s = cos.double()[p[sec].T, d], sin.double()[p[sec].T, d]
    qr, kr = oracle.norm_rope(q, wq, c, s, 1e-5), oracle.norm_rope(k, wk, c, s, 1e-5)
    ok = (slots >= 0) & (slots < pages * page)
    sl = slots[ok].long()
    want_k[sl // page, :, sl % page] = kr[ok]
    want_v[sl // page, :, sl % page] = v[ok].double()
    want_q = torch.where(ok[:, None, None], qr, torch.full_like(qr, 7.0))
    h = half(dtype)
    for a, b in ((got, want_q), (kc, want_k)):
        assert bool(((a.double() - b).abs() <= 1.01 * h * b.abs() + 1e-5 * b.abs().max()).all())
    assert torch.equal(vc.double(), want_v)


def test_store_in_place_and_empty(pkg):
    g = gen(3)
    q, k, v = (torch.randn(9, h, 128, generator=g, device=DEV).to(torch.bfloat16) for h in (16, 8, 8))
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    cos, sin = (torch.rand(20, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    kc, vc = (torch.zeros(2, 8, 16, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    pos, slots = ints(list(range(9))), ints(list(range(9)))
    a = pkg.qk_norm_rope_store(q, k, v, w, w, cos, sin, pos, slots, kc, vc)
    b = pkg.qk_norm_rope_store(q, k, v, w, w, cos, sin, pos, slots, kc, vc, out=q)
    assert torch.equal(a, b) and b.data_ptr() == q.data_ptr()
    e = pkg.qk_norm_rope_store(q[:0], k[:0], v[:0], w, w, cos, sin, pos[:0], slots[:0], kc, vc)
    assert e.shape == (0, 16, 128)


# ---- attention -----------------------------------------------------------------------------------

HEADS = [(16, 8, 128), (4, 4, 64), (9, 3, 128), (20, 1, 64), (16, 1, 128), (40, 2, 128)]


@pytest.mark.parametrize("hq,hkv,dim", HEADS)
@pytest.mark.parametrize("dtype,page,layout", [(torch.bfloat16, 16, "heads_first"), (torch.float16, 64, "tokens_first")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (37, 3), (300, 50), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_decode(pkg, hq, hkv, dim, dtype, page, layout, window, sinks):
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 64, 129, 511, 640, 1025, 2100]
    g = gen(hq * dim + window)
    k, v, table = make_cache(g, lens, page, hkv, dim, dtype, layout)
    q = torch.randn(len(lens), hq, dim, generator=g, device=DEV).to(dtype)
    ref, mag = oracle.attend(q, k, v, table, [n - 1 for n in lens], hq // hkv, window, sinks, dim ** -0.5)
    for max_len in (None, 2100, 1, 700):           # too short a promise only moves the split
        out = pkg.paged_attention_decode(q, k, v, ints(table), ints(lens), window=window, sinks=sinks, max_len=max_len)
        assert bool((out[0] == 0).all())
        check(out, ref, mag, dtype, False)


PROMPTS = [(0, 1), (0, 0), (5, 1), (0, 63), (0, 64), (1, 65), (40, 30), (100, 0), (7, 129), (300, 17), (0, 200), (513, 5)]


@pytest.mark.parametrize("hq,hkv,dim", HEADS)
@pytest.mark.parametrize("dtype,page,layout", [(torch.bfloat16, 16, "heads_first"), (torch.float16, 64, "tokens_first")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (37, 3), (100, 70), (2 ** 31 - 1, 5)])
def test_prefill(pkg, hq, hkv, dim, dtype, page, layout, window, sinks):
    run_prefill(pkg, PROMPTS, hq, hkv, dim, dtype, page, layout, window, sinks)


def run_prefill(pkg, prompts, hq, hkv, dim, dtype, page, layout, window, sinks, pad=3, **kw):
    lens = [a + n for a, n in prompts]
    g = gen(hq * dim + window)
    k, v, table = make_cache(g, lens, page, hkv, dim, dtype, layout)
    total = sum(n for _, n in prompts)
    q = torch.randn(total + pad, hq, dim, generator=g, device=DEV).to(dtype)
    rows = [table[r] for r, (a, n) in enumerate(prompts) for _ in range(n)]
    pos = [a + i for a, n in prompts for i in range(n)]
    cu = [sum(n for _, n in prompts[:r]) for r in range(len(prompts) + 1)]
    out = torch.full_like(q, 5.0)
    got = pkg.paged_attention_prefill(q, k, v, ints(table), ints(lens), ints(cu), window=window, sinks=sinks, out=out, **kw)
    ref, mag = oracle.attend(q[:total], k, v, rows, pos, hq // hkv, window, sinks, dim ** -0.5)
    check(got[:total], ref, mag, dtype, True)
    assert bool((got[total:] == 5.0).all())         # rows behind the last request
    return got


@pytest.mark.parametrize("hq,hkv,dim", [(40, 2, 128), (80, 2, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 40)])
@pytest.mark.parametrize("max_len", [1, 200, 700])
def test_prefill_tiles(pkg, hq, hkv, dim, dtype, window, sinks, max_len):
    """What the host says of the longest request chooses the tile: 1 the rows unsplit, 200 two key splits, 700 four (two
    under the window). Nothing that is computed depends on it."""
    run_prefill(pkg, PROMPTS, hq, hkv, dim, dtype, 32, "heads_first", window, sinks, max_len=max_len)


@pytest.mark.parametrize("max_len", [1, 200, 700])
def test_not_finite_in_each_tile(pkg, max_len):
    """Per tile: an infinite V that half of the rows see, queries that are NaN; the other rows and requests as they were."""
    g = gen(31)
    prompts = PROMPTS[1:]
    lens = [a + n for a, n in prompts]
    k, v, table = make_cache(g, lens, 32, 2, 128, torch.bfloat16)
    total = sum(n for _, n in prompts)
    cu = [sum(n for _, n in prompts[:r]) for r in range(len(prompts) + 1)]
    q = (0.2 * torch.randn(total, 40, 128, generator=g, device=DEV)).to(torch.bfloat16)
    call = lambda: pkg.paged_attention_prefill(q, k, v, ints(table), ints(lens), ints(cu), max_len=max_len)
    before = call()
    v[table[9][100 // 32], :, 100 % 32, 5] = float("inf")     # the request of 200 tokens: rows 100 .. see it
    q[cu[4] + 3] = NAN                                        # a row of the request of 65
    after = call()
    rows = torch.ones(total, dtype=torch.bool, device=DEV)
    rows[cu[9] + 100:cu[10]] = False
    rows[cu[4] + 3] = False
    assert torch.isfinite(after[rows].float()).all()
    assert float((after[rows].float() - before[rows].float()).abs().max()) < 0.02     # (rows summed again in 32 bits)
    assert bool((after[cu[9] + 100:cu[10], :, 5] == float("inf")).all()) and bool(after[cu[4] + 3].isnan().all())
    rest = [d for d in range(128) if d != 5]
    assert torch.isfinite(after[cu[9] + 100:cu[10]][:, :, rest].float()).all()


def test_prefill_many_requests(pkg):
    """More requests than a wave's lanes, most of them with a token or none."""
    prompts = [(r % 7, r % 3) for r in range(150)] + [(20, 140)]
    run_prefill(pkg, prompts, 16, 8, 128, torch.bfloat16, 16, "heads_first", 0, 0)


@pytest.mark.parametrize("prompts", [[(0, 400)] * 3 + [(0, 0), (0, 7), (2, 333)], [(0, 1)] * 30 + [(0, 0)] * 20 + [(0, 300)] * 14,
                                     [(0, 90), (0, 0), (0, 700)]])
@pytest.mark.parametrize("hq,hkv,dim,dtype", [(16, 8, 128, torch.bfloat16), (9, 3, 64, torch.float16)])
def test_prefill_tiles_of_many_requests_in_one_order(pkg, prompts, hq, hkv, dim, dtype):
    """Prompts whose keys grow with their tiles: the longest tiles of all of them first. Lengths shorter than the tokens
    and padding beside them."""
    run_prefill(pkg, prompts, hq, hkv, dim, dtype, 16, "tokens_first", 0, 0, max_len=max(a + n for a, n in prompts))
    n = 150
    g = gen(8)
    k, v, table = make_cache(g, [n, n, n, n], 16, hkv, dim, dtype)
    q = torch.randn(4 * n + 5, hq, dim, generator=g, device=DEV).to(dtype)
    lens, cu = [n, 0, 40, n], [0, n, 2 * n, 3 * n, 4 * n]     # a refused request, one shorter than its tokens
    out = pkg.paged_attention_prefill(q, k, v, ints(table), ints(lens), ints(cu), max_len=n, out=torch.full_like(q, 5.0))
    pos = [lens[r] - n + i for r in range(4) for i in range(n)]
    ref, mag = oracle.attend(q[:4 * n], k, v, [table[r] for r in range(4) for _ in range(n)], pos, hq // hkv, 0, 0, dim ** -0.5)
    check(out[:4 * n], ref, mag, dtype, True)
    assert bool((out[4 * n:] == 5.0).all())


def test_prefill_longer(pkg):
    run_prefill(pkg, [(700, 600), (0, 333)], 4, 2, 128, torch.bfloat16, 32, "heads_first", 0, 0)
    run_prefill(pkg, [(1500, 40)], 4, 2, 64, torch.float16, 32, "heads_first", 200, 9)


def test_decode_equals_prefill_of_one_token(pkg):
    lens = [1, 40, 333]
    g = gen(1)
    k, v, table = make_cache(g, lens, 16, 8, 128, torch.bfloat16)
    q = torch.randn(3, 16, 128, generator=g, device=DEV).to(torch.bfloat16)
    a = pkg.paged_attention_decode(q, k, v, ints(table), ints(lens))
    b = pkg.paged_attention_prefill(q, k, v, ints(table), ints(lens), ints([0, 1, 2, 3]))
    assert float((a.double() - b.double()).abs().max()) < 0.02


def test_tokens_before_position_zero_get_zeros(pkg):
    """A refused request's length is 0, with its tokens still packed; a length below the new tokens' count."""
    g = gen(2)
    k, v, table = make_cache(g, [40, 40, 40], 16, 8, 128, torch.bfloat16)
    q = torch.randn(30, 16, 128, generator=g, device=DEV).to(torch.bfloat16)
    out = pkg.paged_attention_prefill(q, k, v, ints(table), ints([0, 40, 4]), ints([0, 10, 20, 30]))
    ref, mag = oracle.attend(q, k, v, [table[0]] * 10 + [table[1]] * 10 + [table[2]] * 10,
                             list(range(-10, 0)) + list(range(30, 40)) + list(range(-6, 4)), 2, 0, 0, 128 ** -0.5)
    assert bool((out[:10] == 0).all()) and bool((out[20:26] == 0).all())
    check(out, ref, mag, torch.bfloat16, True)


def test_pages_outside_the_cache_are_not_seen(pkg):
    g = gen(4)
    lens = [70, 100, 33]
    k, v, table = make_cache(g, lens, 16, 8, 128, torch.bfloat16)
    table[0][1], table[0][4], table[1][0], table[1][6] = -1, 1 << 30, k.shape[0], -2147483648
    table[2] = [-1] * len(table[2])
    q = torch.randn(3, 16, 128, generator=g, device=DEV).to(torch.bfloat16)
    ref, mag = oracle.attend(q, k, v, table, [n - 1 for n in lens], 2, 0, 0, 128 ** -0.5)
    check(pkg.paged_attention_decode(q, k, v, ints(table), ints(lens)), ref, mag, torch.bfloat16, False)
    out = pkg.paged_attention_prefill(q, k, v, ints(table), ints(lens), ints([0, 1, 2, 3]))
    check(out, ref, mag, torch.bfloat16, True)
    assert bool((out[2] == 0).all())


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), NAN])
def test_hidden_keys_that_are_not_finite(pkg, bad):
    """An infinite or NaN K and V that some rows of a tile see and others do not: the others are untouched."""
    g = gen(5)
    n = 90
    k, v, table = make_cache(g, [n], 16, 2, 128, torch.bfloat16)
    for c, at in ((v, 50), (k, 70)):
        c[table[0][at // 16], :, at % 16] = bad
    q = torch.randn(n, 4, 128, generator=g, device=DEV).to(torch.bfloat16)
    out = pkg.paged_attention_prefill(q, k, v, ints(table), ints([n]), ints([0, n]), window=15, sinks=2)
    clean = [i for i in range(n) if not any(a in (50, 70) for a in oracle.visible(i, 15, 2))]
    ref, mag = oracle.attend(q, k, v, [table[0]] * n, list(range(n)), 2, 15, 2, 128 ** -0.5)
    check(out[clean], ref[clean], mag[clean], torch.bfloat16, True)
    assert len(clean) == n - 30
    dirty = torch.tensor([i for i in range(n) if i not in clean], device=DEV)
    fin = torch.isfinite(ref[dirty])
    assert torch.equal(torch.isfinite(out[dirty].double()), fin)
    one = pkg.paged_attention_decode(q[:1], k, v, ints(table), ints([66]), window=15)
    r1, m1 = oracle.attend(q[:1], k, v, table, [65], 2, 15, 0, 128 ** -0.5)
    check(one, r1, m1, torch.bfloat16, False)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_infinite_values_that_are_seen(pkg, dtype, dim):
    """A visible infinite V makes its channels infinite (both signs: NaN) and leaves the other channels alone."""
    g = gen(12)
    lens = [700, 40]
    k, v, table = make_cache(g, lens, 16, 2, dim, dtype)
    inf = float("inf")
    for r, at, d, x in ((0, 650, 3, inf), (0, 20, 5, -inf), (0, 30, 7, inf), (0, 500, 7, -inf), (1, 39, 1, inf)):
        v[table[r][at // 16], :, at % 16, d] = x
    q = (0.2 * torch.randn(2, 4, dim, generator=g, device=DEV)).to(dtype)   # weights of 1e-3 and more: none rounds to 0
    ref, mag = oracle.attend(q, k, v, table, [n - 1 for n in lens], 2, 0, 0, dim ** -0.5)
    one = pkg.paged_attention_decode(q, k, v, ints(table), ints(lens))
    two = pkg.paged_attention_prefill(q, k, v, ints(table), ints(lens), ints([0, 1, 2]))
    fin = torch.isfinite(ref)
    assert int((~fin).sum()) == 4 * 3 + 4
    for out in (one, two):
        o = out.double()
        assert torch.equal(torch.isfinite(o), fin) and torch.equal(torch.isnan(o), torch.isnan(ref))
        assert torch.equal(o[~fin & ~torch.isnan(ref)], ref[~fin & ~torch.isnan(ref)])
        h = half(dtype)
        assert bool(((o - ref).abs() <= 1.01 * h * ref.abs() + (3e-4 + h) * mag)[fin].all())


def test_large_scores_and_scale(pkg):
    """Scores of some thousands: the running maximum keeps every weight finite."""
    g = gen(6)
    lens = [300]
    k, v, table = make_cache(g, lens, 16, 8, 128, torch.bfloat16)
    q = (torch.randn(300, 16, 128, generator=g, device=DEV) * 300).to(torch.bfloat16)
    ref, _ = oracle.attend(q, k, v, [table[0]] * 300, list(range(300)), 2, 0, 0, 0.5)
    out = pkg.paged_attention_prefill(q, k, v, ints(table), ints(lens), ints([0, 300]), scale=0.5)
    one = pkg.paged_attention_decode(q[299:], k, v, ints(table), ints(lens), scale=0.5)
    # scores up to 2^13: f32 steps of 2^-10 each, 128 products: weights off by at most e^(128 * 2^-11) - 1 = 6.5 %
    for a, b in ((out, ref), (one, ref[299:])):
        assert torch.isfinite(a).all() and float((a.double() - b).abs().max()) < 0.065 * float(v[~v.isnan()].abs().max())


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.float16, 128), (torch.bfloat16, 128)])
@pytest.mark.parametrize("max_len", [1, 8001])
def test_many_small_weights(pkg, dtype, dim, max_len):
    """One key of weight 1 and 8000 of 4e-5 (below fp16's normal numbers): together they weigh a fourth, and V is 1 for
    the one and 2 for the others."""
    n = 8001
    table = [list(range(-(-n // 16)))]
    k = torch.zeros(len(table[0]), 1, 16, dim, device=DEV, dtype=dtype)
    v = torch.full_like(k, 2.0)
    k[70, 0, 5, 0], v[70, 0, 5] = 1.0, 1.0
    q = torch.zeros(2, 3, dim, device=DEV, dtype=dtype)
    q[:, :, 0] = 10.125                                       # e^-10.125 = 4.006e-5
    w = 8000 * math.exp(-10.125)
    one = pkg.paged_attention_decode(q[:1], k, v, ints(table), ints([n]), scale=1.0)
    two = pkg.paged_attention_prefill(q[:1], k, v, ints(table), ints([n]), ints([0, 1]), scale=1.0, max_len=max_len)
    # the output's half step, and a weight's rounding (4e-5 in fp16: steps of 2^-24, 7.4e-4 of it at most) in its share
    tol = half(dtype) * 2 + (7.5e-4 if dtype == torch.float16 else half(dtype)) * w / (1 + w) * 2 + 3e-4
    for out in (one, two):
        assert float((out.double() - (1 + 2 * w) / (1 + w)).abs().max()) < tol


def test_strides_and_tables(pkg):
    """Query and output views, a block table that is part of a wider one, a cache inside a larger allocation."""
    g = gen(7)
    lens = [77, 5, 130]
    k0, v0, table = make_cache(g, lens, 16, 8, 128, torch.bfloat16)
    big = torch.full((2, k0.shape[0], 11, 16, 3, 128), NAN, dtype=torch.bfloat16, device=DEV)
    k, v = big[0, :, 1:9, :, 2], big[1, :, 1:9, :, 2]
    k.copy_(k0)
    v.copy_(v0)
    wide = torch.full((5, 40), -7, dtype=torch.int32, device=DEV)
    t = wide[1:4, 2:2 + len(table[0])]
    t.copy_(ints(table))
    q = torch.randn(20, 3, 128, generator=g, device=DEV).to(torch.bfloat16).transpose(0, 1)[:, 2:18]
    o = torch.empty(3, 16, 2, 128, dtype=torch.bfloat16, device=DEV)[:, :, 1]
    ref, mag = oracle.attend(q, k0, v0, table, [n - 1 for n in lens], 2, 0, 0, 128 ** -0.5)
    check(pkg.paged_attention_decode(q, k, v, t, ints(lens), out=o), ref, mag, torch.bfloat16, False)
    check(pkg.paged_attention_prefill(q, k, v, t, ints(lens), ints([0, 1, 2, 3]), out=o), ref, mag, torch.bfloat16, True)


def test_offsets_past_32_bits(pkg):
    """Pages more than 2^32 bytes apart, written and read."""
    stride, pages = 1 << 27, 36                    # 36 pages, 256 MiB apart
    room = torch.empty(2, (pages - 1) * stride + 8 * 16 * 128, dtype=torch.bfloat16, device=DEV)
    k, v = (room[i].as_strided((pages, 8, 16, 128), (stride, 2048, 128, 1)) for i in range(2))
    g = gen(8)
    table = [[35, 0, 20, 34], [33, 1, 17, 2]]
    n = 61
    kk, vv, q = (torch.randn(n, h, 128, generator=g, device=DEV).to(torch.bfloat16) for h in (8, 8, 16))
    cos, sin = torch.ones(4, 128, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 128, dtype=torch.bfloat16, device=DEV)
    for row in table:
        slots = ints([row[i // 16] * 16 + i % 16 for i in range(n)])
        qr = pkg.qk_norm_rope_store(q, kk, vv, None, None, cos, sin, ints([0] * n), slots, k, v)
        assert torch.equal(qr, q)
    ks, vs = (torch.zeros(pages, 8, 16, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for row in table:
        for i, p in enumerate(row):
            m = min(16, n - 16 * i)
            ks[p, :, :m], vs[p, :, :m] = kk[16 * i:16 * i + m].transpose(0, 1), vv[16 * i:16 * i + m].transpose(0, 1)
            assert torch.equal(k[p, :, :m], ks[p, :, :m]) and torch.equal(v[p, :, :m], vs[p, :, :m])
    ref, mag = oracle.attend(q[:2], ks, vs, table, [n - 1] * 2, 2, 0, 0, 128 ** -0.5)
    check(pkg.paged_attention_decode(q[:2], k, v, ints(table), ints([n, n])), ref, mag, torch.bfloat16, False)
    ref, mag = oracle.attend(q, ks, vs, [table[0]] * n, list(range(n)), 2, 0, 0, 128 ** -0.5)
    check(pkg.paged_attention_prefill(q, k, v, ints(table[:1]), ints([n]), ints([0, n])), ref, mag, torch.bfloat16, True)


def test_results_repeat_bit_for_bit(pkg):
    g = gen(9)
    lens = [3000, 17, 1200]
    k, v, table = make_cache(g, lens, 64, 8, 128, torch.bfloat16)
    q = torch.randn(3, 16, 128, generator=g, device=DEV).to(torch.bfloat16)
    first = pkg.paged_attention_decode(q, k, v, ints(table), ints(lens))
    for _ in range(5):
        assert torch.equal(first, pkg.paged_attention_decode(q, k, v, ints(table), ints(lens)))


# ---- refusals, streams, graphs -------------------------------------------------------------------


def test_refusals(pkg):
    """Every call that a kernel could not carry out raises, and nothing is written."""
    k = torch.zeros(4, 8, 16, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    q = torch.zeros(3, 16, 128, dtype=torch.bfloat16, device=DEV)
    t, lens, cu = ints([[0, 1], [2, 3], [0, 0]]), ints([1, 2, 3]), ints([0, 1, 2, 3])
    tab = torch.zeros(9, 128, dtype=torch.bfloat16, device=DEV)
    pos = ints([0, 1, 2])

    def decode(**kw):
        a = dict(q=q, k_cache=k, v_cache=v, block_table=t, kv_lens=lens)
        a.update(kw)
        return pkg.paged_attention_decode(**a)

    def prefill(**kw):
        a = dict(q=q, k_cache=k, v_cache=v, block_table=t, kv_lens=lens, cu_tokens=cu)
        a.update(kw)
        return pkg.paged_attention_prefill(**a)

    def store(**kw):
        a = dict(q=q, k=q[:, :8], v=q[:, :8], q_weight=None, k_weight=None, cos=tab, sin=tab, positions=pos, slots=pos, k_cache=k, v_cache=v)
        a.update(kw)
        return pkg.qk_norm_rope_store(**a)

    both = [dict(q=q.half()), dict(q=q[:, :12]), dict(q=q[..., :64]), dict(q=q.cpu()), dict(v_cache=v[:2]), dict(v_cache=v.half()),
            dict(k_cache=k.float(), v_cache=v.float()), dict(k_cache=k[:, :, :12], v_cache=v[:, :, :12]),
            dict(k_cache=k[..., :96], v_cache=v[..., :96]), dict(block_table=t.long()), dict(block_table=t[0]), dict(block_table=t.T),
            dict(block_table=t.cpu()), dict(kv_lens=lens.long()), dict(kv_lens=lens[:2]), dict(scale=0.0), dict(scale=-1.0),
            dict(scale=float("nan")), dict(window=-1), dict(sinks=-2), dict(max_len=0), dict(out=q[:2]), dict(out=q.half()),
            dict(q=torch.zeros(3, 16, 256, dtype=torch.bfloat16, device=DEV)[..., ::2]),
            dict(q=torch.zeros(3 * 16 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(3, 16, 128))]
    for bad in both:
        with pytest.raises(RuntimeError):
            decode(**bad)
        with pytest.raises(RuntimeError):
            prefill(**bad)
    with pytest.raises(RuntimeError):
        prefill(cu_tokens=cu.long())
    with pytest.raises(RuntimeError):
        prefill(cu_tokens=ints([0, 1, 2, 3, 3]))          # four requests, three lengths
    for bad in (dict(k=q), dict(v=q[:2, :8]), dict(q=q.half()), dict(cos=tab[:, :64]), dict(sin=tab[:4]), dict(cos=tab.half()), dict(positions=pos[:2]),
                dict(positions=pos.long()), dict(positions=torch.stack([pos, pos])), dict(slots=pos[:2]), dict(slots=ints([0, 1, 2, 3])),
                dict(slots=pos.cpu()), dict(q_weight=tab[0, :64]), dict(k_weight=tab[0].float()), dict(eps=-1.0), dict(out=q[:, :8]),
                dict(positions=torch.stack([pos] * 3), mrope_section=(24, 20, 21)),
                dict(positions=torch.stack([pos] * 3), mrope_section=(0, 32, 32))):
        with pytest.raises(RuntimeError):
            store(**bad)
    one = ints([1])
    for bad in (dict(new_tokens=one.long()), dict(lengths=ints([])), dict(block_table=ints([1])), dict(page_size=24), dict(page_size=0),
                dict(total_tokens=-1), dict(free_count=ints([])), dict(lengths_out=one.cpu())):
        a = dict(new_tokens=one, lengths=ints([0]), block_table=ints([[-1]]), free_pages=ints([3]), free_count=ints([1]), page_size=16, total_tokens=1)
        a.update(bad)
        with pytest.raises(RuntimeError):
            pkg.paged_plan(**a)
    for bad in (dict(out=q[:1].expand(3, 16, 128)), dict(out=q[:, :1].expand(3, 16, 128))):
        for call in (decode, prefill, store):
            with pytest.raises(RuntimeError, match="overlap|single memory"):
                call(**bad)
    with pytest.raises(RuntimeError, match="overlap|single memory"):
        store(k_cache=k[:1].expand(4, 8, 16, 128), v_cache=v[:1].expand(4, 8, 16, 128))
    assert bool((k == 0).all()) and bool((v == 0).all())
    assert store().shape == (3, 16, 128) and decode().shape == (3, 16, 128)


def step_state(seed, dtype=torch.bfloat16):
    """A batch before a step: pages, lengths and one layer's cache."""
    g = gen(seed)
    lens = [37, 0, 300, 64]
    k, v, table = make_cache(g, lens, 16, 8, 128, dtype, spare=40, width=24)
    used = {p for row in table for p in row}
    free = [p for p in range(k.shape[0]) if p not in used]
    angle = torch.rand(400, 64, generator=g, device=DEV) * 6
    cos, sin = (torch.cat((f(angle), f(angle)), -1).to(dtype) for f in (torch.cos, torch.sin))
    qkv = torch.randn(4, 32, 128, generator=g, device=DEV).to(dtype)
    w = torch.ones(128, dtype=dtype, device=DEV)
    return dict(k=k, v=v, table=ints(table), lens=ints(lens), free=ints(free), count=ints([len(free)]), cos=cos, sin=sin, qkv=qkv, w=w,
                new=ints([1, 1, 1, 1]))


def step(pkg, s, max_len=None):
    """One layer's step as a server runs it: plan, store, attend (lengths grow in place)."""
    p = pkg.paged_plan(s["new"], s["lens"], s["table"], s["free"], s["count"], 16, 4)
    q, k, v = s["qkv"][:, :16], s["qkv"][:, 16:24], s["qkv"][:, 24:]
    q = pkg.qk_norm_rope_store(q, k, v, s["w"], s["w"], s["cos"], s["sin"], p.positions, p.slots, s["k"], s["v"])
    a = pkg.paged_attention_decode(q, s["k"], s["v"], s["table"], p.kv_lens, max_len=max_len)
    b = pkg.paged_attention_prefill(q, s["k"], s["v"], s["table"], p.kv_lens, p.cu_tokens, window=50, sinks=2)
    return a, b


def test_a_run_of_steps(pkg):
    """Steps on end, each against the 64-bit form on the cache as it then is; pages come in as lengths pass their end."""
    s = step_state(1)
    for i in range(20):
        a, b = step(pkg, s)
        lens, table = s["lens"].tolist(), s["table"].tolist()
        assert lens == [38 + i, 1 + i, 301 + i, 65 + i]
        q = oracle.norm_rope(s["qkv"][:, :16], s["w"], *(x.double()[[n - 1 for n in lens], :64] for x in (s["cos"], s["sin"])), 1e-6)
        q = q.to(torch.bfloat16)
        for out, window, sinks, rounded in ((a, 0, 0, False), (b, 50, 2, True)):
            ref, mag = oracle.attend(q, s["k"], s["v"], table, [n - 1 for n in lens], 2, window, sinks, 128 ** -0.5)
            # the kernels' queries were rounded from f32 sums, these from f64: a query now and then differs by a step, its
            # scores (at most 4 at these norms) by 2^-8 of a channel's part: 1e-2 of the outputs' size in all
            assert float((out.double() - ref).abs().max()) < 1e-2 * float(ref.abs().max()), (i, window)


def test_captured_steps_replay_with_growing_lengths(pkg):
    """A step captured once and replayed: lengths, pages and slots are read on the device, so every replay is the next
    step. Eager steps of another batch and synchronizations go between the replays."""
    s, e, other = step_state(2), step_state(2), step_state(3)
    step(pkg, step_state(4), 400)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, b = step(pkg, s, 400)
    for i in range(6):
        g.replay()
        want = step(pkg, e, 400)
        step(pkg, other)
        torch.cuda.synchronize()
        assert s["lens"].tolist() == e["lens"].tolist() == [38 + i, 1 + i, 301 + i, 65 + i]
        assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and torch.equal(s["table"], e["table"])


def test_two_streams_at_once(pkg):
    """Two batches stepped on two streams at the same time, their split calls' workspaces apart: as one after the other."""
    def batch(seed):
        g = gen(seed)
        lens = [3000, 700]
        k, v, table = make_cache(g, lens, 64, 8, 128, torch.bfloat16)
        return torch.randn(2, 16, 128, generator=g, device=DEV).to(torch.bfloat16), k, v, ints(table), ints(lens)
    x, y = batch(1), batch(2)
    want = [pkg.paged_attention_decode(*z) for z in (x, y)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, z in enumerate((x, y)):
            with torch.cuda.stream(streams[i]):
                got[i].append(pkg.paged_attention_decode(*z))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_padded_batch_leaves_the_padding_alone(pkg):
    """A captured size larger than the batch: tokens past the last request get slot -1 and store nothing; idle requests
    (no new token, length 0 among them) attend what they hold."""
    s = step_state(5)
    k0, v0 = s["k"].clone(), s["v"].clone()
    p = pkg.paged_plan(ints([0, 2, 0, 0]), s["lens"], s["table"], s["free"], s["count"], 16, 4)
    assert p.slots.tolist()[2:] == [-1, -1] and p.kv_lens.tolist() == [37, 2, 300, 64] and p.cu_tokens.tolist() == [0, 0, 2, 2, 2]
    q = torch.full((4, 16, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    x = s["qkv"]
    out = pkg.qk_norm_rope_store(x[:, :16], x[:, 16:24], x[:, 24:], s["w"], s["w"], s["cos"], s["sin"], p.positions, p.slots, s["k"], s["v"], out=q)
    assert bool((out[2:] == 3.0).all())
    new = s["table"][1, 0].item()
    keep = [i for i in range(k0.shape[0]) if i != new]
    assert torch.equal(s["k"][keep].nan_to_num(9.0), k0[keep].nan_to_num(9.0)) and torch.equal(s["v"][keep].nan_to_num(9.0), v0[keep].nan_to_num(9.0))
    o = torch.full((4, 16, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    pkg.paged_attention_prefill(q, s["k"], s["v"], s["table"], p.kv_lens, p.cu_tokens, out=o)
    assert bool((o[2:] == 5.0).all()) and torch.isfinite(o).all() and not bool((o[:2] == 5.0).all())
