"""Paged key/value cache on the GPU against the restatement in 64 bits (kv_reference.py)."""
import pytest
import torch

from tests import kv_reference as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def device_copy(t, strided=False):
    """On the GPU with the same strides (a transposed pool stays one)."""
    if strided:
        return t.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    return t.contiguous().cuda()


def handles(s):
    from turbovec_b200.kvcache import KVBatch, PagedKVCache
    k, v = device_copy(s.k, s.tokens_first), device_copy(s.v, s.tokens_first)
    cache = PagedKVCache(k, v, s.bounds.cuda(), s.scales.cuda())
    batch = KVBatch(s.table.cuda(), torch.tensor(s.lens, dtype=torch.int32, device="cuda"), torch.tensor(s.offsets, dtype=torch.int32, device="cuda"))
    return cache, batch


def check_rows(s, out, lse, want):
    """Rows of sequences within their tolerances, the others untouched (they held 7)."""
    out, lse = out.cpu().double(), lse.cpu().double() if lse is not None else None
    for t in range(s.tokens):
        if t not in want:
            assert (out[t] == 7).all(), t
            continue
        for j, (o, l, tol, ltol) in enumerate(want[t]):
            bad = (out[t, j] - o).abs() - tol
            assert (bad <= 0).all(), (t, j, float(bad.max()), float(tol.max()))
            if lse is not None:
                assert lse[t, j] == l or abs(float(lse[t, j]) - l) <= ltol, (t, j, float(lse[t, j]), l, ltol)


def attend(s, **more):
    cache, batch = handles(s)
    out = torch.full((s.tokens, s.heads, s.dim), 7.0, dtype=s.dtype, device="cuda")
    lse = torch.full((s.tokens, s.heads), 7.0, device="cuda")
    pre = dict(prefix_pages=s.prefix_pages.cuda(), prefix_len=s.prefix) if s.prefix else {}
    assert cache.attend(batch, s.q.cuda(), out=out, lse=lse, **pre, **more) is out
    cache.check()
    return out, lse


ATTEND = [
    # dtype, dim, page, heads, kv_heads, new, lens, prefix, tokens_first, padding
    (BF, 128, 64, 4, 1, [1], [1], 0, False, 0),
    (BF, 128, 64, 8, 2, [1], [700], 0, False, 0),
    (FP, 64, 16, 6, 2, [1, 1, 1], [1, 65, 300], 0, True, 2),
    (BF, 64, 32, 3, 3, [1, 0, 2, 1], [5, 9, 2, 129], 0, False, 1),          # a sequence without rows, one that is all new
    (FP, 128, 128, 5, 1, [3, 4], [130, 400], 0, True, 0),                   # pages larger than a tile, rows over two row tiles
    (BF, 128, 16, 20, 1, [1, 2], [33, 90], 0, False, 0),                    # more heads to a key head than a row tile holds
    (FP, 64, 64, 2, 2, [1, 1], [0, 3], 0, False, 0),                        # a row that sees nothing
    (BF, 64, 64, 2, 2, [3, 1], [1, 70], 0, False, 0),                       # tokens before position 0
    (BF, 128, 64, 4, 2, [1], [10], 1, False, 0),
    (BF, 128, 64, 4, 2, [1, 1, 1], [10, 0, 64], 64, False, 3),
    (FP, 64, 16, 4, 4, [1, 2, 1, 1], [1, 17, 300, 64], 333, True, 0),
    (BF, 128, 32, 8, 2, [2, 1, 5], [40, 1, 90], 1000, True, 0),
    (FP, 128, 128, 14, 2, [1] * 11, list(range(1, 12)), 257, False, 0),
    (BF, 64, 64, 4, 1, [40], [50], 0, False, 0),                            # a piece of a prompt
    (BF, 128, 64, 8, 1, [1] * 4, [3] * 4, 128, False, 0),                   # a prefix on the tensor cores: one tile of keys
    (BF, 128, 64, 8, 2, [1] * 9, [5] * 9, 1111, False, 2),                  # 36 rows a key head
    (FP, 64, 16, 16, 2, [1] * 16, [2] * 16, 129, True, 0),                  # 128 rows; one key in the second tile
    (BF, 128, 128, 16, 2, [1] * 17, [2] * 17, 900, False, 0),               # 136: two row tiles
    (FP, 128, 32, 10, 1, [1, 3, 2] * 9, [4] * 27, 5000, True, 1),           # 540 rows, three pairs
    (BF, 64, 64, 24, 8, [2] * 50, [70] * 50, 2050, False, 0),               # 300 rows, eight key heads
    (BF, 128, 64, 24, 2, [1] * 3, [9] * 3, 192, False, 0),                  # half a tile of keys at the end
    (FP, 128, 32, 24, 2, [1] * 30, [9] * 30, 193, False, 0),
    (FP, 64, 128, 24, 1, [1] * 3, [9] * 3, 40_000, False, 0),               # several tiles to a block
]


@pytest.fixture
def prefix_kernel():
    """Sets which kernel reads prefixes, and puts the rule back."""
    from turbovec_b200 import kvcache
    yield lambda value: kvcache.set_option(kvcache.OPT_TENSOR_PREFIX, value)
    kvcache.set_option(kvcache.OPT_TENSOR_PREFIX, -1)


@pytest.mark.parametrize("tensor", [0, 1])
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attend(case, tensor, prefix_kernel):
    prefix_kernel(tensor)
    dtype, dim, page, heads, kv_heads, new, lens, prefix, first, padding = ATTEND[case]
    s = R.Setup(case, dtype=dtype, dim=dim, page=page, heads=heads, kv_heads=kv_heads, new=new, lens=lens, prefix=prefix, tokens_first=first,
                padding=padding, leading=1 if padding else 0)
    out, lse = attend(s)
    check_rows(s, out, lse, R.attend(s))


SELECTED = [
    # dtype, dim, page, heads, kv_heads, new, lens, budget, first, recent, padding
    (BF, 128, 64, 4, 1, [1], [1000], 4, 1, 1, 0),
    (FP, 64, 16, 6, 2, [1, 1, 1], [1, 300, 700], 5, 1, 2, 2),
    (BF, 64, 32, 20, 1, [2, 1], [300, 900], 6, 0, 0, 0),                    # 20 heads to a key head
    (FP, 128, 128, 4, 2, [1, 3], [129, 1500], 3, 0, 1, 0),
    (BF, 128, 16, 2, 2, [1], [500], 8, 4, 4, 0),                            # nothing left for the score
    (BF, 128, 16, 2, 2, [1, 1], [500, 0], 1, 0, 0, 0),                      # one page; a row that sees nothing
    (FP, 64, 16, 8, 4, [1], [4500], 40, 2, 3, 0),                           # more pages than threads of a block
]


def run_selected(s, budget, first, recent):
    cache, batch = handles(s)
    out = torch.full((s.tokens, s.heads, s.dim), 7.0, dtype=s.dtype, device="cuda")
    lse = torch.full((s.tokens, s.heads), 7.0, device="cuda")
    pages = torch.full((s.tokens, s.kv_heads, budget), 7, dtype=torch.int32, device="cuda")
    cache.attend_selected(batch, s.q.cuda(), budget=budget, first=first, recent=recent, out=out, lse=lse, pages=pages)
    cache.check()
    return out, lse, pages


def check_pages(s, pages, picks, budget):
    got = pages.cpu().tolist()
    for t in range(s.tokens):
        for h in range(s.kv_heads):
            want = picks[t][h] + [-1] * (budget - len(picks[t][h])) if t in picks else [7] * budget
            assert got[t][h] == want, (t, h)


@pytest.mark.parametrize("case", range(len(SELECTED)))
def test_attend_selected(case):
    dtype, dim, page, heads, kv_heads, new, lens, budget, first, recent, padding = SELECTED[case]
    s = R.Setup(100 + case, dtype=dtype, dim=dim, page=page, heads=heads, kv_heads=kv_heads, new=new, lens=lens, padding=padding)
    out, lse, pages = run_selected(s, budget, first, recent)
    want, picks = R.attend_selected(s, budget, first, recent)
    check_pages(s, pages, picks, budget)
    check_rows(s, out, lse, want)


def test_equal_scores_go_to_the_lower_page():
    s = R.Setup(7, dtype=BF, dim=64, page=16, heads=2, kv_heads=1, new=[1], lens=[16 * 300])
    s.bounds[:] = s.bounds[0]
    s.scales[:] = 1.0
    s.scales[s.table[0, 40:50].long()] = 2.0 if float(s.q.abs().max()) else 1.0
    out, lse, pages = run_selected(s, 20, 1, 1)
    _, picks = R.attend_selected(s, 20, 1, 1)
    check_pages(s, pages, picks, 20)


APPEND = [
    # dtype, dim, page, heads, kv_heads, new, lens, rotary, interleaved, offset, tokens_first, padding
    (BF, 128, 64, 4, 1, [1], [1], 128, False, 0, False, 0),
    (FP, 64, 16, 6, 2, [1, 1, 1], [16, 17, 300], 64, True, 11, True, 2),
    (BF, 128, 32, 4, 2, [70, 0, 1, 33], [100, 5, 32, 33], 64, True, 0, True, 0),
    (BF, 128, 128, 3, 3, [200, 129], [300, 129], 32, False, 1000, False, 3),
    (FP, 128, 16, 8, 8, [5, 1], [3, 1], 16, False, 0, False, 0),             # tokens before position 0
    (BF, 64, 64, 2, 2, [9], [64], 0, False, 0, False, 0),                    # no rotation
]


@pytest.mark.parametrize("case", range(len(APPEND)))
@pytest.mark.parametrize("in_place", [False, True])
def test_append(case, in_place):
    dtype, dim, page, heads, kv_heads, new, lens, rotary, interleaved, offset, first, padding = APPEND[case]
    s = R.Setup(200 + case, dtype=dtype, dim=dim, page=page, heads=heads, kv_heads=kv_heads, new=new, lens=lens, tokens_first=first, padding=padding,
                leading=1 if padding else 0)
    g = torch.Generator().manual_seed(case)
    angle = torch.rand(max(lens) + offset, rotary // 2, generator=g) * 6.28
    cos, sin = torch.cos(angle), torch.sin(angle)
    # earlier tokens of a page: its bounds are those of the keys before
    for b in range(len(lens)):
        at = lens[b] - new[b]
        if at > 0 and at % page and s.page_at(b, at // page) is not None:
            p = s.page_at(b, at // page)
            for h in range(kv_heads):
                both, step = R.bounds_of(s.k[p, h, :at % page])
                s.bounds[p, h], s.scales[p, h] = both.to(torch.int8), step
    cache, batch = handles(s)
    q = s.q.cuda()
    q_out = q if in_place else torch.full_like(q, 7.0)
    more = dict(cos=cos.cuda(), sin=sin.cuda()) if rotary else {}
    got = cache.append(batch, s.k_new.cuda(), s.v_new.cuda(), q=q, q_out=q_out, interleaved=interleaved, position_offset=offset, **more)
    assert got is q_out
    k, v, bounds, scales, got = cache.k.cpu(), cache.v.cpu(), cache.bounds.cpu(), cache.scales.cpu(), got.cpu()
    want_k, want_v = s.k.clone(), s.v.clone()
    touched, turned = set(), set()
    for t, b, p in s.rows():
        if p < 0:
            continue
        turned.add(t)
        c, sn = (cos[p + offset], sin[p + offset]) if rotary else (cos.new_zeros(0), sin.new_zeros(0))
        y, tol = R.rotate(s.q[t], c, sn, interleaved)
        assert ((got[t].double() - y).abs() <= tol).all(), t
        pg = s.page_at(b, p // page)
        y, tol = R.rotate(s.k_new[t], c, sn, interleaved)
        assert ((k[pg, :, p % page].double() - y).abs() <= tol).all(), t
        want_k[pg, :, p % page] = k[pg, :, p % page]
        want_v[pg, :, p % page] = s.v_new[t]
        touched.add((pg, b, p // page))
    for t in range(s.tokens):
        if t not in turned:
            assert torch.equal(got[t], s.q[t] if in_place else torch.full_like(s.q[t], 7.0))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)               # nothing else was written
    want_b, want_s = s.bounds.clone(), s.scales.clone()
    for pg, b, index in touched:
        n = min(page, lens[b] - index * page)
        for h in range(kv_heads):
            both, step = R.bounds_of(k[pg, h, :n])
            want_b[pg, h], want_s[pg, h] = both.to(torch.int8), step
    assert torch.equal(bounds, want_b) and torch.equal(scales, want_s)


# ---------------------------------------------------------------------------------------------- what the caller leaves lying about

def spoil(s, value):
    """Puts `value` into every place of the pool that holds no key of a sequence or of the prefix."""
    used = torch.zeros(s.pages, s.page, dtype=torch.bool)
    for b, n in enumerate(s.lens):
        for i in range(max(0, n)):
            p = s.page_at(b, i // s.page)
            if p is not None:
                used[p, i % s.page] = True
    for p, o in s.prefix_keys():
        used[p, o] = True
    gone = (~used)[:, None, :, None]
    for t in (s.k, s.v):
        t.copy_(torch.where(gone, torch.full_like(t, value), t))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("tensor", [0, 1])
@pytest.mark.parametrize("dim,page", [(128, 64), (64, 16), (64, 128)])
def test_places_behind_the_keys_may_hold_anything(value, tensor, dim, page, prefix_kernel):
    prefix_kernel(tensor)
    s = R.Setup(31, dtype=BF, dim=dim, page=page, heads=8, kv_heads=2, new=[1, 3, 1, 1], lens=[1, 70, 129, 0], prefix=201)
    spoil(s, value)
    out, lse = attend(s)
    check_rows(s, out, lse, R.attend(s))
    out, lse, pages = run_selected(s, 3, 1, 1)
    want, picks = R.attend_selected(s, 3, 1, 1)
    check_pages(s, pages, picks, 3)
    check_rows(s, out, lse, want)


@pytest.mark.parametrize("tensor", [0, 1])
def test_page_numbers_outside_the_pool_hold_no_keys(tensor, prefix_kernel):
    prefix_kernel(tensor)
    s = R.Setup(32, dtype=FP, dim=128, page=16, heads=4, kv_heads=2, new=[1, 2, 1], lens=[100, 300, 20], prefix=400)
    s.table[0, 2], s.table[1, 0], s.table[1, 17], s.table[2] = -7, s.pages, 2 ** 31 - 1, -1
    s.prefix_pages[3], s.prefix_pages[9], s.prefix_pages[24] = -2 ** 31, s.pages + 5, -1
    out, lse = attend(s)
    check_rows(s, out, lse, R.attend(s))
    for budget in (4, 30):                              # bad pages come last by score, and count as pages all the same
        out, lse, pages = run_selected(s, budget, 1, 2)
        want, picks = R.attend_selected(s, budget, 1, 2)
        check_pages(s, pages, picks, budget)
        check_rows(s, out, lse, want)
    before = s.k.clone(), s.v.clone(), s.bounds.clone(), s.scales.clone()
    cache, batch = handles(s)
    batch.table.fill_(-3)
    batch.table[1] = s.pages
    cache.append(batch, s.k_new.cuda(), s.v_new.cuda())
    for got, want in zip((cache.k, cache.v, cache.bounds, cache.scales), before):
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("tensor", [0, 1])
def test_lengths_that_the_table_does_not_cover(tensor, prefix_kernel):
    prefix_kernel(tensor)
    s = R.Setup(33, dtype=BF, dim=64, page=16, heads=4, kv_heads=1, new=[1, 1, 2], lens=[40, 33, 20], prefix=100)
    s.lens = [500, -3, 2 ** 31 - 1]                     # more than the table has pages for, and fewer than none
    out, lse = attend(s)
    check_rows(s, out, lse, R.attend(s))
    out, lse, pages = run_selected(s, 2, 1, 1)
    want, picks = R.attend_selected(s, 2, 1, 1)
    check_pages(s, pages, picks, 2)
    check_rows(s, out, lse, want)
    cache, batch = handles(s)
    before = cache.k.clone()
    cache.append(batch, s.k_new.cuda(), s.v_new.cuda())
    assert torch.equal(cache.k, before)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=123.0), torch.nan_to_num(b, nan=123.0)) and torch.equal(a.isnan(), b.isnan())


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_one_token_may_not_see_does_not_reach_it(value):
    """A draft's later tokens hold NaN or infinities: the earlier ones are as without them, the others are what the formula gives."""
    s = R.Setup(34, dtype=BF, dim=128, page=64, heads=4, kv_heads=1, new=[4], lens=[70])
    clean, clean_lse = attend(s)
    p = s.page_at(0, 1)
    s.v[p, 0, 68 - 64, 5] = value                       # the third token's value
    out, lse = attend(s)
    assert torch.equal(out[:2], clean[:2]) and torch.equal(lse, clean_lse)
    assert not torch.isfinite(out[2:, :, 5]).any() and torch.equal(out[2:, :, 6:], clean[2:, :, 6:])
    s = R.Setup(34, dtype=BF, dim=128, page=64, heads=4, kv_heads=1, new=[4], lens=[70])
    s.k[p, 0, 69 - 64] = float("nan")                   # the fourth token's key
    out, lse = attend(s)
    assert torch.equal(out[:3], clean[:3]) and torch.equal(lse[:3], clean_lse[:3])
    assert out[3].isnan().all() and lse[3].isnan().all()


@pytest.mark.parametrize("tensor", [0, 1])
def test_a_query_that_is_not_a_number_spoils_its_own_row(tensor, prefix_kernel):
    prefix_kernel(tensor)
    s = R.Setup(35, dtype=FP, dim=64, page=32, heads=6, kv_heads=2, new=[1] * 5, lens=[3] * 5, prefix=500)
    clean, clean_lse = attend(s)
    s.q[2, 4, 7] = float("nan")
    out, lse = attend(s)
    assert out[2, 4].isnan().all() and lse[2, 4].isnan()
    out[2, 4], lse[2, 4] = clean[2, 4], clean_lse[2, 4]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


def test_bounds_leave_nan_out_and_reach_every_power_of_two():
    from turbovec_b200.kvcache import KVBatch, PagedKVCache
    tops = [0.0, 1e-30, 127 * 2.0 ** -24, 127.5 * 2.0 ** -24, 2.0 ** -17, 0.99, 1.0, 127.0, 127.5, 128.0, 1e4, 127 * 2.0 ** 40, 1e15, 1e30, float("inf")]
    n, page, dim = len(tops), 16, 64
    cache = PagedKVCache.empty(n, page, 1, dim, dtype=BF, device="cuda")
    lens = torch.full((n,), 3, dtype=torch.int32, device="cuda")
    table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None]
    k = torch.zeros(3 * n, 1, dim, dtype=BF)
    for i, top in enumerate(tops):
        k[3 * i, 0] = torch.linspace(-1, 1, dim).double().mul(min(top, 3e38)).to(BF)
        k[3 * i + 1, 0, 3] = -top
    k[2::3, 0, 5] = float("nan")
    cache.append(KVBatch(table, lens, torch.arange(0, 3 * n + 1, 3, dtype=torch.int32, device="cuda")), k.cuda(), k.cuda())
    for i, top in enumerate(tops):
        rows = k[3 * i:3 * i + 3, 0].double()
        rows[2, 5] = rows[0, 5]
        rows[rows.isnan()] = 0.0                        # (0 times infinity does not occur: the ramp is finite)
        both, step = R.bounds_of(rows)
        assert float(cache.scales[i, 0]) == step, top
        assert torch.equal(cache.bounds[i, 0].cpu().double(), both), top


# ---------------------------------------------------------------------------------------------- views, sizes, streams, graphs

def test_views_of_larger_tensors():
    """A pool that is a layer of many, queries out of a fused projection, an output with room between its rows."""
    from turbovec_b200.kvcache import KVBatch, PagedKVCache
    s = R.Setup(41, dtype=BF, dim=64, page=32, heads=6, kv_heads=2, new=[2, 1, 3], lens=[2, 100, 64], prefix=90)
    pool = torch.full((s.pages, 3, 2, s.kv_heads, s.page, s.dim), 9.0, dtype=BF, device="cuda")
    k, v = pool[:, 1, 0], pool[:, 1, 1]
    k.copy_(s.k), v.copy_(s.v)
    cache = PagedKVCache(k, v, s.bounds.cuda(), s.scales.cuda())
    table = torch.full((len(s.lens), s.table.shape[1] + 5), 77, dtype=torch.int32, device="cuda")[:, 2:2 + s.table.shape[1]]
    table.copy_(s.table)
    batch = KVBatch(table, torch.tensor(s.lens, dtype=torch.int32, device="cuda"), torch.tensor(s.offsets, dtype=torch.int32, device="cuda"))
    fused = torch.full((s.tokens, s.heads + 2 * s.kv_heads, s.dim), 3.0, dtype=BF, device="cuda")
    q, kn, vn = fused[:, :s.heads], fused[:, s.heads:s.heads + s.kv_heads], fused[:, s.heads + s.kv_heads:]
    q.copy_(s.q), kn.copy_(s.k_new), vn.copy_(s.v_new)
    room = torch.full((s.tokens, s.heads, 2 * s.dim), 7.0, dtype=BF, device="cuda")
    out = room[:, :, 8:8 + s.dim]
    cache.attend(batch, q, prefix_pages=s.prefix_pages.cuda(), prefix_len=s.prefix, out=out)
    check_rows(s, out, None, R.attend(s))
    assert (room[:, :, :8] == 7).all() and (room[:, :, 8 + s.dim:] == 7).all()
    cache.append(batch, kn, vn)
    for t, b, p in s.rows():
        pg = s.page_at(b, p // s.page)
        assert torch.equal(k[pg, :, p % s.page].cpu(), s.k_new[t]) and torch.equal(v[pg, :, p % s.page].cpu(), s.v_new[t])
    assert (pool[:, 0] == 9).all() and (pool[:, 2] == 9).all()


@pytest.mark.parametrize("tensor", [0, 1])
def test_more_sequences_than_threads(tensor, prefix_kernel):
    prefix_kernel(tensor)
    g = torch.Generator().manual_seed(9)
    n = 700
    lens = torch.randint(0, 40, (n,), generator=g).tolist()
    new = [min(1, x) if i % 5 else 0 for i, x in enumerate(lens)]
    s = R.Setup(42, dtype=BF, dim=64, page=16, heads=2, kv_heads=1, new=new, lens=lens, prefix=33)
    out, lse = attend(s)
    check_rows(s, out, lse, R.attend(s))
    out, lse, pages = run_selected(s, 2, 0, 1)
    want, picks = R.attend_selected(s, 2, 0, 1)
    check_pages(s, pages, picks, 2)
    check_rows(s, out, lse, want)
    cache, batch = handles(s)
    cache.append(batch, s.k_new.cuda(), s.v_new.cuda())
    k = cache.k.cpu()
    for t, b, p in s.rows():
        assert torch.equal(k[s.page_at(b, p // s.page), :, p % s.page], s.k_new[t])


def test_more_heads_to_a_key_head_than_a_tile_of_rows(prefix_kernel):
    prefix_kernel(1)
    s = R.Setup(43, dtype=FP, dim=64, page=16, heads=150, kv_heads=1, new=[1, 1], lens=[20, 3], prefix=300)
    out, lse = attend(s)
    check_rows(s, out, lse, R.attend(s))
    out, lse, pages = run_selected(s, 1, 0, 0)
    want, picks = R.attend_selected(s, 1, 0, 0)
    check_pages(s, pages, picks, 1)
    check_rows(s, out, lse, want)


def test_offsets_beyond_32_bits():
    """A pool of 5 GB: the elements of its last pages lie beyond 2^31, their bytes beyond 2^32."""
    from turbovec_b200.kvcache import KVBatch, PagedKVCache
    s = R.Setup(44, dtype=BF, dim=128, page=64, heads=4, kv_heads=2, new=[1, 2], lens=[130, 200], prefix=70)
    pages = 5 * 2 ** 30 // (2 * 2 * 64 * 128)
    k = torch.empty(pages, 2, 64, 128, dtype=BF, device="cuda")
    v = torch.empty_like(k)
    bounds = torch.zeros(pages, 2, 2, 128, dtype=torch.int8, device="cuda")
    scales = torch.ones(pages, 2, device="cuda")
    shift = pages - s.pages
    k[shift:], v[shift:], bounds[shift:], scales[shift:] = s.k.cuda(), s.v.cuda(), s.bounds.cuda(), s.scales.cuda()
    cache = PagedKVCache(k, v, bounds, scales)
    batch = KVBatch(torch.where(s.table >= 0, s.table + shift, -1).to(torch.int32).cuda(), torch.tensor(s.lens, dtype=torch.int32, device="cuda"),
                    torch.tensor(s.offsets, dtype=torch.int32, device="cuda"))
    out = cache.attend(batch, s.q.cuda(), prefix_pages=(s.prefix_pages + shift).cuda(), prefix_len=s.prefix)
    check_rows(s, out, None, R.attend(s))
    out, pages_out = cache.attend_selected(batch, s.q.cuda(), budget=2, first=1, recent=0)
    want, picks = R.attend_selected(s, 2, 1, 0)
    check_pages(s, pages_out, picks, 2)
    check_rows(s, out, None, want)
    cache.append(batch, s.k_new.cuda(), s.v_new.cuda())
    for t, b, p in s.rows():
        assert torch.equal(k[s.page_at(b, p // s.page) + shift, :, p % s.page].cpu(), s.k_new[t])


def step(cache, batch, s, q, k, v, cos, sin, prefix):
    """One decode step as a model makes it: append, attention, attention over selected pages."""
    q = cache.append(batch, k, v, q=q, cos=cos, sin=sin, position_offset=s.prefix)
    out = cache.attend(batch, q, prefix_pages=prefix, prefix_len=s.prefix)
    selected, pages = cache.attend_selected(batch, q, budget=3, first=1, recent=1)
    return q, out, selected, pages


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("tensor", [0, 1])
def test_decoding_step_by_step(graph, tensor, prefix_kernel):
    """Several steps over growing sequences, lengths and inputs changed in place, eagerly or by one captured graph: every step is
    what the restatement gives for the cache as it then is, and a sequence that has ended keeps its pages."""
    prefix_kernel(tensor)
    s = R.Setup(51, dtype=BF, dim=64, page=16, heads=12, kv_heads=2, new=[1] * 4, lens=[14, 1, 47, 90], prefix=77, spare=6)
    s.table = torch.cat([s.table, torch.full((4, 1), -1, dtype=torch.int32)], 1)
    free = sorted(set(range(s.pages)) - set(s.table.flatten().tolist()) - set(s.prefix_pages.tolist()))
    for b, n in enumerate(s.lens):                      # a page more for each
        s.table[b, -(-n // s.page)] = free.pop()
    angle = torch.rand(300, 32) * 6.28
    cos, sin = torch.cos(angle).cuda(), torch.sin(angle).cuda()
    cache, batch = handles(s)
    # the last page of a sequence holds fewer keys than the setup's bounds know of: bounds of what is there
    for b, n in enumerate(s.lens):
        at = n - 1
        p = s.page_at(b, at // s.page)
        for h in range(s.kv_heads):
            if at % s.page:
                both, sc = R.bounds_of(s.k[p, h, :at % s.page])
                cache.bounds[p, h], cache.scales[p, h] = both.to(torch.int8).cuda(), sc
    q, k, v = s.q.cuda(), s.k_new.cuda(), s.v_new.cuda()
    prefix = s.prefix_pages.cuda()
    captured = None
    g = torch.Generator().manual_seed(5)
    for turn in range(5):
        if turn:
            s.lens = [n + 1 for n in s.lens]
            batch.lens.add_(1)
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g).to(BF))
        if not graph:
            got = step(cache, batch, s, q, k, v, cos, sin, prefix)
        else:
            if captured is None:
                keep = [t.clone() for t in (cache.k, cache.v, cache.bounds, cache.scales)]
                side = torch.cuda.Stream()
                with torch.cuda.stream(side):
                    step(cache, batch, s, q, k, v, cos, sin, prefix)      # first calls set kernels up
                side.synchronize()
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured):
                    got = step(cache, batch, s, q, k, v, cos, sin, prefix)
                for t, old in zip((cache.k, cache.v, cache.bounds, cache.scales), keep):
                    t.copy_(old)
            captured.replay()
        cache.check()
        rq, out, selected, pages = (t.cpu() for t in got)
        s.k, s.v, s.bounds, s.scales = cache.k.cpu(), cache.v.cpu(), cache.bounds.cpu(), cache.scales.cpu()
        s.q = rq
        for t, b, p in s.rows():
            pg = s.page_at(b, p // s.page)
            y, tol = R.rotate(k[t].cpu(), cos[p + s.prefix].cpu(), sin[p + s.prefix].cpu(), False)
            assert ((s.k[pg, :, p % s.page].double() - y).abs() <= tol).all()
            y, tol = R.rotate(q[t].cpu(), cos[p + s.prefix].cpu(), sin[p + s.prefix].cpu(), False)
            assert ((rq[t].double() - y).abs() <= tol).all()
            for h in range(s.kv_heads):
                both, sc = R.bounds_of(s.k[pg, h, :p % s.page + 1])
                assert torch.equal(s.bounds[pg, h].double(), both) and float(s.scales[pg, h]) == sc
        check_rows(s, out, None, R.attend(s))
        want, picks = R.attend_selected(s, 3, 1, 1)
        check_pages(s, pages, picks, 3)
        check_rows(s, selected, None, want)


def test_two_graphs_and_two_streams_do_not_share_workspaces():
    """Graphs of different caches, replayed at the same time on two streams, and eager calls on both, give what each gives alone."""
    work = []
    for seed, prefix in ((61, 3000), (62, 0)):
        s = R.Setup(seed, dtype=BF, dim=128, page=64, heads=16, kv_heads=2, new=[1] * 20, lens=list(range(100, 2100, 100)), prefix=prefix)
        cache, batch = handles(s)
        q, pre = s.q.cuda(), s.prefix_pages.cuda()

        def run(cache=cache, batch=batch, q=q, pre=pre, prefix=prefix):
            out = cache.attend(batch, q, prefix_pages=pre if prefix else None, prefix_len=prefix)
            return out, cache.attend_selected(batch, q, budget=8, first=1, recent=2)[0]
        alone = [t.clone() for t in run()]
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = run()
        work.append((run, alone, graph, got, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for run, alone, graph, got, stream in work:
            for t in got:
                t.zero_()
        torch.cuda.synchronize()
        for run, alone, graph, got, stream in work:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for run, alone, graph, got, stream in work:
            assert all(torch.equal(a, b) for a, b in zip(alone, got))
        eager = []
        for run, alone, graph, got, stream in work:
            with torch.cuda.stream(stream):
                eager.append(run())
        torch.cuda.synchronize()
        for (run, alone, graph, got, stream), now in zip(work, eager):
            assert all(torch.equal(a, b) for a, b in zip(alone, now))


def test_a_graph_whose_first_node_is_a_copy():
    s = R.Setup(63, dtype=FP, dim=64, page=16, heads=4, kv_heads=2, new=[1] * 3, lens=[30, 9, 64], prefix=50)
    cache, batch = handles(s)
    q, pre, source = torch.zeros_like(s.q, device="cuda"), s.prefix_pages.cuda(), s.q.cuda()
    out = cache.attend(batch, source, prefix_pages=pre, prefix_len=50)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        q.copy_(source)                                  # contiguous, same type: a memory copy
        got = cache.attend(batch, q, prefix_pages=pre, prefix_len=50)
        twice = got * 2
    q.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, out) and torch.equal(twice, out * 2)


def test_refusals_with_tensors_in_hand():
    from turbovec_b200.kvcache import KVBatch, PagedKVCache
    s = R.Setup(71, dtype=BF, dim=64, page=16, heads=4, kv_heads=2, new=[1, 1], lens=[5, 40], prefix=20)
    cache, batch = handles(s)
    q, pre = s.q.cuda(), s.prefix_pages.cuda()
    kn, vn = s.k_new.cuda(), s.v_new.cuda()
    cos = torch.ones(100, 32, device="cuda")
    value, kind = (ValueError,), (TypeError,)
    for error, call in [
            (value, lambda: cache.attend(batch, q.cpu())), (kind, lambda: cache.attend(batch, q.float())), (kind, lambda: cache.attend(batch, q.half())),
            (value, lambda: cache.attend(batch, q[:, :3])), (value, lambda: cache.attend(batch, q[..., :32])), (value, lambda: cache.attend(batch, q[0])),
            (value, lambda: cache.attend(batch, q, out=q)), (value, lambda: cache.attend(batch, q, out=q[:1])), (kind, lambda: cache.attend(None, q)),
            (value, lambda: cache.attend(batch, q.transpose(1, 2).contiguous().transpose(1, 2))),
            (value, lambda: cache.attend(batch, q, prefix_len=5)), (value, lambda: cache.attend(batch, q, prefix_pages=pre, prefix_len=33)),
            (value, lambda: cache.attend(batch, q, prefix_pages=pre, prefix_len=-1)), (kind, lambda: cache.attend(batch, q, prefix_pages=pre.long(), prefix_len=5)),
            (value, lambda: cache.attend(batch, q, scale=0.0)), (value, lambda: cache.attend(batch, q, scale=float("nan"))),
            (value, lambda: cache.attend(batch, q, lse=torch.zeros(2, 3, device="cuda"))), (kind, lambda: cache.attend(batch, q, lse=q[..., 0])),
            (value, lambda: cache.attend_selected(batch, q, budget=0)), (value, lambda: cache.attend_selected(batch, q, budget=2, first=2, recent=1)),
            (value, lambda: cache.attend_selected(batch, q, budget=2, first=-1)),
            (value, lambda: cache.attend_selected(batch, q, budget=2, pages=torch.zeros(2, 2, 3, dtype=torch.int32, device="cuda"))),
            (value, lambda: PagedKVCache(cache.k, cache.v).attend_selected(batch, q, budget=2)),
            (value, lambda: cache.append(batch, kn, vn[:1])), (value, lambda: cache.append(batch, kn[:, :1], vn)), (kind, lambda: cache.append(batch, kn.float(), vn)),
            (value, lambda: cache.append(batch, kn, vn, q_out=q)), (value, lambda: cache.append(batch, kn, vn, cos=cos)),
            (value, lambda: cache.append(batch, kn, vn, cos=cos, sin=cos[:50])), (kind, lambda: cache.append(batch, kn, vn, cos=cos.double(), sin=cos.double())),
            (value, lambda: cache.append(batch, kn, vn, cos=cos[:, :5].contiguous(), sin=cos[:, :5].contiguous())),
            (value, lambda: cache.append(batch, kn, vn, cos=torch.ones(9, 40, device="cuda"), sin=torch.ones(9, 40, device="cuda"))),
            (value, lambda: KVBatch(batch.table, batch.lens, batch.offsets.cpu())), (value, lambda: PagedKVCache(cache.k, cache.v.cpu())),
            (value, lambda: cache.attend(KVBatch(s.table, torch.tensor(s.lens, dtype=torch.int32)), q)),
            (value, lambda: PagedKVCache(cache.k[..., :64], cache.v.flatten()[1:1 + 64 * 16].view(1, 1, 16, 64).expand(cache.k.shape)))]:
        with pytest.raises(error):
            call()
    assert cache.attend(batch, q[:0]).shape == (0, 4, 64)                  # no rows: nothing to do
    empty = KVBatch(batch.table[:0], batch.lens[:0])
    kept = torch.full_like(q, 3.0)
    assert (cache.attend(empty, q, out=kept) == 3).all()                    # no sequences: every row is behind the last one


def test_the_current_device_and_errors_stay_as_they_were():
    s = R.Setup(72, dtype=BF, dim=64, page=16, heads=2, kv_heads=1, new=[1], lens=[5])
    out, lse = attend(s)
    assert torch.cuda.current_device() == 0
    from turbovec_b200 import kvcache
    with pytest.raises(ValueError):
        kvcache.set_option(99, 1)
    with pytest.raises(ValueError):
        kvcache.set_option(kvcache.OPT_TENSOR_PREFIX, 2)


def test_equal_calls_give_equal_bits():
    s = R.Setup(73, dtype=BF, dim=128, page=64, heads=16, kv_heads=2, new=[1] * 24, lens=[37 * (i + 1) for i in range(24)], prefix=4000)
    first, first_lse = attend(s)
    for _ in range(3):
        out, lse = attend(s)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)


@pytest.mark.parametrize("tensor", [0, 1])
@pytest.mark.parametrize("offsets", [[2, 6, 3, 9], [9, 5, 4, 2], [-4, 100, 1, 2 ** 31 - 1], [-2 ** 31, 8, -1, 8]])
def test_offsets_that_do_not_ascend_stay_within_the_call(offsets, tensor, prefix_kernel):
    """Such rows have no meaning, but the calls end, and write to their own rows and to pages of the table alone."""
    prefix_kernel(tensor)
    s = R.Setup(35, dtype=BF, dim=128, page=16, heads=4, kv_heads=2, new=[4, 3, 2], lens=[100, 300, 20], prefix=400)
    cache, batch = handles(s)
    batch.offsets.copy_(torch.tensor(offsets, dtype=torch.int32))
    heads, rows = s.heads, s.tokens
    around = torch.full((rows + 16, heads, s.dim), 7.0, dtype=s.dtype, device="cuda")
    out, lse_around = around[8:8 + rows], torch.full((rows + 16, heads), 7.0, device="cuda")
    q = s.q.cuda()
    cache.attend(batch, q, out=out, lse=lse_around[8:8 + rows], prefix_pages=s.prefix_pages.cuda(), prefix_len=s.prefix)
    cache.attend_selected(batch, q, budget=3, out=out, lse=lse_around[8:8 + rows])
    used = set(s.table.flatten().tolist())
    unused = torch.tensor([p for p in range(s.pages) if p not in used], device="cuda")
    before = cache.k[unused].clone(), cache.v[unused].clone(), cache.bounds[unused].clone(), cache.scales[unused].clone()
    cache.append(batch, s.k_new.cuda(), s.v_new.cuda(), q=q, q_out=out)
    cache.check()
    assert unused.numel() > 0 and (around[:8] == 7).all() and (around[8 + rows:] == 7).all()
    assert (lse_around[:8] == 7).all() and (lse_around[8 + rows:] == 7).all()
    for got, want in zip((cache.k, cache.v, cache.bounds, cache.scales), before):
        assert torch.equal(got[unused], want)
