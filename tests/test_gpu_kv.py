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
