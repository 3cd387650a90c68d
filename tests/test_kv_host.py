"""Paged key/value cache: refusals of the C entry points and of the Python classes, which need no device, and the operators'
restatement against independent arithmetic."""
import ctypes as C
import math

import pytest
import torch

from tests import kv_reference as R


@pytest.fixture(scope="module")
def lib():
    from turbovec_b200 import _native, build
    build.build()
    return _native.load()


def views(**change):
    """A valid cache, batch and rows over host memory: every call below is refused before a device is touched."""
    from turbovec_b200 import _native as N
    buf = (C.c_char * 65536)()
    at = (C.addressof(buf) + 255) & ~255
    cache = dict(device=0, dtype=0, head_dim=128, kv_heads=2, page_size=16, pages=4, k=at, v=at, k_page_stride=4096, k_head_stride=2048, k_token_stride=128,
                 v_page_stride=4096, v_head_stride=2048, v_token_stride=128, bounds=at, scales=at)
    batch = dict(sequences=1, table_width=2, table_stride=2, table=at, lens=at, offsets=at)
    rows = dict(data=at, token_stride=512, head_stride=128)
    for d in (cache, batch, rows):
        d.update({k: v for k, v in change.items() if k in d})
    return buf, at, N.KvCacheView(**cache), N.KvBatchView(**batch), N.KvRowsView(**rows)


BAD = [dict(dtype=2), dict(head_dim=96), dict(page_size=24), dict(kv_heads=0), dict(pages=0), dict(pages=1 << 31), dict(k=None), dict(v=8),
       dict(k_page_stride=-4096), dict(v_head_stride=0), dict(k_token_stride=132), dict(scales=None), dict(bounds=None), dict(bounds=48),
       dict(sequences=-1), dict(table_width=3), dict(table_width=1 << 40, table_stride=1 << 40), dict(lens=None), dict(table=None), dict(offsets=None),
       dict(tokens=-1), dict(tokens=1 << 31), dict(heads=3), dict(heads=0), dict(data=None), dict(data=8), dict(head_stride=4), dict(token_stride=0)]


def call(lib, op, **change):
    buf, at, cache, batch, rows = views(**change)
    tokens, heads = change.get("tokens", 1), change.get("heads", 4)
    out = type(rows)(at + change.get("out_at", 16384), 512, 128)
    if op == "append":
        a = dict(k_new=rows, v_new=rows, q=rows, q_out=out, cos=at, sin=at, positions=8, rotary=64, offset=0)
        a.update({k: v for k, v in change.items() if k in a})
        return lib.tv_kv_append(cache, batch, tokens, heads, a["k_new"], a["v_new"], a["q"], a["q_out"], a["cos"], a["sin"], a["positions"], a["rotary"], 0,
                                a["offset"], None)
    a = dict(q=rows, out=out, prefix_pages=at, prefix_width=2, prefix_len=20, scale=0.1, ws=at, ws_bytes=1 << 40, budget=2, first=1, recent=1, pages_out=at)
    a.update({k: v for k, v in change.items() if k in a})
    if op == "attend":
        return lib.tv_kv_attend(cache, batch, tokens, heads, a["q"], a["prefix_pages"], a["prefix_width"], a["prefix_len"], a["scale"], a["out"], None,
                                a["ws"], a["ws_bytes"], None)
    return lib.tv_kv_attend_selected(cache, batch, tokens, heads, a["q"], a["budget"], a["first"], a["recent"], a["scale"], a["out"], None,
                                     a["pages_out"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("change", BAD, ids=lambda c: ",".join(f"{k}={v}" for k, v in c.items()))
@pytest.mark.parametrize("op", ["append", "attend", "selected"])
def test_bad_arguments_are_refused(lib, op, change):
    assert call(lib, op, **change) in (90, 93)
    assert lib.tv_last_error(None)


def test_arguments_of_one_operator(lib):
    assert call(lib, "append", rotary=24) == 90 and call(lib, "append", rotary=144) == 90
    assert call(lib, "append", cos=None) == 90 and call(lib, "append", sin=8) == 90
    assert call(lib, "append", q=None) == 90 and b"together" in lib.tv_last_error(None)
    assert call(lib, "append", offset=1 << 50) == 90
    for change in (dict(prefix_len=33), dict(prefix_len=-1), dict(prefix_width=-1), dict(prefix_pages=None), dict(scale=0.0), dict(scale=-1.0),
                   dict(scale=math.inf), dict(scale=math.nan)):
        assert call(lib, "attend", **change) == 90, change
    for change in (dict(budget=0), dict(budget=1 << 20), dict(first=-1), dict(first=2), dict(recent=3), dict(pages_out=None), dict(scale=math.nan)):
        assert call(lib, "selected", **change) == 90, change
    assert call(lib, "selected", bounds=None, scales=None) == 90
    assert call(lib, "selected", table_width=50_000, table_stride=50_000) == 93
    for op in ("append", "attend", "selected"):
        assert call(lib, op, out_at=256) == 90 and b"overlap" in lib.tv_last_error(None)


def test_empty_calls_do_nothing(lib):
    for op in ("append", "attend", "selected"):
        assert call(lib, op, tokens=0) == 0
        assert call(lib, op, sequences=0, lens=None, offsets=None, table=None) == 0


def test_no_device_is_an_error_and_not_a_fallback(lib):
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    for op in ("append", "attend", "selected"):
        assert call(lib, op) in (91, 92) and lib.tv_last_error(None)
    assert lib.tv_kv_status(0) == 91
    from turbovec_b200.kvcache import PagedKVCache
    with pytest.raises(RuntimeError, match="no CPU path"):
        PagedKVCache.empty(2, 16, 1, 64, device="cpu")


def test_python_argument_errors():
    from turbovec_b200.kvcache import KVBatch, PagedKVCache
    table, lens, offsets = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.arange(3, dtype=torch.int32)
    assert len(KVBatch(table, lens, offsets)) == 2 and KVBatch(table, lens).offsets.tolist() == [0, 1, 2]
    for bad in ((table.long(), lens, offsets), (table, lens.long(), offsets), (table, lens, offsets.long()), (table, [0, 0], offsets)):
        with pytest.raises(TypeError):
            KVBatch(*bad)
    for bad in ((table[:1], lens, offsets), (table, lens, offsets[:2]), (table.T, lens[:1].expand(3), None), (table[:, ::2], lens, offsets),
                (table[0], lens, offsets), (table[:1].expand(2, 3), lens, offsets)):
        with pytest.raises(ValueError):
            KVBatch(*bad)
    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    b, s = torch.zeros(2, 1, 2, 64, dtype=torch.int8), torch.zeros(2, 1)
    for bad in ((k.float(), k), (k, k.half()), ([k], k), (k, k, b.float(), s), (k, k, b, s.half())):
        with pytest.raises(TypeError):
            PagedKVCache(*bad)
    for bad in ((k, k[:1]), (k[..., :32], k[..., :32]), (k[:, :, :8], k[:, :, :8]), (k[0], k[0]), (k, k, b), (k, k, b[:1], s), (k, k, b, s[:1]),
                (k[..., ::2], k[..., ::2])):
        with pytest.raises(ValueError):
            PagedKVCache(*bad)


@pytest.mark.parametrize("seed", range(4))
def test_bounds_do_not_depend_on_how_keys_arrive(seed):
    """ceil(ceil(x / a) / b) = ceil(x / (a b)) for powers of two: widening 8-bit bounds gives the bounds of all keys."""
    g = torch.Generator().manual_seed(seed)
    keys = (torch.randn(20, 32, generator=g) * torch.exp(2 * torch.randn(20, 1, generator=g))).bfloat16()
    both, step = R.bounds_of(keys[:1])
    for i in range(1, 20):
        new, s = R.bounds_of(keys[i:i + 1])
        wide = max(step, s)
        old = both * (step / wide)
        lo, hi = torch.floor(keys[i].double() / wide), torch.ceil(keys[i].double() / wide)
        both, step = torch.stack([torch.minimum(torch.floor(old[0]), lo), torch.maximum(torch.ceil(old[1]), hi)]), wide
    want, s = R.bounds_of(keys)
    assert s == step and torch.equal(both, want)


def test_workspace_sizes_that_cannot_be_are_refused_with_a_message(lib):
    _, _, cache, batch, _ = views()
    assert call(lib, "attend", scale=-1.0) == 90                        # a message that must not be met again below
    for prefix_len in (-1, (1 << 30) + 1, 1 << 32, 1 << 62):
        assert lib.tv_kv_attend_workspace(cache, batch, 1, 4, prefix_len) == 0
        assert b"prefix_len" in lib.tv_last_error(None), prefix_len
    for budget in (0, -1, 40_000, 1 << 40):
        assert lib.tv_kv_attend_selected_workspace(cache, batch, 1, 4, budget) == 0
        assert b"budget" in lib.tv_last_error(None), budget
    cache.device = 63                                                   # no machine has so many
    for size in (lib.tv_kv_attend_workspace(cache, batch, 1, 4, 20), lib.tv_kv_attend_selected_workspace(cache, batch, 1, 4, 2)):
        assert size == 0
        assert b"no such CUDA device" in lib.tv_last_error(None)


def test_the_restatement_of_one_sequence_is_that_of_many():
    for prefix, lens, padding in ((0, 40, 0), (70, 23, 2), (33, 7, 0)):
        s = R.Setup(81, dtype=torch.bfloat16, dim=64, page=16, heads=6, kv_heads=2, new=[7], lens=[lens], prefix=prefix, padding=padding, leading=1)
        out, lse, tol, ltol = R.attend_sequence(s)
        want = R.attend(s)
        for i, (t, _, _) in enumerate(s.rows()):
            for j, (o, l, to, tl) in enumerate(want[t]):
                assert torch.allclose(out[i, j], o, rtol=1e-12, atol=1e-12) and abs(float(lse[i, j]) - l) < 1e-12
                assert torch.allclose(tol[i, j], to, rtol=1e-9) and abs(float(ltol[i, j]) - tl) < 1e-12


def test_addresses_that_no_kernel_could_read_are_refused(lib):
    """32-bit numbers at an odd address would be an error on the device."""
    buf, at, cache, batch, rows = views()
    for op in ("append", "attend", "selected"):
        for change in (dict(table=at + 2), dict(lens=at + 1), dict(offsets=at + 3)):
            assert call(lib, op, **change) == 90, (op, change)
            assert b"4-byte aligned" in lib.tv_last_error(None)
    out = type(rows)(at + 16384, 512, 128)
    assert call(lib, "attend", prefix_pages=at + 2) == 90 and b"4-byte aligned" in lib.tv_last_error(None)
    assert call(lib, "selected", pages_out=at + 1) == 90 and b"4-byte aligned" in lib.tv_last_error(None)
    for lse in (at + 1, at + 2):
        assert lib.tv_kv_attend(cache, batch, 1, 4, rows, at, 2, 20, 0.1, out, lse, at, 1 << 40, None) == 90
        assert b"4-byte aligned" in lib.tv_last_error(None)
        assert lib.tv_kv_attend_selected(cache, batch, 1, 4, rows, 2, 1, 1, 0.1, out, lse, at, at, 1 << 40, None) == 90
        assert b"4-byte aligned" in lib.tv_last_error(None)


def chunks(at, tokens, heads, token_stride, head_stride, dim):
    """16-byte pieces of a view (strides in elements of two bytes)."""
    return {(at + 2 * (t * token_stride + h * head_stride)) // 16 + i for t in range(tokens) for h in range(heads) for i in range(dim // 8)}


def refused_for_overlap(lib, rc):
    assert rc != 0
    return rc == 90 and b"overlap" in lib.tv_last_error(None)


@pytest.mark.parametrize("seed", range(3))
def test_views_of_one_buffer_that_interleave_are_told_from_those_that_overlap(lib, seed):
    """q and out, or k and the rotated queries, as heads of one buffer, in rows of tokens or of heads: refused where they share a byte."""
    import random
    rng = random.Random(seed)
    dim, seen = 64, {True: 0, False: 0}
    buf, at, cache, batch, row = views(device=63, head_dim=dim, k_head_stride=1024, k_token_stride=64, v_head_stride=1024, v_token_stride=64)     # no machine has so many devices
    Row = type(row)
    for _ in range(600):
        tokens, heads = rng.choice([1, 2, 3, 5]), 4
        by_heads = rng.random() < 0.3
        outer = 8 * rng.choice([32, 40, 64, 96, 97])

        def view(n):
            rows, runs = (n, tokens) if by_heads else (tokens, n)
            inner = 8 * rng.choice([8, 8, 9, 12, 16])
            if (runs - 1) * inner + dim > outer:
                inner = 64
            if (runs - 1) * inner + dim > outer:
                return None
            where = at + 16 * rng.choice([0, rng.randrange(0, 8 * tokens), rng.randrange(0, 200), 8 * rng.randrange(0, 30)])
            ts, hs = (inner, outer) if by_heads else (outer, inner)
            return Row(where, ts, hs), chunks(where, tokens, n, ts, hs, dim)
        a, b, k = view(heads), view(heads), view(2)
        if not a or not b or not k:
            continue
        rc = lib.tv_kv_attend(cache, batch, tokens, heads, a[0], at, 2, 20, 0.1, b[0], None, at, 1 << 40, None)
        assert refused_for_overlap(lib, rc) == bool(a[1] & b[1])
        seen[bool(a[1] & b[1])] += 1
        same = (a[0].data, a[0].token_stride, a[0].head_stride)
        for first, second in ((a, a), (a, b)):
            rc = lib.tv_kv_append(cache, batch, tokens, heads, k[0], k[0], first[0], second[0], at, at, 8, 64, 0, 0, None)
            apart = (second[0].data, second[0].token_stride, second[0].head_stride) == same or not first[1] & second[1]
            assert refused_for_overlap(lib, rc) == (not apart or bool(k[1] & second[1]))
    assert min(seen.values()) > 50


@pytest.mark.parametrize("seed", range(2))
def test_views_that_share_bytes_are_never_let_through(lib, seed):
    """Any strides: what overlaps is refused, and what lies in ranges of its own is not."""
    import random
    rng = random.Random(10 + seed)
    dim = 64
    buf, at, cache, batch, row = views(device=63, head_dim=dim, k_head_stride=1024, k_token_stride=64, v_head_stride=1024, v_token_stride=64)
    hit = 0
    for _ in range(600):
        tokens, heads = rng.choice([1, 2, 3, 7]), rng.choice([2, 4])
        a, b = ((at + 16 * rng.randrange(0, 300), 8 * rng.randrange(1, 120), 8 * rng.randrange(1, 120)) for _ in range(2))
        ca, cb = chunks(a[0], tokens, heads, *a[1:], dim), chunks(b[0], tokens, heads, *b[1:], dim)
        rc = lib.tv_kv_attend(cache, batch, tokens, heads, type(row)(*a), at, 2, 20, 0.1, type(row)(*b), None, at, 1 << 40, None)
        refused = refused_for_overlap(lib, rc)
        hit += bool(ca & cb)
        assert refused if ca & cb else not (refused and (max(ca) < min(cb) or max(cb) < min(ca)))
    assert hit > 100
    # sums are contiguous
    q, out = type(row)(at, 512, 128), type(row)(at + 16384, 512, 128)
    for lse in (at, at + 64, at + 16384 + 1020):
        assert refused_for_overlap(lib, lib.tv_kv_attend(cache, batch, 2, 4, q, at, 2, 20, 0.1, out, lse, at, 1 << 40, None))
    # strides that no memory has do not wrap
    far = type(row)(at, (1 << 38) - 8, 128)
    assert lib.tv_kv_attend(cache, batch, 1 << 29, 4, far, at, 2, 20, 0.1, type(row)(at + 4096, 512, 128), None, at, 1 << 40, None) == 90


def host_cache(monkeypatch, lib, **change):
    """The Python class over host memory: its calls reach the C entries, which refuse them."""
    from turbovec_b200 import kvcache
    buf, at, view, batch_view, _ = views(head_dim=64, k_head_stride=1024, k_token_stride=64, v_head_stride=1024, v_token_stride=64, **change)
    cache = object.__new__(kvcache.PagedKVCache)
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    bounds, scales = torch.zeros(4, 2, 2, 64, dtype=torch.int8), torch.zeros(4, 2)
    for name, x in dict(k=k, v=k.clone(), bounds=bounds, scales=scales).items():
        object.__setattr__(cache, "_" + name if hasattr(kvcache.PagedKVCache, name) else name, x)
    cache._lib, cache._view, cache._buf = lib, view, buf
    cache.device, cache.dtype, cache.pages, cache.kv_heads, cache.page_size, cache.head_dim = torch.device("cpu"), torch.bfloat16, 4, 2, 16, 64
    cache._index, cache._scale, cache._sizes = -1, 0.125, {}
    monkeypatch.setattr(kvcache, "_stream", lambda index: 0)
    batch = kvcache.KVBatch(torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    return cache, batch, torch.zeros(1, 4, 64, dtype=torch.bfloat16)


def test_a_device_that_fails_is_no_wrong_argument(monkeypatch, lib):
    """Also where the size of a workspace is asked for first; sizes that are refused stay wrong arguments."""
    cache, batch, q = host_cache(monkeypatch, lib, device=63)
    kv = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: cache.attend(batch, q), lambda: cache.attend_selected(batch, q, budget=2), lambda: cache.append(batch, kv, kv)):
        with pytest.raises(RuntimeError, match="no such CUDA device"):
            call()
    for call in (lambda: cache.attend(batch, q, scale=-1.0), lambda: cache.attend_selected(batch, q, budget=40_000)):
        with pytest.raises(ValueError):
            call()


def test_tensors_that_calls_use_are_changed_in_place_and_not_replaced(monkeypatch, lib):
    """A call reads the tensors that a batch or a cache was made of: another one in their place would be passed over in silence."""
    cache, batch, _ = host_cache(monkeypatch, lib)
    address = batch.lens.data_ptr()
    batch.lens += 1
    batch.table[0, 1] = 3
    assert batch.lens.tolist() == [2] and batch.table.tolist() == [[0, 3]] and batch.lens.data_ptr() == address == batch._view.lens
    for name in ("table", "lens", "offsets"):
        with pytest.raises(AttributeError, match="in place"):
            setattr(batch, name, getattr(batch, name).clone())
    for name in ("k", "v", "bounds", "scales"):
        t = getattr(cache, name)
        setattr(cache, name, t)
        with pytest.raises(AttributeError, match="in place"):
            setattr(cache, name, t.clone())
        assert getattr(cache, name) is t


def test_position_offsets_beyond_64_bits_do_not_wrap(monkeypatch, lib):
    cache, batch, _ = host_cache(monkeypatch, lib, device=63)
    kv = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    cos = torch.zeros(4, 32)
    for offset in (1 << 41, 1 << 64, -(1 << 64), (1 << 65) + 3):
        with pytest.raises(ValueError, match="position_offset"):
            cache.append(batch, kv, kv, cos=cos, sin=cos, position_offset=offset)
    with pytest.raises(RuntimeError, match="no such CUDA device"):
        cache.append(batch, kv, kv, cos=cos, sin=cos, position_offset=1 << 40)
