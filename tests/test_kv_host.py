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
