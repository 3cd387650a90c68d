"""Attention over a prefix by the tensor-memory kernel where its blocks have several parts (runs of keys that go from one key head to the
next), against the restatement in 64 bits."""
import pytest
import torch

from tests import kv_reference as R
from tests.test_gpu_kv import attend, prefix_kernel  # noqa: F401  (a fixture)

BF, FP = torch.bfloat16, torch.float16
MULTIPROCESSORS = 148


def check(s, out, lse, **steps):
    want, want_lse, tol, ltol = R.attend_sequence(s, **steps)
    at = [t for t, _, _ in s.rows()]
    bad = (out.cpu().double()[at] - want).abs() - tol
    assert (bad <= 0).all(), (int((bad > 0).sum()), float(bad.max()))
    assert ((lse.cpu().double()[at] - want_lse).abs() <= ltol).all()
    rest = [t for t in range(s.tokens) if t not in set(at)]
    assert (out[rest] == 7).all() and (lse[rest] == 7).all()


ONE_TILE = [
    # dtype, dim, page, group, kv_heads, tokens, prefix
    (BF, 128, 64, 1, 256, 128, 128),            # a block's two parts are one tile of keys each
    (FP, 64, 16, 1, 256, 128, 128),
    (BF, 64, 64, 1, 32, 64, 20_000),            # 1 and then 33 tiles
    (FP, 128, 128, 1, 40, 64, 10_000),          # 1 and then 21
    (BF, 128, 64, 5, 160, 9, 300),              # 3 + 1, 2 + 2, 1 + 3; rows of Q's tile that no copy writes
]


def test_sizes_whose_parts_have_one_tile():
    for dtype, dim, page, group, kv_heads, tokens, prefix in ONE_TILE:
        paired, units, parts = R.prefix_parts(tokens, group, kv_heads, prefix, MULTIPROCESSORS)
        assert not paired and any(len(p) > 1 and p[0][1] == 1 for p in parts)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(ONE_TILE)))
def test_parts_of_one_tile(case, prefix_kernel):  # noqa: F811
    """One tile of rows, its tiles of keys dealt to two streams: one of them has nothing to do in a part of one tile."""
    dtype, dim, page, group, kv_heads, tokens, prefix = ONE_TILE[case]
    prefix_kernel(1)
    s = R.Setup(300 + case, dtype=dtype, dim=dim, page=page, heads=group * kv_heads, kv_heads=kv_heads, new=[tokens], lens=[tokens], prefix=prefix, padding=1)
    first, first_lse = attend(s)
    check(s, first, first_lse)
    for _ in range(3):
        out, lse = attend(s)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)


MANY_TILES = [
    # dtype, dim, page, group, kv_heads, tokens, prefix: one tile of rows, many of keys
    (BF, 128, 16, 3, 1, 40, 60_000),            # pages all over the pool
    (FP, 64, 16, 7, 2, 18, 50_000),
    (BF, 128, 128, 1, 149, 20, 1_500),          # more key heads than multiprocessors: runs of 12 tiles and more
    (FP, 128, 64, 2, 150, 64, 700),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(MANY_TILES)))
def test_tiles_that_are_dealt_to_two_streams(case, prefix_kernel):  # noqa: F811
    """Each stream waits for the tiles that it uses, whatever has become of the other one's."""
    dtype, dim, page, group, kv_heads, tokens, prefix = MANY_TILES[case]
    prefix_kernel(1)
    s = R.Setup(320 + case, dtype=dtype, dim=dim, page=page, heads=group * kv_heads, kv_heads=kv_heads, new=[tokens], lens=[tokens], prefix=prefix)
    first, first_lse = attend(s)
    check(s, first, first_lse)
    for _ in range(10):
        out, lse = attend(s)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)


PAIRED = [
    # dtype, dim, page, group, kv_heads, tokens, prefix: two tiles of rows and more to a block
    (BF, 128, 64, 3, 160, 60, 300),             # 126 rows to a tile: Q's rows that no copy writes are zeroed again after each part
    (FP, 128, 16, 5, 151, 40, 640),
    (BF, 64, 32, 7, 152, 30, 1_000),
    (FP, 128, 64, 1, 150, 129, 260),            # one row in the second tile
    (BF, 128, 128, 7, 75, 90, 700),             # five tiles of rows: three units, the last with one
]


def test_sizes_whose_blocks_have_several_parts():
    for dtype, dim, page, group, kv_heads, tokens, prefix in MANY_TILES[2:]:
        paired, units, parts = R.prefix_parts(tokens, group, kv_heads, prefix, MULTIPROCESSORS)
        assert not paired and any(len(p) > 1 for p in parts)
    for dtype, dim, page, group, kv_heads, tokens, prefix in PAIRED:
        paired, units, parts = R.prefix_parts(tokens, group, kv_heads, prefix, MULTIPROCESSORS)
        assert paired and any(len(p) > 1 for p in parts)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(PAIRED)))
def test_parts_of_two_tiles_of_rows(case, prefix_kernel):  # noqa: F811
    dtype, dim, page, group, kv_heads, tokens, prefix = PAIRED[case]
    prefix_kernel(1)
    s = R.Setup(340 + case, dtype=dtype, dim=dim, page=page, heads=group * kv_heads, kv_heads=kv_heads, new=[tokens], lens=[tokens], prefix=prefix, padding=2)
    first, first_lse = attend(s)
    check(s, first, first_lse)
    for _ in range(3):
        out, lse = attend(s)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)
