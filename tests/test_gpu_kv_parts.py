"""Attention over a prefix by the tensor-memory kernel where its blocks have several parts (runs of keys that go from one key head to the
next), against the restatement in 64 bits."""
import pytest
import torch

from tests import kv_reference as R
from tests.test_gpu_kv import attend, prefix_kernel  # noqa: F401  (a fixture)

BF, FP = torch.bfloat16, torch.float16
MULTIPROCESSORS = 148


def check(s, out, lse, weight_step=None):
    want, want_lse, tol, ltol = R.attend_sequence(s, weight_step=weight_step)
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
