"""How exact the attention's weights are, against the restatement in 64 bits."""
import pytest
import torch

from tests import kv_reference as R
from tests.test_gpu_kv import attend, prefix_kernel, run_selected  # noqa: F401  (a fixture)
from tests.test_gpu_kv_parts import check

BF, FP = torch.bfloat16, torch.float16


def with_a_sink(dtype, dim, prefix, lens, place, logit):
    """One key whose logit is `logit` above zero and whose value is zero; values of the others around 400: what the row gives comes from weights
    of exp(-logit) times the largest."""
    s = R.Setup(400, dtype=dtype, dim=dim, page=64, heads=6, kv_heads=2, new=[3], lens=[lens], prefix=prefix)
    s.q *= 0.25
    s.q[..., 0] = 8.0
    s.k[..., 0] = 0.0
    s.v += 400
    p, o = (s.prefix_keys() + s.own_keys(0, lens - 1))[place]
    s.k[p, :, o, 0] = logit * dim ** 0.5 / 8
    s.v[p, :, o] = 0.0
    return s


# float16 has steps of 2^-24 and no smaller ones: half of one is 2^-36 of a row's largest weight, which is 2^11 at least
LEAST = {FP: 2.0 ** -36, BF: 0.0}


@pytest.mark.gpu
@pytest.mark.parametrize("tensor", [0, 1])
@pytest.mark.parametrize("place", [0, 150, -4])
@pytest.mark.parametrize("dtype,dim", [(FP, 128), (FP, 64), (BF, 128)])
def test_keys_beside_a_much_larger_one(dtype, dim, place, tensor, prefix_kernel):  # noqa: F811
    """Weights of 2^-26 times the largest: below float16's range, and together all that the row gives."""
    prefix_kernel(tensor)
    for prefix, lens in ((333, 70), (0, 403)):
        s = with_a_sink(dtype, dim, prefix, lens, place, 18.0)
        out, lse = attend(s)
        check(s, out, lse, least=LEAST[dtype])
    out, lse, _ = run_selected(s, 7, 1, 1)              # all pages: the same keys
    check(s, out, lse, least=LEAST[dtype])


# Weights that are two numbers of the type, the second what the first leaves, are off by half a step of half a step: 2^-16 in bfloat16, 2^-22 in float16.
CARRIED = {BF: 2.0 ** -16, FP: 2.0 ** -22}
EXACT = [
    # dtype, dim, page, group, prefix, lens
    (BF, 128, 64, 4, 0, 700), (FP, 64, 16, 3, 0, 300), (BF, 64, 32, 2, 500, 90), (FP, 128, 128, 5, 300, 60),
]


def plain_logits(case):
    """Queries of one channel: logits are single products, and what 32 bits may be off by is far below a step of the type."""
    dtype, dim, page, group, prefix, lens = EXACT[case]
    s = R.Setup(420 + case, dtype=dtype, dim=dim, page=page, heads=2 * group, kv_heads=2, new=[5], lens=[lens], prefix=prefix)
    s.q[..., 1:] = 0.0
    return s


@pytest.mark.parametrize("case", range(len(EXACT)))
def test_the_tolerance_of_carried_weights_tells_them_from_rounded_ones(case):
    """Weights rounded to the type once, everything else in 64 bits and the result rounded, is outside of it."""
    s = plain_logits(case)
    want, lse, tol, _ = R.attend_sequence(s, weight_step=CARRIED[s.dtype], least=LEAST[s.dtype], terms=1)
    pre, own = s.prefix_keys(), s.own_keys(0, s.lens[0] - 1)
    pp, oo = [p for p, _ in pre + own], [o for _, o in pre + own]
    k, v = s.k[pp, 0, oo].double(), s.v[pp, 0, oo].double()
    t = s.offsets[0] + s.new[0] - 1                    # the last row sees all keys
    logits = k @ s.q[t, 0].double() * s.dim ** -0.5
    w = torch.exp(logits - logits.max())
    rounded = ((w.to(s.dtype).double() @ v) / w.sum()).to(s.dtype).double()
    exact = ((w @ v) / w.sum()).to(s.dtype).double()
    assert ((exact - want[-1, 0]).abs() <= tol[-1, 0]).all()
    assert ((rounded - want[-1, 0]).abs() > tol[-1, 0]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(EXACT)))
def test_the_warp_level_kernel_carries_what_rounding_a_weight_leaves(case, prefix_kernel):  # noqa: F811
    prefix_kernel(0)
    s = plain_logits(case)
    out, lse = attend(s)
    check(s, out, lse, weight_step=CARRIED[s.dtype], least=LEAST[s.dtype], terms=1)
    if s.prefix == 0:
        out, lse, _ = run_selected(s, s.table.shape[1], 1, 1)
        check(s, out, lse, weight_step=CARRIED[s.dtype], least=LEAST[s.dtype], terms=1)
