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
