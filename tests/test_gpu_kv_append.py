"""Appends that leave tokens out, and bounds of the pages that they concern, against the restatement in 64 bits."""
import pytest
import torch

from tests import kv_reference as R
from tests.test_gpu_kv import handles

BF, FP = torch.bfloat16, torch.float16


def widened(old, old_step, keys):
    """Bounds of a page that `keys` [n, dim] are added to."""
    new, step = R.bounds_of(keys)
    wide = max(step, old_step)
    keys = keys.double()
    lo, hi = torch.floor(keys.amin(0) / wide), torch.ceil(keys.amax(0) / wide)
    old = old.double() * (old_step / wide)
    return torch.stack([torch.minimum(torch.floor(old[0]), lo), torch.maximum(torch.ceil(old[1]), hi)]), wide


LEFT_OUT = [
    # dtype, dim, page, kv_heads, new, lens, positions, offset, pieces
    (BF, 64, 16, 2, 40, 40, 100, -20, 1),                 # angles from position 20 on: a page without any, one that begins at place 4
    (FP, 128, 16, 1, 70, 70, 50, 0, 1),                   # ... up to position 49: a page of two, and one without any
    (BF, 128, 64, 3, 200, 230, 150, -40, 1),              # nothing below 40 and from 190 on; the first page holds earlier tokens
    (BF, 64, 32, 8, 90, 90, 60, -10, 9),                  # the same in pieces of ten
    (FP, 64, 128, 2, 5, 300, 10, 0, 1),                   # none at all
    (FP, 64, 16, 1, 20, 20, 8, -2 ** 40, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(LEFT_OUT)))
def test_tokens_without_an_angle_change_nothing(case):
    """They are neither stored nor rotated, and a page's bounds are those of the tokens that are: a page whose first place is written starts anew, one
    with later places written is widened, one without any is as it was."""
    dtype, dim, page, kv_heads, new, lens, positions, offset, pieces = LEFT_OUT[case]
    s = R.Setup(500 + case, dtype=dtype, dim=dim, page=page, heads=2 * kv_heads, kv_heads=kv_heads, new=[new], lens=[lens])
    g = torch.Generator().manual_seed(case)
    angle = torch.rand(positions, dim // 2, generator=g) * 6.28
    cos, sin = torch.cos(angle), torch.sin(angle)
    cache, batch = handles(s)
    q_out = torch.full_like(s.q, 7.0).cuda()
    size = new // pieces
    for i in range(pieces):
        rows = slice(i * size, (i + 1) * size)
        batch.lens.fill_(lens - new + (i + 1) * size)
        batch.offsets.copy_(torch.tensor([0, size], dtype=torch.int32))
        cache.append(batch, s.k_new[rows].cuda(), s.v_new[rows].cuda(), q=s.q[rows].cuda(), q_out=q_out[rows], cos=cos.cuda(), sin=sin.cuda(), position_offset=offset)
    k, v, got = cache.k.cpu(), cache.v.cpu(), q_out.cpu()
    want_k, want_v = s.k.clone(), s.v.clone()
    stored = {}
    for t, b, p in s.rows():
        if not 0 <= p + offset < positions:
            assert (got[t] == 7).all(), t
            continue
        c, sn = cos[p + offset], sin[p + offset]
        y, tol = R.rotate(s.q[t], c, sn, False)
        assert ((got[t].double() - y).abs() <= tol).all(), t
        pg = s.page_at(b, p // page)
        y, tol = R.rotate(s.k_new[t], c, sn, False)
        assert ((k[pg, :, p % page].double() - y).abs() <= tol).all(), t
        want_k[pg, :, p % page], want_v[pg, :, p % page] = k[pg, :, p % page], s.v_new[t]
        stored.setdefault(pg, []).append(p % page)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    want_b, want_s = s.bounds.clone(), s.scales.clone()
    for pg, places in stored.items():
        for h in range(kv_heads):
            keys = k[pg, h, places]
            both, step = R.bounds_of(keys) if places[0] == 0 else widened(s.bounds[pg, h], float(s.scales[pg, h]), keys)
            want_b[pg, h], want_s[pg, h] = both.to(torch.int8), step
    assert torch.equal(cache.bounds.cpu(), want_b) and torch.equal(cache.scales.cpu(), want_s)
