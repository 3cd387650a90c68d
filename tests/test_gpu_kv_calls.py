"""Calls of the paged key/value cache that its documents allow or forbid and that nothing else makes."""
import pytest
import torch

from tests import kv_reference as R
from tests.test_gpu_kv import check_rows, handles

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def fused(s):
    """q, k and v as heads of one projection's output, with room for results behind them."""
    buf = torch.full((s.tokens, 2 * s.heads + 2 * s.kv_heads, s.dim), 3.0, dtype=s.dtype, device="cuda")
    q, k, v, out = buf.split([s.heads, s.kv_heads, s.kv_heads, s.heads], 1)
    q.copy_(s.q), k.copy_(s.k_new), v.copy_(s.v_new)
    return buf, q, k, v, out


def test_results_beside_their_inputs_in_one_buffer():
    s = R.Setup(600, dtype=BF, dim=64, page=16, heads=6, kv_heads=2, new=[2, 1, 3], lens=[2, 100, 64], prefix=90)
    cache, batch = handles(s)
    buf, q, k, v, out = fused(s)
    before = buf.clone()
    cache.attend(batch, q, prefix_pages=s.prefix_pages.cuda(), prefix_len=s.prefix, out=out)
    check_rows(s, out, None, R.attend(s))
    _, pages = cache.attend_selected(batch, q, budget=2, out=out)
    want, picks = R.attend_selected(s, 2, 1, 1)
    check_rows(s, out, None, want)
    assert torch.equal(buf[:, :-s.heads], before[:, :-s.heads])
    angle = torch.rand(200, 32) * 6.28
    cos, sin = torch.cos(angle).cuda(), torch.sin(angle).cuda()
    cache.append(batch, k, v, q=q, q_out=out, cos=cos, sin=sin)
    assert torch.equal(buf[:, :-s.heads], before[:, :-s.heads])
    apart = out.clone()
    cache.append(batch, k, v, q=q, q_out=q, cos=cos, sin=sin)       # in place, between the keys and values it reads
    assert torch.equal(q, apart) and torch.equal(buf[:, s.heads:-s.heads], before[:, s.heads:-s.heads])


def test_results_over_one_another_are_refused():
    s = R.Setup(601, dtype=BF, dim=64, page=16, heads=4, kv_heads=4, new=[1, 1], lens=[5, 40])
    cache, batch = handles(s)
    q, k, v = s.q.cuda(), s.k_new.cuda(), s.v_new.cuda()
    out, lse = torch.zeros_like(q), torch.zeros(2, 4, device="cuda")

    def numbers(t, n):
        return t.view(-1).view(torch.int32)[:n]
    for call in (lambda: cache.append(batch, k, v, q=q, q_out=k), lambda: cache.append(batch, k, v, q=q, q_out=v),
                 lambda: cache.attend(batch, q, out=out, lse=numbers(q, 8).view(torch.float32).view(2, 4)),
                 lambda: cache.attend(batch, q, out=out, lse=numbers(out, 8).view(torch.float32).view(2, 4)),
                 lambda: cache.attend_selected(batch, q, budget=2, out=out, pages=numbers(q, 16).view(2, 4, 2)),
                 lambda: cache.attend_selected(batch, q, budget=2, out=out, pages=numbers(out, 16).view(2, 4, 2)),
                 lambda: cache.attend_selected(batch, q, budget=1, recent=0, out=out, lse=lse, pages=lse.view(torch.int32).view(2, 4, 1))):
        with pytest.raises(ValueError, match="overlap"):
            call()


def test_gradients_are_refused_and_not_dropped():
    from turbovec_b200.kvcache import PagedKVCache
    s = R.Setup(602, dtype=BF, dim=64, page=16, heads=4, kv_heads=2, new=[1, 1], lens=[5, 40])
    cache, batch = handles(s)
    q, k, v = s.q.cuda(), s.k_new.cuda(), s.v_new.cuda()
    cos = torch.rand(60, 32, device="cuda")

    def asks(t):
        return t.detach().clone().requires_grad_()
    calls = [lambda: cache.attend(batch, asks(q)), lambda: cache.attend_selected(batch, asks(q), budget=2), lambda: cache.attend(batch, q, out=asks(q)),
             lambda: cache.attend(batch, q, lse=asks(torch.zeros(2, 4, device="cuda"))),
             lambda: cache.append(batch, asks(k), v), lambda: cache.append(batch, k, asks(v)), lambda: cache.append(batch, k, v, q=asks(q)),
             lambda: cache.append(batch, k, v, cos=asks(cos), sin=cos), lambda: cache.append(batch, k, v, cos=cos, sin=asks(cos))]
    k_pool, v_pool = asks(cache.k), asks(cache.v)
    for pools in ((k_pool, cache.v), (cache.k, v_pool)):
        other = PagedKVCache(*pools, cache.bounds, cache.scales)
        calls += [lambda o=other: o.attend(batch, q), lambda o=other: o.attend_selected(batch, q, budget=2), lambda o=other: o.append(batch, k, v)]
    kept = cache.k.clone()
    for call in calls:
        with pytest.raises(RuntimeError, match="gradient"):
            call()
    assert torch.equal(cache.k, kept)
    want = cache.attend(batch, q)
    with torch.no_grad():                               # nobody asks for one
        assert torch.equal(cache.attend(batch, asks(q)), want)
        assert torch.equal(PagedKVCache(k_pool, v_pool).attend(batch, asks(q)), want)
        cache.append(batch, asks(k), asks(v), q=asks(q), cos=asks(cos), sin=asks(cos))


def test_a_reported_error_does_not_wait_for_the_next_call():
    """A device number that no machine has: the call says so, and torch's next call meets no error."""
    from turbovec_b200 import _native
    s = R.Setup(603, dtype=BF, dim=64, page=16, heads=4, kv_heads=2, new=[1, 1], lens=[5, 40])
    cache, batch = handles(s)
    q, k = s.q.cuda(), s.k_new.cuda()
    clean = cache.attend(batch, q)
    index, cache._view.device = cache._view.device, 63
    calls = (lambda: cache.append(batch, k, k), lambda: cache.attend(batch, q), lambda: cache.attend_selected(batch, q, budget=2))
    for call in calls:
        cache._sizes.clear()
        with pytest.raises(RuntimeError, match="no such CUDA device"):
            call()
        assert float((q.float() * 0 + 1).sum()) == q.numel()
    assert _native.load().tv_kv_status(63) != 0
    torch.cuda.synchronize()
    cache._view.device = index
    assert torch.cuda.current_device() == index and torch.equal(cache.attend(batch, q), clean)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two devices are needed")
def test_the_callers_device_stays_the_current_one():
    s = R.Setup(604, dtype=BF, dim=64, page=16, heads=4, kv_heads=2, new=[1, 1], lens=[5, 40], prefix=30)
    cache, batch = handles(s)
    q, k, pre = s.q.cuda(), s.k_new.cuda(), s.prefix_pages.cuda()
    want = cache.attend(batch, q, prefix_pages=pre, prefix_len=30)
    with torch.cuda.device(1):
        assert torch.equal(cache.attend(batch, q, prefix_pages=pre, prefix_len=30), want)
        cache.attend_selected(batch, q, budget=2)
        cache.append(batch, k, k)
        cache.check()
        assert torch.cuda.current_device() == 1


@pytest.mark.parametrize("tensor", [0, 1])
def test_a_batch_without_pages_of_its_own(tensor):
    """Tables of no width: rows see the prefix alone, choose nothing, and append nothing."""
    from turbovec_b200 import kvcache
    s = R.Setup(605, dtype=BF, dim=128, page=16, heads=4, kv_heads=2, new=[1, 2], lens=[0, 0], prefix=150)
    cache, _ = handles(s)
    batch = kvcache.KVBatch(torch.zeros(2, 0, dtype=torch.int32, device="cuda"), torch.tensor([0, 9], dtype=torch.int32, device="cuda"),
                            torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda"))
    s.lens, s.table = [-5, -5], s.table[:, :0]
    q, k = s.q.cuda(), s.k_new.cuda()
    kvcache.set_option(kvcache.OPT_TENSOR_PREFIX, tensor)
    try:
        out = cache.attend(batch, q, prefix_pages=s.prefix_pages.cuda(), prefix_len=150)
    finally:
        kvcache.set_option(kvcache.OPT_TENSOR_PREFIX, -1)
    want = R.attend(s)
    check_rows(s, out, None, {t: want[t] for t in range(3)})
    assert (cache.attend(batch, q) == 0).all()
    out, pages = cache.attend_selected(batch, q, budget=3)
    assert (out == 0).all() and (pages == -1).all()
    before = cache.k.clone()
    cache.append(batch, k, k)
    cache.check()
    assert torch.equal(cache.k, before)
