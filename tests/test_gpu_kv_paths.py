"""Paths of the paged key/value cache that take more of something than the other tests have: heads and blocks to a choice of pages, tiles of rows
than multiprocessors, tokens of a prompt, prefix kernels of several parts at once."""
import pytest
import torch

from tests import kv_reference as R
from tests import test_gpu_kv as T
from tests.test_gpu_kv import attend, check_pages, check_rows, handles, prefix_kernel, run_selected  # noqa: F401  (a fixture)
from tests.test_gpu_kv_parts import MULTIPROCESSORS, check

BF, FP = torch.bfloat16, torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,page,heads,kv_heads,new,lens,budget", [
    (BF, 64, 16, 40, 1, [1], [16 * 601], 9),                 # eight blocks, three rounds of 16 heads
    (FP, 128, 16, 34, 2, [2, 1], [16 * 300 + 5, 70], 6),      # the second sequence has fewer pages than the budget
    (BF, 128, 32, 17, 1, [1], [32 * 130], 129),               # one of 127 pages is left out
])
def test_several_blocks_choose_pages_for_many_heads(dtype, dim, page, heads, kv_heads, new, lens, budget):
    s = R.Setup(700, dtype=dtype, dim=dim, page=page, heads=heads, kv_heads=kv_heads, new=new, lens=lens)
    assert s.table.shape[1] > 64 and s.tokens * kv_heads * 2 <= MULTIPROCESSORS          # more than one block to a choice
    out, lse, pages = run_selected(s, budget, 1, 2)
    want, picks = R.attend_selected(s, budget, 1, 2)
    check_pages(s, pages, picks, budget)
    check_rows(s, out, lse, want)


UNITS = [
    # dtype, dim, page, group, kv_heads, tokens, prefix: pairs of row tiles beyond one round of multiprocessors
    (BF, 64, 64, 128, 1, 298, 200),                          # 149
    (FP, 128, 16, 100, 2, 301, 130),                         # 151, the last of one tile; runs over both key heads
    (BF, 128, 128, 64, 1, 1200, 400),                        # 300
]


def test_sizes_with_more_units_than_multiprocessors():
    for dtype, dim, page, group, kv_heads, tokens, prefix in UNITS:
        paired, units, parts = R.prefix_parts(tokens, group, kv_heads, prefix, MULTIPROCESSORS)
        assert paired and units > MULTIPROCESSORS and all(len(p) == kv_heads for p in parts)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(UNITS)))
def test_more_units_than_multiprocessors(case, prefix_kernel):  # noqa: F811
    dtype, dim, page, group, kv_heads, tokens, prefix = UNITS[case]
    prefix_kernel(1)
    s = R.Setup(710 + case, dtype=dtype, dim=dim, page=page, heads=group * kv_heads, kv_heads=kv_heads, new=[tokens], lens=[tokens], prefix=prefix, padding=1)
    out, lse = attend(s)
    check(s, out, lse)


PROMPTS = [
    # dtype, dim, page, group, kv_heads, new, lens, prefix
    (BF, 128, 64, 4, 2, 700, 700, 0), (FP, 64, 16, 3, 1, 1000, 1300, 0), (FP, 128, 128, 1, 2, 513, 600, 300), (BF, 64, 32, 8, 1, 300, 300, 1000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("tensor", [0, 1])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompts(case, tensor, prefix_kernel):  # noqa: F811
    dtype, dim, page, group, kv_heads, new, lens, prefix = PROMPTS[case]
    prefix_kernel(tensor)
    s = R.Setup(720 + case, dtype=dtype, dim=dim, page=page, heads=group * kv_heads, kv_heads=kv_heads, new=[new], lens=[lens], prefix=prefix, padding=2, leading=1)
    out, lse = attend(s)
    check(s, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("tensor", [0, 1])
def test_prompts_beside_single_tokens(tensor, prefix_kernel):  # noqa: F811
    prefix_kernel(tensor)
    s = R.Setup(730, dtype=FP, dim=64, page=16, heads=6, kv_heads=2, new=[1, 150, 1, 0, 70], lens=[400, 150, 1, 30, 333], prefix=100, padding=3)
    out, lse = attend(s)
    check_rows(s, out, lse, R.attend(s))


@pytest.mark.gpu
@pytest.mark.parametrize("tensor", [0, 1])
def test_two_graphs_and_two_streams_by_either_prefix_kernel(tensor, prefix_kernel):  # noqa: F811
    prefix_kernel(tensor)
    T.test_two_graphs_and_two_streams_do_not_share_workspaces()
    T.test_equal_calls_give_equal_bits()


@pytest.mark.gpu
def test_prefix_kernels_of_several_parts_on_two_streams(prefix_kernel):  # noqa: F811
    """Eager calls and replays of two caches side by side give the bits that each gives alone, however often."""
    prefix_kernel(1)
    work = []
    for seed, (group, kv_heads, tokens, prefix) in enumerate(((5, 160, 9, 700), (3, 150, 60, 900))):
        paired, units, parts = R.prefix_parts(tokens, group, kv_heads, prefix, MULTIPROCESSORS)
        assert paired == bool(seed) and any(len(p) > 1 for p in parts)
        s = R.Setup(740 + seed, dtype=BF, dim=128, page=64, heads=group * kv_heads, kv_heads=kv_heads, new=[1] * tokens, lens=[40 * i % 130 + 1 for i in range(tokens)], prefix=prefix)
        cache, batch = handles(s)
        q, pre = s.q.cuda(), s.prefix_pages.cuda()

        def run(cache=cache, batch=batch, q=q, pre=pre, prefix=prefix):
            return cache.attend(batch, q, prefix_pages=pre, prefix_len=prefix)
        alone = run().clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = run()
        work.append((run, alone, graph, got, torch.cuda.Stream(), cache))
    for _ in range(10):
        torch.cuda.synchronize()
        eager = []
        for run, alone, graph, got, stream, cache in work:
            got.zero_()
        torch.cuda.synchronize()
        for run, alone, graph, got, stream, cache in work:
            with torch.cuda.stream(stream):
                eager.append(run())
                graph.replay()
                eager.append(run())
        torch.cuda.synchronize()
        for i, (run, alone, graph, got, stream, cache) in enumerate(work):
            assert torch.equal(got, alone) and torch.equal(eager[2 * i], alone) and torch.equal(eager[2 * i + 1], alone)
            cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [[0, 3, 1, 3], [2, 0, 3, 1], [0, 2, 0, 3], [-5, 9, -5, 9]])
def test_blocks_of_a_choice_agree_where_sequences_overlap(offsets):
    """Offsets that do not ascend put a row into several sequences, some with fewer pages than the budget: all blocks take the lowest of them."""
    s = R.Setup(750, dtype=BF, dim=64, page=16, heads=2, kv_heads=1, new=[1, 1, 1], lens=[30, 16 * 700, 16 * 500], padding=0)
    cache, batch = handles(s)
    batch.offsets.copy_(torch.tensor(offsets, dtype=torch.int32))
    spans = [(max(0, min(a, 3)), max(max(0, min(a, 3)), min(b, 3))) for a, b in zip(offsets, offsets[1:])]
    q = s.q.cuda()
    for _ in range(3):
        pages = torch.full((3, 1, 6), 7, dtype=torch.int32, device="cuda")
        cache.attend_selected(batch, q, budget=6, first=1, recent=2, pages=pages)
        cache.check()
        for t in range(3):
            mine = [b for b, (first, last) in enumerate(spans) if first <= t < last]
            if not mine:
                assert (pages[t] == 7).all()
                continue
            b = mine[0]
            want = R.choose(s, t, 0, b, s.lens[b] - spans[b][1] + t, 6, 1, 2)
            assert pages[t, 0].tolist() == want + [-1] * (6 - len(want)), (t, b)
