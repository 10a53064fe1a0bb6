"""The maps of a step (paged.step_maps) against one loop over requests and tokens: whole numbers, equal."""
from __future__ import annotations

import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from oracle import kv4_oracle as orc

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def run(dev, q, past, width, page, tokens, free=None, head=0, seed=0, table=None):
    from qwen_a100_fastpath_b200.paged import step_maps
    rng = random.Random(seed)
    if table is None:
        table = [[rng.randrange(-1, 5000) for _ in range(width)] for _ in q]
    t = i32(table, dev).view(len(q), width)
    want = orc.step_maps(q, past, table, page, tokens, free, head)
    if free is None:
        m = step_maps(i32(q, dev), i32(past, dev), t, page, tokens)
        assert m.free_head is None
    else:
        h = i32([head], dev)
        m = step_maps(i32(q, dev), i32(past, dev), t, page, tokens, free_pages=i32(free, dev), free_head=h)
        assert m.free_head.tolist() == [want[4]] and h.tolist() == [head]
    assert m.query_start.tolist() == want[0] and m.seq_lens.tolist() == want[1]
    assert m.positions.dtype == torch.int64 and m.positions.tolist() == want[2]
    assert m.slots.dtype == torch.int64 and m.slots.tolist() == want[3]
    assert t.tolist() == want[5]
    return m


@pytest.mark.parametrize("grow", [False, True])
@pytest.mark.parametrize("page", [1, 7, 16, 800])
@pytest.mark.parametrize("b", [1, 2, 31, 33, 255, 256, 257, 700])
def test_random_requests(dev, b, page, grow):
    rng = random.Random(b * page)
    q = [rng.choice((0, 1, 1, 1, 5, rng.randrange(40))) for _ in range(b)]
    past = [rng.choice((0, rng.randrange(3 * page + 2), page, 2 * page)) for _ in range(b)]
    width = 6 if page > 7 else 40
    pad = rng.choice((0, 9))
    free = list(range(10000, 10000 + 45 * b)) if grow else None
    run(dev, q, past, width, page, sum(q) + pad, free, 3 if grow else 0, seed=b)


@pytest.mark.parametrize("q,past,width,page,tokens,free,head", [
    ([], [], 3, 16, 5, None, 0), ([], [], 3, 16, 0, [1, 2], 1),
    ([0, 0], [0, 0], 2, 16, 4, [5, 6], 0),
    ([-4, 3], [5, -2], 2, 16, 6, [5, 6], 0),                  # negative lengths count as zero
    ([40, 40], [0, 0], 4, 16, 80, [9, 8, 7, 6], 0),           # the list runs out inside the second request
    ([40, 40], [0, 0], 4, 16, 80, [9, 8], 5),                 # a head behind the list
    ([40, 40], [0, 0], 4, 16, 80, [], 0),                     # no pages at all
    ([40, 40], [0, 0], 4, 16, 10, list(range(20)), 0),        # fewer places than tokens: pages are taken all the same
    ([100], [30], 4, 16, 100, list(range(20)), 0),            # behind the table's width
    ([100], [30], 0, 16, 100, list(range(20)), 0),            # a table of no entries
    ([5], [2147483640], 3, 16, 5, [1], 0), ([5], [33], 3, 2147483647, 5, [1], 0),
    ([16, 1, 15, 17], [16, 15, 1, 0], 4, 16, 49, list(range(50, 60)), 2),
])
def test_edges(dev, q, past, width, page, tokens, free, head):
    run(dev, q, past, width, page, tokens, free, head)


def test_many_requests(dev):
    rng = random.Random(4)
    b = 16384
    q = [rng.randrange(3) for _ in range(b)]
    run(dev, q, [rng.randrange(20) for _ in range(b)], 3, 8, sum(q) + 1, list(range(b)), 0)


def test_request_counts_around_48_kilobytes_of_scan(dev):
    """In a process of its own: no earlier call with more requests has asked for the larger shared memory."""
    code = """
import random, torch
from tests.test_gpu_step_maps import run
rng = random.Random(6)
for b in (4088, 4090, 4091, 4093, 4095, 4096, 4097):
    q = [rng.randrange(3) for _ in range(b)]
    run(torch.device("cuda", 0), q, [rng.randrange(20) for _ in range(b)], 3, 8, sum(q) + 1, list(range(b)), 0)
"""
    got = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True,
                         timeout=600)
    assert got.returncode == 0, got.stderr[-2000:]


def test_one_long_prompt_among_others(dev):
    run(dev, [1, 70000, 1, 0, 300], [10, 0, 5, 9, 2], 1200, 64, 70400, list(range(3000)), 0)


def test_pages_behind_the_map_are_opened_page_by_page(dev):
    """Lengths far above the places for tokens: the work goes by the pages that are opened, not by the tokens."""
    from qwen_a100_fastpath_b200.paged import step_maps
    huge = 2 ** 31 - 10
    for tokens in (0, 8, 300):
        run(dev, [3, huge, 5], [2, 3, 7], 6, 16, tokens, list(range(100, 140)), 1)
        run(dev, [huge, 0, 9], [0, 31, 2 ** 31 - 20], 4, 1, tokens, list(range(5)), 0)
    rng = random.Random(2)
    q = [rng.randrange(4000) for _ in range(300)]
    run(dev, q, [rng.randrange(200) for _ in q], 70, 64, 100, list(range(9000)), 3)
    # the pages of contexts that are there already, without a place for any token: 400000 entries
    b, n = 64, 100000
    lens, none = i32([n] * b, dev), i32([0] * b, dev)
    table, head = torch.full((b, n // 16), -1, dtype=torch.int32, device=dev), i32([0], dev)
    free = torch.randperm(b * n // 16, device=dev).to(torch.int32)
    times = []
    for _ in range(6):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        m = step_maps(lens, none, table, 16, 0, free_pages=free, free_head=head)
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    assert torch.equal(table.view(-1), free) and m.free_head.item() == free.numel()
    assert min(times) < 1.0, times      # 25000 turns of one CTA over 6.4 million tokens took several milliseconds


def test_sums_stop_at_the_largest_number(dev):
    from qwen_a100_fastpath_b200.paged import step_maps
    big = 2 ** 31 - 1
    m = step_maps(i32([big, big, 7], dev), i32([big, 0, 3], dev), i32([[0, 1]] * 3, dev), 16, 40)
    assert m.query_start.tolist() == [0, big, big, big] and m.seq_lens.tolist() == [big, big, 10]
    assert m.slots.tolist() == [-1] * 40


def test_wide_rows_views_and_repeats(dev):
    """A table that is a view of a wider one, strided lengths; the same call again; entries around the new ones untouched."""
    from qwen_a100_fastpath_b200.paged import step_maps
    wide = torch.full((4, 9), -5, dtype=torch.int32, device=dev)
    table = wide[1:3, 2:8]
    q, past = i32([20, 99, 4, 99], dev)[::2], i32([[3, 30], [0, 0]], dev)[0]
    free, head = i32([70, 71, 72, 73], dev), i32([1], dev)
    version = table._version
    a = step_maps(q, past, table, 16, 24, free_pages=free, free_head=head)
    assert table._version > version
    want = wide.clone()
    b = step_maps(q, past, table, 16, 24, free_pages=free, free_head=head)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(wide, want)
    assert a.free_head.tolist() == [3]
    exp = torch.full((4, 9), -5, dtype=torch.int32)
    exp[1, 3], exp[2, 4] = 71, 72           # past 3 of 23: page 1; past 30 of 34: page 2
    assert torch.equal(wide.cpu(), exp)
    c = step_maps(q, past, table.t().contiguous().t(), 16, 24)     # columns adjacent: read through a copy
    assert torch.equal(c.slots, a.slots)


def test_graph_with_other_lengths(dev):
    from qwen_a100_fastpath_b200.paged import step_maps
    q, past = i32([1, 2, 3], dev), i32([4, 5, 6], dev)
    table, free, head = i32([[0, 1, 2]] * 3, dev), i32(list(range(9, 30)), dev), i32([0], dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m = step_maps(q, past, table, 4, 16, free_pages=free, free_head=head)
    for seed in range(5):
        rng = random.Random(seed)
        ql, pl, h = [rng.randrange(5) for _ in range(3)], [rng.randrange(9) for _ in range(3)], rng.randrange(4)
        q.copy_(i32(ql, dev)), past.copy_(i32(pl, dev)), head.copy_(i32([h], dev)), table.copy_(i32([[0, 1, 2]] * 3, dev))
        graph.replay()
        torch.cuda.synchronize()
        want = orc.step_maps(ql, pl, [[0, 1, 2]] * 3, 4, 16, list(range(9, 30)), h)
        assert [t.tolist() for t in m] == [*want[:4], [want[4]]] and table.tolist() == want[5]
