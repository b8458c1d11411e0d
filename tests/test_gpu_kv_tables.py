"""Block tables, slots and positions on the GPU: whole numbers, equal to the oracle's."""
import random

import pytest
import torch

from oracle import kv_oracle as K
from pasa_amd.kv_cache import extend_block_tables

pytestmark = pytest.mark.gpu


def run(device, lens, new, page, tokens, width, spare, pad=0):
    """The step on the GPU and in the oracle, from tables that hold random page ids."""
    rng = random.Random(len(lens) * 7 + tokens)
    have = [-(-n // page) for n in lens]
    ids = list(range(sum(have) + spare))
    rng.shuffle(ids)
    it = iter(ids)
    table = [[next(it) for _ in range(min(h, width))] + [-1] * (width - h) for h in have]
    free = list(it)
    dev = torch.full((len(lens), width + pad), 777, dtype=torch.int32)
    dev[:, :width] = torch.tensor(table, dtype=torch.int32)
    dev = dev.to(device)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    args = i32(lens), i32(new), i32(free), i32([len(free)])
    keep = [a.clone() for a in args]
    step = extend_block_tables(dev[:, :width], *args, page, tokens)
    ref = K.block_tables(table, lens, new, free, len(free), page, tokens)
    got = (dev[:, :width].tolist(), step.cu_q.tolist(), step.slots.tolist(), step.positions.tolist(), step.lens.tolist(),
           step.num_free.tolist()[0])
    for name, g, r in zip(("tables", "cu_q", "slots", "positions", "lens", "num_free"), got, ref):
        assert g == r, name
    assert all(torch.equal(a, b) for a, b in zip(args, keep)), "the inputs stay"
    assert bool((dev[:, width:] == 777).all()), "what lies beside the table stays"
    return step


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("R", [1, 2, 63, 255, 256, 257, 1000, 4096])
def test_single_tokens(device, R, page):
    rng = random.Random(R)
    lens = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, 6 * page)]) for _ in range(R)]
    run(device, lens, [1] * R, page, R, 8, R)


@pytest.mark.parametrize("R,most,page", [(1, 5000, 64), (3, 700, 16), (48, 900, 64), (300, 40, 32), (1024, 9, 128)])
def test_ragged(device, R, most, page):
    rng = random.Random(R)
    lens = [rng.randint(0, 4 * page) for _ in range(R)]
    new = [rng.choice([0, 1, rng.randint(0, most)]) for _ in range(R)]
    width = max(-(-(a + b) // page) for a, b in zip(lens, new)) + 1
    run(device, lens, new, page, sum(new) + 11, width, sum(-(-n // page) + 1 for n in new), pad=3)


def test_where_pages_end(device):
    run(device, [10, 0, 64, 5], [100, 200, 64, 3], 64, 367, 6, 3)           # the free list ends inside request 1
    run(device, [10, 0, 64, 5], [100, 200, 64, 3], 64, 367, 6, 0)           # nothing free: what the pages hold yet
    run(device, [10, 100, 0], [500, 20, 300], 64, 820, 3, 50)               # the table is too narrow
    run(device, [10, 0, 7], [30, 40, 50], 64, 60, 4, 9)                     # more new tokens than the step's size
    run(device, [10, 0, 7], [30, -4, 50], 64, 80, 4, 9)                     # negative: none
    run(device, [0], [0], 64, 0, 1, 0)
    run(device, [5], [0], 64, 4, 1, 0)


def test_out_of_range_lengths_stay_in_bounds(device):
    """Lengths and counts that no step gives: nothing outside the buffers is read or written, slots stay in the cache."""
    table = torch.zeros(3, 4, dtype=torch.int32, device=device)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    step = extend_block_tables(table, i32([2 ** 31 - 1, -5, 300]), i32([2 ** 31 - 1, 3, 2 ** 31 - 1]), i32([1, 2, 3]), i32([99]), 64, 50)
    assert step.cu_q.tolist() == [0, 50, 50, 50] and set(step.slots.tolist()) == {-1}
    assert step.num_free.tolist() == [3]
    dropped = torch.tensor([[-1, 8, -1]], dtype=torch.int32, device=device)   # early pages were given back
    step = extend_block_tables(dropped, i32([70]), i32([3]), i32([1]), i32([1]), 64, 3)
    assert step.slots.tolist() == [8 * 64 + 6, 8 * 64 + 7, 8 * 64 + 8]


def test_graph(device):
    """A captured step, replayed on changed lengths, gives what the eager one gives."""
    R, page = 37, 16
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    table = torch.full((R, 20), -1, dtype=torch.int32, device=device)
    lens, new, free, left = i32([0] * R), i32([3] * R), torch.randperm(500, device=device).int(), i32([500])
    first = table.clone()
    extend_block_tables(table, lens, new, free, left, page, 120)
    torch.cuda.synchronize()
    table.copy_(first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step = extend_block_tables(table, lens, new, free, left, page, 120)
    table.copy_(first)
    other = first.clone()
    for _ in range(4):
        eager = extend_block_tables(other, lens, new, free, left, page, 120)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(table, other)
        for a, b in zip(vars(step).values(), vars(eager).values()):
            assert torch.equal(a, b)
        lens.copy_(eager.lens)
        left.copy_(eager.num_free)
        new.copy_(torch.randint(0, 6, (R,), device=device).int())
