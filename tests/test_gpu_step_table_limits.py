"""build_step_tables at the most tokens and the most blocks that it takes: every
index past the last step of 256 that 31 bits hold."""

import pytest
import torch

from sglang_mlx_amd import kernels

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1


def ints(*a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def free_after():
    yield
    torch.cuda.empty_cache()


def test_most_tokens():
    pool = ints([3, -1, -1])
    tables, slots, positions, start = kernels.build_step_tables(pool, ints(0), ints(40), ints(30), ints(7, 5), 16, MOST)
    assert tables.tolist() == [[3, 7, 5]] and pool.tolist() == [[3, 7, 5]] and start.tolist() == [0, 30]
    assert positions[:30].tolist() == list(range(10, 40))
    assert slots[:30].tolist() == [[3, 7, 5][p // 16] * 16 + p % 16 for p in range(10, 40)]
    assert len(slots) == len(positions) == MOST
    for at in range(30, MOST, 1 << 28):
        assert (slots[at:at + (1 << 28)] == -1).all() and not positions[at:at + (1 << 28)].any()


def test_most_blocks():
    pool = torch.full((1, MOST), 9, dtype=torch.int32, device="cuda")
    tables, slots, positions, _ = kernels.build_step_tables(pool, ints(0), ints(40), ints(9), ints(7, 5), 16, 9)
    assert tables[0, :3].tolist() == [9, 9, 7] and pool[0, :3].tolist() == [9, 9, 7]
    assert positions.tolist() == list(range(31, 40)) and slots.tolist() == [159] + list(range(112, 120))
    for at in range(3, MOST, 1 << 28):
        assert (tables[0, at:at + (1 << 28)] == -1).all() and (pool[0, at:at + (1 << 28)] == 9).all()
