"""Rows behind the last sequence and rows that see nothing, in batches padded to
fixed sizes: all zero, the other rows as without padding, whatever the output's
memory held, and at no cost that grows out of proportion."""

import pytest
import torch

from sglang_mlx_amd import kernels
from test_gpu_extend import BF, HF, U8, Batch

pytestmark = pytest.mark.gpu


def padded(b, rows, seqs=0):
    """`rows` more query rows, `seqs` sequences without rows before them."""
    n = b.q.shape[0]
    b.q = torch.cat([b.q, torch.ones((rows, b.Hq, b.D), dtype=b.q.dtype, device="cuda")])
    b.lens = torch.cat([b.lens, torch.zeros(seqs, dtype=torch.int32, device="cuda")])
    b.start = torch.cat([b.start, torch.full((seqs,), n, dtype=torch.int32, device="cuda")])
    b.table = torch.cat([b.table, torch.full((seqs, b.table.shape[1]), -1, dtype=torch.int32, device="cuda")])
    return n


def over_nan(b, call):
    """The call's output, in memory that held NaN."""
    torch.cuda.synchronize()
    dirty = torch.full(b.q.shape, float("nan"), dtype=b.q.dtype, device="cuda")
    at = dirty.data_ptr()
    del dirty
    out = call()
    assert out.data_ptr() == at
    return out


@pytest.mark.parametrize("heads,D,types", [((8, 2), 128, (BF, BF)), ((1, 1), 32, (HF, HF)), ((28, 4), 80, (BF, U8)),
                                           ((40, 2), 256, (HF, HF)), ((9, 3), 120, (BF, BF)), ((64, 64), 192, (BF, BF))])
@pytest.mark.parametrize("rows,seqs", [(1, 0), (7, 3), (255, 255), (1000, 1)])
def test_rows_behind_the_last_sequence(heads, D, types, rows, seqs):
    for new in ([1, 1, 0, 1], [4, 1, 0, 3], [70, 1, 0, 3]):
        b = Batch(rows + D, [600, 1, 9, 300], new, heads, D, 16, *types)
        alone = [b.extend(), b.extend(100, 5)]
        n = padded(b, rows, seqs)
        for want, window in zip(alone, ((0, 0), (100, 5))):
            got = over_nan(b, lambda: b.extend(*window))
            # (Other sizes may cut the length into other parts: the bound instead of the bits.)
            b.new, b.ctx = list(new), [600, 1, 9, 300]
            value, bound = b.expected(*window)
            assert ((got[:n].double() - value[:n]).abs() <= bound[:n]).all()
            assert ((want.double() - value[:n]).abs() <= bound[:n]).all()
            assert (got[n:] == 0).all()


def test_sequences_without_a_context_or_of_too_many_rows():
    for new, most in (([1, 1, 1], 1), ([3, 2, 3], 3), ([300, 5, 4], 5), ([300, 200, 1], 200)):
        b = Batch(5, [0, 300, 0], new, (8, 2))
        got = over_nan(b, lambda: b.extend(max_query_len=most))
        value, bound = b.expected()
        seen = slice(new[0], new[0] + new[1])
        assert ((got[seen].double() - value[seen]).abs() <= bound[seen]).all()
        assert (got[:new[0]] == 0).all() and (got[new[0] + new[1]:] == 0).all()


def test_more_padding_than_sequences_costs_little():
    # One sequence in a batch of 256 rows: the call that a captured graph of 256
    # slots replays when one user is left.  (10 us and 12 us; 77 us when one
    # workgroup per KV head wrote all zeros.)
    def timed(call):
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                call()
        best = float("inf")
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    b = Batch(6, [4000], [1], (32, 8))
    alone = timed(b.extend)
    padded(b, 255)
    assert timed(b.extend) < 3 * alone
