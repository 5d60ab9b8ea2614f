"""Calls of several threads on one stream, which share the stream's scratch: calls
of two launches (split row tiles, partitions that a second kernel merges, cascades)
beside others give the bits that they give alone."""

import threading

import pytest
import torch

from sglang_mlx_amd import kernels
from sglang_mlx_amd.srt.mem_cache import build_cascade_plan
from test_gpu_extend import Batch

pytestmark = pytest.mark.gpu

CALLS = 100


def decode(b):
    return kernels.paged_attention_v1(b.q, b.k, b.v, b.table, b.lens, b.H, b.scale, b.bs, b.max_seq)


def cascade():
    b = Batch(33, [900, 700, 800], [1, 1, 1], (8, 2))
    b.table[1:, :32] = b.table[0, :32]  # 512 tokens shared
    plan = build_cascade_plan(b.table.cpu().numpy(), b.ctx, b.bs, b.Hq, b.H, device="cuda", chunk_tokens=128)
    return lambda: kernels.paged_attention_cascade(b.q, b.k, b.v, b.table, b.lens, b.H, b.scale, b.bs, b.max_seq, plan)


def calls():
    split, few = Batch(30, [6000, 500], [40, 9], (8, 2)), Batch(31, [7000, 90], [1, 1], (8, 2))
    long = Batch(32, [30000], [1], (4, 1), 64)
    return {"row tiles": split.extend, "window": lambda: few.window(5000, 4), "decode": lambda: decode(few),
            "long decode": lambda: decode(long), "cascade": cascade()}


@pytest.mark.parametrize("pair", [("row tiles", "window"), ("row tiles", "decode"), ("row tiles", "long decode"),
                                  ("row tiles", "cascade"), ("cascade", "window"), ("cascade", "decode")],
                         ids=" + ".join)
def test_two_threads_on_one_stream(pair):
    every = calls()
    run = [every[name] for name in pair]
    want = [f() for f in run]
    torch.cuda.synchronize()
    got = [[], []]

    def loop(i):
        for _ in range(CALLS):
            got[i].append(run[i]())

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert [len(g) for g in got] == [CALLS, CALLS]
    assert all(o.equal(w) for g, w in zip(got, want) for o in g)
