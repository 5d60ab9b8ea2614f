"""build_step_tables against the same rules in NumPy, bit for bit: empty and
padded batches, no new tokens, blocks that run out, contexts that end at and
inside a block, rows that are outside the table, more tokens than listed, the
largest batch; and RequestBlocks' steps against BlockTable's slots."""

import numpy as np
import pytest
import torch

from sglang_mlx_amd import kernels
from sglang_mlx_amd.srt.mem_cache import BlockAllocator, BlockTable, RequestBlocks

pytestmark = pytest.mark.gpu


def reference(pool, rows, ctx, new, fresh, bs, num_tokens):
    pool = pool.copy()
    R, W = pool.shape
    B = len(rows)
    tables = np.full((B, W), -1, dtype=np.int64)
    slots, pos = np.full(num_tokens, -1, dtype=np.int64), np.zeros(num_tokens, dtype=np.int64)
    start, taken = [0], 0
    for s in range(B):
        c = int(ctx[s])
        if not 0 <= rows[s] < R or c <= 0 or c > W * bs:
            c = 0
        n = min(max(int(new[s]), 0), c)
        have, need = -(-(c - n) // bs), -(-c // bs)
        ids = list(pool[rows[s], :have]) if c else []
        for _ in range(have, need):
            ids.append(int(fresh[taken]) if taken < len(fresh) else -1)
            taken += 1
        tables[s, :need] = ids
        if need > have:
            pool[rows[s], have:need] = ids[have:]
        for i in range(n):
            t, p = start[-1] + i, c - n + i
            if t < num_tokens:
                pos[t] = p
                slots[t] = ids[p // bs] * bs + p % bs if ids[p // bs] >= 0 else -1
        start.append(start[-1] + n)
    return tables, slots, pos, np.array(start), pool


def run(pool, rows, ctx, new, fresh, bs, num_tokens, dtype=torch.int32):
    dev = lambda a, dt=dtype: torch.from_numpy(np.asarray(a, dtype=np.int64)).to(dt).cuda()
    p = dev(pool, torch.int32)
    out = kernels.build_step_tables(p, dev(rows), dev(ctx), dev(new), dev(fresh), bs, num_tokens)
    return [t.cpu().numpy().astype(np.int64) for t in (*out, p)]


def check(*args, **kw):
    for name, a, b in zip(("tables", "slots", "positions", "start", "pool"), run(*args, **kw), reference(*args)):
        assert np.array_equal(a, b), name


def random_case(seed, B, bs, lo, hi, new_hi, pad=0, short=0):
    rng = np.random.default_rng(seed)
    W = -(-hi // bs) + 1
    R = B + 5
    ctx = rng.integers(lo, hi + 1, B)
    new = np.minimum(rng.integers(0, new_hi + 1, B), ctx)
    pool = np.full((R, W), -1)
    rows = rng.permutation(R)[:B]
    ids = rng.permutation(int((-(-ctx // bs)).sum()) + 10) + 1
    at = 0
    for r, c, n in zip(rows, ctx, new):
        h = -(-(c - n) // bs)
        pool[r, :h] = ids[at:at + h]
        at += h
    count = int((-(-ctx // bs)).sum()) - at
    fresh = ids[at:at + max(count - short, 0)]
    rows = np.concatenate([rows, np.full(pad, -1)])
    ctx, new = (np.concatenate([a, np.zeros(pad, dtype=np.int64)]) for a in (ctx, new))
    return pool, rows, ctx, new, fresh, bs, int(new.sum()) + 3 * pad


@pytest.mark.parametrize("args", [
    dict(B=1, bs=16, lo=1, hi=1, new_hi=1), dict(B=1, bs=16, lo=5000, hi=5000, new_hi=4999),
    dict(B=64, bs=16, lo=1, hi=4096, new_hi=1), dict(B=37, bs=8, lo=0, hi=300, new_hi=200, pad=11),
    dict(B=211, bs=32, lo=0, hi=2000, new_hi=90, short=40), dict(B=257, bs=1, lo=1, hi=60, new_hi=60),
    dict(B=33, bs=100, lo=1, hi=999, new_hi=300, pad=1), dict(B=4096, bs=16, lo=1, hi=100, new_hi=7),
    dict(B=3000, bs=16, lo=1, hi=40, new_hi=1, pad=1000),
])
@pytest.mark.parametrize("seed", [1, 2])
def test_against_numpy(seed, args):
    check(*random_case(seed, **args))


def test_odd_batches():
    pool = np.arange(1, 13).reshape(3, 4)
    # No sequences; no tokens listed; fewer tokens listed than there are.
    check(pool, [], [], [], [], 16, 5)
    check(pool, [], [], [], [5], 16, 0)
    check(pool, [1, 0], [40, 20], [9, 20], [50, 51], 16, 0)
    check(pool, [1, 0], [40, 20], [9, 20], [50, 51], 16, 11)
    # Rows outside the table, contexts beyond it, negative lengths, more new tokens than context.
    check(pool, [3, -5, 2, 0, 1], [9, 9, 65, -4, 7], [1, 1, 5, 2, 99], [50, 51], 16, 12)
    # A context that fills the table; block ids of which slots leave 32 bits.
    check(pool, [1], [64], [64], [50, 51, 52, 53], 16, 64)
    out = run(np.full((1, 2), -1), [0], [32], [32], [1, 1 << 28], 16, 32)
    assert out[1][:16].tolist() == list(range(16, 32)) and (out[1][16:] == -1).all()


def test_index_types_and_strides():
    args = random_case(3, B=20, bs=16, lo=1, hi=200, new_hi=30)
    check(*args, dtype=torch.int64)
    pool, rows, ctx, new, fresh, bs, n = args
    both = torch.tensor(np.stack([ctx, new], 1), dtype=torch.int32).cuda()
    p = torch.tensor(pool, dtype=torch.int32).cuda()
    out = kernels.build_step_tables(p, torch.tensor(rows, dtype=torch.int32).cuda(), both[:, 0], both[:, 1],
                                    torch.tensor(fresh, dtype=torch.int32).cuda(), bs, n)
    ref = reference(*args)
    for a, b in zip((*out, p), ref):
        assert np.array_equal(a.cpu().numpy(), b)


def test_step_again_is_the_same():
    pool, rows, ctx, new, fresh, bs, n = random_case(4, B=50, bs=16, lo=1, hi=500, new_hi=100)
    first = run(pool, rows, ctx, new, fresh, bs, n)
    second = run(first[4], rows, ctx, new, fresh, bs, n)
    for a, b in zip(first, second):
        assert np.array_equal(a, b)


def test_captured_step_replays_with_new_lengths():
    dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32).cuda()
    cases = [random_case(s, B=24, bs=16, lo=1, hi=300, new_hi=20) for s in (5, 6, 7)]
    width = max(c[0].shape[1] for c in cases)
    n = max(c[6] for c in cases) + 5
    pool, rows, ctx, new, fresh = (dev(np.zeros(s)) for s in ((29, width), 24, 24, 24, 2000))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        kernels.build_step_tables(pool, rows, ctx, new, fresh, 16, n)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = kernels.build_step_tables(pool, rows, ctx, new, fresh, 16, n)
    for c in cases + cases[::-1]:
        p = np.full((29, width), -1)
        p[:, :c[0].shape[1]] = c[0]
        pool.copy_(dev(p)), rows.copy_(dev(c[1])), ctx.copy_(dev(c[2])), new.copy_(dev(c[3]))
        fresh.fill_(-1)
        fresh[:len(c[4])] = dev(c[4])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*out, pool), reference(p, c[1], c[2], c[3], c[4], 16, n)):
            assert np.array_equal(a.cpu().numpy(), b)


def test_request_blocks_follow_block_tables():
    bs = 16
    alloc, twin = BlockAllocator(400), BlockAllocator(400)
    rb = RequestBlocks(8, 20, bs, alloc, "cuda")
    rng = np.random.default_rng(8)
    open_rows, host = [], {}
    for step in range(12):
        if len(open_rows) < 6:
            r = rb.open()
            open_rows.append(r)
            host[r] = BlockTable(bs)
        if step in (5, 9):
            gone = open_rows.pop(0)
            rb.close(gone)
            host.pop(gone).release(twin)
        batch = [r for r in open_rows if rng.random() < 0.8] or open_rows[:1]
        new = [int(min(rng.integers(0, 40), 320 - rb.num_tokens(r))) for r in batch]
        st = rb.step(batch, new, num_seqs=8, num_tokens=sum(new) + 4)
        # The same blocks in the same order from a second allocator's one call per step.
        need = [-(-(host[r].num_tokens + n) // bs) - len(host[r].blocks) for r, n in zip(batch, new)]
        ids = twin.alloc(sum(need))
        slots = []
        for r, n, k in zip(batch, new, need):
            t = host[r]
            t.blocks += ids[:k]
            ids = ids[k:]
            p = np.arange(t.num_tokens, t.num_tokens + n)
            slots += (np.array(t.blocks, dtype=np.int64)[p // bs] * bs + p % bs).tolist() if n else []
            t.num_tokens += n
            assert rb.blocks(r) == t.blocks and rb.num_tokens(r) == t.num_tokens
        assert st.slot_mapping.tolist() == slots + [-1] * 4
        assert st.context_lens.tolist() == [host[r].num_tokens for r in batch] + [0] * (8 - len(batch))
        table = st.block_tables.cpu().numpy()
        for i, r in enumerate(batch):
            k = len(host[r].blocks)
            assert table[i, :k].tolist() == host[r].blocks and (table[i, k:] == -1).all()
        assert (table[len(batch):] == -1).all()
        assert st.query_start_loc.tolist() == np.cumsum([0] + new + [0] * (8 - len(batch))).tolist()
        assert st.max_query_len == max(new + [1])
    for r in open_rows:
        rb.close(r)
    assert alloc.available_size == 399
