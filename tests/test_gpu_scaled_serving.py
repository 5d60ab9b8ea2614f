"""Caches with a scale per block and head as a server uses them: requests open, prefill,
go on in chunks, draft and decode; a shared block is copied with its scales; calls are
captured, come from two threads or streams, and reach past 32-bit offsets.  Outputs are
compared with attention in 64 bits over what the cache holds, and what the cache holds with
the keys and values that went in."""

import threading

import numpy as np
import pytest
import torch

import pkv_scaled as ps
from sglang_mlx_amd import _ext, kernels
from sglang_mlx_amd.srt.mem_cache import BlockAllocator, RequestBlocks

pytestmark = pytest.mark.gpu

DEV = "cuda"
Hq, H, D, BS = 8, 2, 64, 16
SCALE = D ** -0.5


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def caches(nb, h=H, d=D, bs=BS):
    """Full of NaN codes and of scales that no store wrote."""
    return (torch.full((nb, h, d // 16, bs, 16), 0x7f, dtype=torch.uint8, device=DEV),
            torch.full((nb, h, d, bs), 0x7f, dtype=torch.uint8, device=DEV),
            torch.full((nb, h, 2), float("nan"), device=DEV))


def close(got, q, k, v, first, window=0, sinks=0):
    want, off = ps.attend(q, k, v, first, SCALE, window, sinks)
    worst = ((got.double() - want).abs() - off).max()
    assert worst <= 0, float(worst)


def stored(got, x, scale):
    """A code is half a step from its value (2^-4 of it).  Where a scale grows, a code that becomes subnormal is
    rounded again, by half a subnormal step (2^-10 of that scale): over all growths less than 2^-9 of the last scale,
    the first storing's own subnormal rounding among them."""
    x = x.double()
    assert ((got - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -9 * scale).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 5)])
def test_prefill_chunks_drafts_and_decode(dtype, window, sinks):
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    nb = 90
    kc, vc, scales = caches(nb)
    rb = RequestBlocks(6, 24, BS, BlockAllocator(nb), DEV)
    history = {}

    def step(rows, new, pad_seqs=0, pad_tokens=0):
        n = sum(new)
        fresh = all(rb.num_tokens(r) == 0 for r in rows)
        st = rb.step(rows, new, len(rows) + pad_seqs, n + pad_tokens)
        qkv = torch.empty((n + pad_tokens, (Hq + 2 * H) * D), device=DEV).normal_(generator=g)
        qkv *= 2.0 ** torch.empty((n + pad_tokens, 1), device=DEV).uniform_(-2, 2, generator=g)  # (scales grow)
        qkv = qkv.to(dtype)
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, H * D, H * D], 1))
        kernels.quantize_and_cache(k, v, kc, vc, scales, st.block_tables, st.context_lens, st.query_start_loc)
        ctx = [rb.num_tokens(r) for r in rows]
        if fresh:
            out = kernels.prompt_attention(q, k, v, st.query_start_loc, SCALE, st.max_query_len, window=window,
                                           num_sinks=sinks)
        elif st.max_query_len > 8:
            total = sum(ctx)
            loc = ints(np.concatenate([[0], np.cumsum(ctx + [0] * pad_seqs)]))
            ck, cv = kernels.dequantize_cache(kc, vc, scales, st.block_tables, loc, total + 3, dtype)
            assert (ck[total:] == 0).all() and (cv[total:] == 0).all()
            out = kernels.prompt_attention(q, ck, cv, st.query_start_loc, SCALE, st.max_query_len, loc,
                                           st.max_seq_len, window, sinks)
        else:
            single = max(new) == 1 and pad_tokens == pad_seqs == 0
            out = kernels.paged_attention_scaled(q, kc, vc, scales, st.block_tables, st.context_lens,
                                                 None if single else st.query_start_loc, H, SCALE, BS, st.max_seq_len,
                                                 st.max_query_len, window, sinks)
        at = key_at = 0
        for i, (r, m) in enumerate(zip(rows, new)):
            hk, hv = history.get(r, (k[:0], v[:0]))
            history[r] = hk, hv = torch.cat([hk, k[at:at + m]]), torch.cat([hv, v[at:at + m]])
            T = hk.shape[0]
            assert T == ctx[i]
            got_k, got_v = ps.rows_of(kc, vc, scales, st.block_tables[i], 0, T)
            of = scales[st.block_tables[i].long()[torch.arange(T, device=DEV) // BS]].double()
            stored(got_k, hk, of[:, :, :1])
            stored(got_v, hv, of[:, :, 1:])
            if fresh:
                got_k, got_v = hk.double(), hv.double()
            elif st.max_query_len > 8:
                # 4 significant bits times a power of two: nothing is rounded on the way back.
                assert torch.equal(ck[key_at:key_at + T].double(), got_k)
                assert torch.equal(cv[key_at:key_at + T].double(), got_v)
            close(out[at:at + m], q[at:at + m], got_k, got_v, T - m, window, sinks)
            at, key_at = at + m, key_at + T
        assert (out[at:] == 0).all()

    a, b, c = (rb.open() for _ in range(3))
    step([a, b, c], [70, 1, 33], 2, 9)      # prompts
    step([a, c], [100, 47], 1, 5)           # their next chunks
    step([c, b, a], [1, 1, 1])              # single tokens
    step([a, b, c], [4, 3, 5])              # drafted ones
    step([b, a], [1, 4], 3, 11)             # both, padded
    rb.close(a), history.pop(a)
    d = rb.open()                           # on blocks that others wrote
    step([d], [17])
    step([d, b, c], [31, 20, 60], 0, 1)     # chunks of sequences that begin inside a block
    for _ in range(4):
        step([b, c, d], [1, 1, 1])


def test_a_shared_block_is_copied_with_its_scales():
    """Two sequences go on from one half-full block, each in its own copy."""
    g = torch.Generator(device=DEV)
    g.manual_seed(6)
    kc, vc, scales = caches(4)
    rows = lambda n, gain: torch.empty((n, H, D), device=DEV).normal_(generator=g).mul_(gain).bfloat16()  # noqa: E731
    k, v = rows(25, 1.0), rows(25, 0.1)
    kernels.quantize_and_cache(k, v, kc, vc, scales, ints([[0, 1]]), ints([25]), ints([0, 25]))
    mapping = torch.tensor([[1, 2]], device=DEV)
    kernels.copy_blocks([kc], [vc], mapping)
    assert kernels.swap_blocks(scales, scales, mapping) is scales
    assert torch.equal(scales[1], scales[2]) and torch.equal(kc[1], kc[2]) and torch.equal(vc[1], vc[2])
    before = [t[2].clone() for t in (kc, vc, scales)]
    table = ints([[0, 1], [0, 2]])
    k1, v1 = rows(1, 8.0), rows(1, 0.01)
    kernels.quantize_and_cache(k1, v1, kc, vc, scales, table[:1], ints([26]), ints([0, 1]))
    assert all(torch.equal(a, b[2]) for a, b in zip(before, (kc, vc, scales)))
    k2, v2 = rows(2, 0.5), rows(2, 20.0)
    kernels.quantize_and_cache(k2, v2, kc, vc, scales, table[1:].contiguous(), ints([27]), ints([0, 2]))
    q = rows(2, 1.0).repeat(1, Hq // H, 1)
    out = kernels.paged_attention_scaled(q, kc, vc, scales, table, ints([26, 27]), None, H, SCALE, BS, 32)
    for i, (x, y) in enumerate([(k1, v1), (k2, v2)]):
        T = 25 + x.shape[0]
        gk, gv = ps.rows_of(kc, vc, scales, table[i], 0, T)
        of = scales[table[i].long()[torch.arange(T, device=DEV) // BS]].double()
        stored(gk, torch.cat([k, x]), of[:, :, :1])
        stored(gv, torch.cat([v, y]), of[:, :, 1:])
        close(out[i:i + 1], q[i:i + 1], gk, gv, T - 1)


def test_a_captured_step_serves_other_lengths():
    """Store, read and both attentions in one graph; before each replay lengths, tables and rows change."""
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    B, N, W, nb = 3, 12, 6, 24
    table = torch.randperm(nb, generator=torch.Generator().manual_seed(1))[:B * W].view(B, W).int().to(DEV)
    qkv = torch.empty((N, (Hq + 2 * H) * D), device=DEV, dtype=torch.bfloat16)
    lens, loc, key_loc = ints([20, 30, 5]), ints([0, 4, 8, 12]), ints([0, 20, 50, 55])
    total = B * W * BS

    def step(kc, vc, scales):
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, H * D, H * D], 1))
        kernels.quantize_and_cache(k, v, kc, vc, scales, table, lens, loc)
        ck, cv = kernels.dequantize_cache(kc, vc, scales, table, key_loc, total)
        return (kernels.paged_attention_scaled(q, kc, vc, scales, table, lens, loc, H, SCALE, BS, W * BS, N),
                kernels.prompt_attention(q, ck, cv, loc, SCALE, N, key_loc, W * BS), ck, cv)

    qkv.normal_(generator=g)
    mine, eager = caches(nb), caches(nb)
    for t, u in zip(mine, eager):
        t.zero_(), u.zero_()
    step(*caches(nb))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*mine)
    for ctx, new in [([20, 30, 5], [4, 4, 4]), ([24, 31, 5], [4, 1, 0]), ([25, 40, 17], [1, 9, 2]), ([96, 41, 18], [1, 1, 1])]:
        qkv.normal_(generator=g)
        lens.copy_(ints(ctx))
        loc.copy_(ints(np.concatenate([[0], np.cumsum(new)])))
        key_loc.copy_(ints(np.concatenate([[0], np.cumsum(ctx)])))
        want = step(*eager)
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) for a, b in zip(outs, want))
        assert all(torch.equal(a, b) for a, b in zip(mine, eager))


class Work:
    """Sizes that both attentions split, so that they use their workspaces."""

    def __init__(self, seed, ctx=(900, 2500, 37)):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        need = [-(-c // BS) for c in ctx]
        nb = sum(need)
        self.ctx = ctx
        self.table = torch.full((len(ctx), max(need)), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = torch.arange(at, at + n)
            at += n
        self.table = self.table.to(DEV)
        self.cache = caches(nb)
        k, v = (torch.empty((sum(ctx), H, D), device=DEV).normal_(generator=g).bfloat16() for _ in range(2))
        self.lens, self.loc = ints(ctx), ints(np.concatenate([[0], np.cumsum(ctx)]))
        kernels.quantize_and_cache(k, v, *self.cache, self.table, self.lens, self.loc)
        self.q = torch.empty((len(ctx), Hq, D), device=DEV).normal_(generator=g).bfloat16()
        self.one = ints(range(len(ctx) + 1))
        self.k, self.v = k, v

    def decode(self):
        return kernels.paged_attention_scaled(self.q, *self.cache, self.table, self.lens, None, H, SCALE, BS,
                                              self.table.shape[1] * BS)

    def prompt(self):
        return kernels.prompt_attention(self.q, self.k, self.v, self.one, SCALE, 1, self.loc, max(self.ctx))

    def read(self):
        return kernels.dequantize_cache(*self.cache, self.table, self.loc, sum(self.ctx))[0]


@pytest.mark.parametrize("own_streams", [False, True])
def test_two_threads(own_streams):
    """On one stream (one workspace) and on one each."""
    works = [Work(11), Work(12, (3000, 64, 1200, 1))]
    want = [(w.decode(), w.prompt(), w.read()) for w in works]
    torch.cuda.synchronize()
    bad = []

    def run(w, expect):
        stream = torch.cuda.Stream() if own_streams else torch.cuda.current_stream()
        with torch.cuda.stream(stream):
            got = [(w.decode(), w.prompt(), w.read()) for _ in range(30)]
            stream.synchronize()
            if not all(torch.equal(a, b) for x in got for a, b in zip(x, expect)):
                bad.append(w)

    threads = [threading.Thread(target=run, args=a) for a in zip(works, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_two_graphs_and_eager_calls_share_a_workspace():
    """Captured from one stream after its buffer grew, replayed in turn with eager calls between."""
    works = [Work(13), Work(14, (5000, 400))]
    want = [(w.decode(), w.prompt()) for w in works]
    torch.cuda.synchronize()
    graphs = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for w in works:
            w.decode(), w.prompt()
        side.synchronize()
        for w in works:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs = w.decode(), w.prompt()
            graphs.append((graph, outs))
        for i in (0, 1, 1, 0, 1, 0):
            for t in graphs[i][1]:
                t.fill_(7.0)
            graphs[i][0].replay()
            eager = works[1 - i].decode(), works[1 - i].prompt()
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want[i]))
            assert all(torch.equal(a, b) for a, b in zip(eager, want[1 - i]))


def test_python_path_gives_the_same(monkeypatch):
    w = Work(15)
    new = 3
    k, v = w.k[:new * len(w.ctx)], w.v[:new * len(w.ctx)]
    loc = ints(np.arange(len(w.ctx) + 1) * new)

    def everything():
        cache = [t.clone() for t in w.cache]
        out = kernels.quantize_and_cache(k, v, *cache, w.table, w.lens, loc)
        assert all(a is b for a, b in zip(out, cache))
        return [*cache, w.decode(), w.prompt(), w.read(),
                kernels.prompt_attention(w.k.repeat(1, 4, 1), w.k, w.v, w.loc, SCALE, 2500, window=700, num_sinks=3),
                kernels.paged_attention_scaled(w.k[:new * len(w.ctx)].repeat(1, 4, 1), *cache, w.table, w.lens, loc, H,
                                               SCALE, BS, w.table.shape[1] * BS, new, 100, 7)]

    native = everything()
    # (None of them went to the Python path.)
    assert _ext._native.quantize_and_cache(k, v, *[t.clone() for t in w.cache], w.table, w.lens, loc) is not None
    assert _ext._native.dequantize_cache(*w.cache, w.table, w.loc, sum(w.ctx), torch.float16) is not None
    assert _ext._native.paged_attention_scaled(_ext._ws_cache, w.q, *w.cache, w.table, w.lens, None, H, SCALE, BS, 2500,
                                               1, 0, 0) is not None
    assert _ext._native.prompt_attention(_ext._ws_cache, w.q, w.k, w.v, w.one, SCALE, 1, w.loc, 2500, 0, 0) is not None
    with monkeypatch.context() as m:
        m.setattr(_ext, "_native", None)
        python = everything()
    assert all(torch.equal(a, b) for a, b in zip(native, python))


def test_no_tokens_and_no_sequences():
    w = Work(16)
    empty = w.q[:0]
    none = ints([0])
    cache = [t.clone() for t in w.cache]
    kernels.quantize_and_cache(w.k[:0], w.v[:0], *cache, w.table, w.lens, ints([0, 0, 0, 0]))
    kernels.quantize_and_cache(w.k[:5], w.v[:5], *cache, w.table[:0], w.lens[:0], none)
    assert all(torch.equal(a, b) for a, b in zip(cache, w.cache))
    args = (H, SCALE, BS, 2512)
    assert kernels.paged_attention_scaled(empty, *w.cache, w.table[:0], w.lens[:0], None, *args).shape == (0, Hq, D)
    out = kernels.paged_attention_scaled(w.q, *w.cache, w.table[:0], w.lens[:0], none, *args, 3)
    assert out.shape == w.q.shape and (out == 0).all()
    assert kernels.prompt_attention(empty, w.k[:0], w.v[:0], none, SCALE, 1).shape == (0, Hq, D)
    for k, loc, key_loc in ((w.k, none, none), (w.k[:0], w.one, ints([0, 0, 0, 0]))):
        out = kernels.prompt_attention(w.q, k, k, loc, SCALE, 1, key_loc, 5)
        assert out.shape == w.q.shape and (out == 0).all()


def test_starts_that_decrease_reach_nothing_else():
    """No call may have them; what they name is then unspecified, and nothing outside it is written."""
    nb, n = 40, 400
    guard = 1 << 16
    sizes = [nb * H * D * BS] * 2
    whole = [torch.full((size + 2 * guard,), 0x55, dtype=torch.uint8, device=DEV) for size in sizes]
    kc = whole[0][guard:-guard].view(nb, H, D // 16, BS, 16)
    vc = whole[1][guard:-guard].view(nb, H, D, BS)
    scales = torch.ones((nb, H, 2), device=DEV)
    table = torch.arange(5 * 6, device=DEV).int().view(5, 6)  # blocks 30 .. 39 stand in no table
    k = torch.ones((n, H, D), device=DEV, dtype=torch.bfloat16)
    q = torch.ones((n, Hq, D), device=DEV, dtype=torch.bfloat16)
    lens = ints([90, 60, 80, 96, 33])
    for starts in ([0, 300, 100, 250, 20, 200], [399, 350, 300, 200, 100, 0], [50, -7, 1000, 3, 2, 1]):
        loc = ints(starts)
        kernels.quantize_and_cache(k, k, kc, vc, scales, table, lens, loc)
        ck, cv = kernels.dequantize_cache(kc, vc, scales, table, loc, n)
        assert ck.shape == cv.shape == (n, H, D)
        assert kernels.paged_attention_scaled(q, kc, vc, scales, table, lens, loc, H, SCALE, BS, 96, 300).shape == q.shape
        assert kernels.prompt_attention(q, k, k, loc, SCALE, 300).shape == q.shape
        assert kernels.prompt_attention(q, k, k, ints([0, 90, 150, 230, 326, 359]), SCALE, 96, loc, 300).shape == q.shape
    torch.cuda.synchronize()
    for t, cache in zip(whole, (kc, vc)):
        assert (t[:guard] == 0x55).all() and (t[-guard:] == 0x55).all() and (cache[30:] == 0x55).all()
    assert (scales[30:] == 1).all()


def test_caches_past_32_bit_offsets():
    """Blocks whose bytes lie beyond 2^32, of caches and of scales' table rows."""
    nb, h, d = 300000, 8, 128  # 4.9 GB of K and of V
    kc = torch.zeros((nb, h, d // 16, BS, 16), dtype=torch.uint8, device=DEV)
    vc = torch.zeros((nb, h, d, BS), dtype=torch.uint8, device=DEV)
    scales = torch.zeros((nb, h, 2), device=DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(17)
    ctx = [100, 33]
    table = ints([[nb - 1, 5, nb - 40, 262144, 262143, nb - 2, 131072], [nb - 3, 7, nb - 4, -1, -1, -1, -1]])
    k, v = (torch.empty((sum(ctx), h, d), device=DEV).normal_(generator=g).bfloat16() for _ in range(2))
    loc = ints([0, 100, 133])
    kernels.quantize_and_cache(k, v, kc, vc, scales, table, ints(ctx), loc)
    q = torch.empty((2, 32, d), device=DEV).normal_(generator=g).bfloat16()
    out = kernels.paged_attention_scaled(q, kc, vc, scales, table, ints(ctx), None, h, SCALE, BS, 112)
    ck, cv = kernels.dequantize_cache(kc, vc, scales, table, loc, 133, torch.float32)
    for i, (a, n) in enumerate(zip((0, 100), ctx)):
        gk, gv = ps.rows_of(kc, vc, scales, table[i], 0, n)
        of = scales[table[i].long()[torch.arange(n, device=DEV) // BS]].double()
        stored(gk, k[a:a + n], of[:, :, :1])
        stored(gv, v[a:a + n], of[:, :, 1:])
        assert torch.equal(ck[a:a + n].double(), gk) and torch.equal(cv[a:a + n].double(), gv)
        close(out[i:i + 1], q[i:i + 1], gk, gv, n - 1)


def test_rows_past_32_bit_offsets():
    """Prompts whose queries and keys lie beyond 2^31 elements of the tensors that hold them."""
    n, d, hq = 1 << 17, 128, 120
    g = torch.Generator(device=DEV)
    g.manual_seed(18)
    width = (hq + 2 * 8) * d  # 17408 elements a row, 2^31.08 in all
    qkv = torch.empty((n, width), device=DEV, dtype=torch.bfloat16)
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, 8 * d, 8 * d], 1))
    some = [slice(0, 64), slice(123392, 123456), slice(n - 64, n)]
    qkv.zero_()
    for s in some:
        qkv[s] = torch.empty((64, width), device=DEV).normal_(generator=g).bfloat16()
    out = kernels.prompt_attention(q, k, v, ints(np.arange(0, n + 1, 64)), SCALE, 64)
    for s in some:
        close(out[s], q[s], k[s].double(), v[s].double(), 0)
    assert (out[64:123392] == 0).all()
