"""paged_attention_window and paged_attention_extend against the formula in 64
bits, row by row.

Bound of a row's element, with weights p (sum 1) and u half a step of the
queries' type: weights are rounded to that type, u sum p |v| (float16: and half
its smallest subnormal, 2^-25, each); the output is rounded, u |o|; a score is
off by at most (D + 4) 2^-24 scale sum |q k| in float32, which its weight and the
sum of weights take relatively, twice; the exponential, sums over T keys and the
splits' factors add at most (T + 64) 2^-23 sum p |v|.  The expected values
themselves are exact to 2^-50."""

import threading

import numpy as np
import pytest
import torch

from sglang_mlx_amd import kernels

pytestmark = pytest.mark.gpu

BF, HF, U8 = torch.bfloat16, torch.float16, torch.uint8
K_SCALE, V_SCALE = 0.05, 0.02


def code_values():
    c = torch.arange(256)
    e, m = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e.double() - 7))
    return torch.where(c >= 128, -mag, mag)


class Batch:
    """Sequences of `ctx` tokens, the last `new` of them queries, over a paged cache."""

    def __init__(self, seed, ctx, new, heads=(8, 2), D=128, bs=16, q=BF, cache=None, gain=2.0, spread=1):
        self.ctx, self.new, self.bs, self.D = list(ctx), list(new), bs, D
        self.Hq, self.H = heads
        cache = cache or q
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rng = np.random.default_rng(seed)
        need = [-(-max(c, 0) // bs) for c in ctx]
        nb = sum(need) + 3
        ids = rng.permutation(nb - 1)[:sum(need)] + 1
        table = np.full((len(ctx), max(need + [1]) + 1), -1)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = ids[at:at + n]
            at += n
        x = 16 if cache == U8 else 8
        shapes = (spread * nb, self.H, D // x, bs, x), (spread * nb, self.H, D, bs)
        if cache == U8:
            self.k, self.v = (torch.empty(s, device="cuda").normal_(generator=g).mul_(20).clamp_(-240, 240)
                              .to(torch.float8_e4m3fn).view(U8) for s in shapes)
        else:
            self.k, self.v = (torch.empty(s, device="cuda").normal_(generator=g).to(cache) for s in shapes)
        self.k, self.v = self.k[::spread], self.v[::spread]
        n = sum(new)
        self.q = torch.empty((n, self.Hq, D), device="cuda").normal_(generator=g).mul_(gain).to(q)
        self.table = torch.tensor(table, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor(ctx, dtype=torch.int32, device="cuda")
        self.start = torch.tensor(np.cumsum([0] + list(new)), dtype=torch.int32, device="cuda")
        self.scale = D ** -0.5
        self.scales = dict(k_scale=K_SCALE, v_scale=V_SCALE) if cache == U8 else {}
        self.max_seq, self.max_query = max(list(ctx) + [1]), max(list(new) + [1])

    def extend(self, window=0, sinks=0, **kw):
        a = dict(max_seq_len=min(self.max_seq, self.table.shape[1] * self.bs), max_query_len=self.max_query)
        a.update(kw)
        return kernels.paged_attention_extend(self.q, self.k, self.v, self.table, self.lens, self.start, self.H,
                                              self.scale, self.bs, a["max_seq_len"], a["max_query_len"], window, sinks,
                                              **self.scales)

    def window(self, window, sinks=0):
        return kernels.paged_attention_window(self.q, self.k, self.v, self.table, self.lens, self.H, self.scale,
                                              self.bs, self.max_seq, window, sinks, **self.scales)

    def expected(self, window=0, sinks=0):
        """(value, bound) of every row; zero rows where nothing is seen."""
        values = code_values().cuda() if self.k.dtype == U8 else None
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        group, D, at = self.Hq // self.H, self.D, 0
        u = torch.finfo(self.q.dtype).eps / 2
        for i, (c, n) in enumerate(zip(self.ctx, self.new)):
            if n and c > 0:
                t = torch.arange(c, device="cuda")
                ids = self.table[i].long()[t // self.bs]
                real = (ids >= 0) & (ids < self.k.shape[0])
                ids = ids.clamp(0, self.k.shape[0] - 1)
                k = self.k[ids, :, :, t % self.bs, :].reshape(c, self.H, D)
                v = self.v[ids, :, :, t % self.bs]
                k, v = (values[k.long()] * K_SCALE, values[v.long()] * V_SCALE) if values is not None else (
                    k.double(), v.double())
                pos = torch.arange(c - n, c, device="cuda")[:, None]
                sees = (t <= pos) & real
                if window:
                    sees &= (t > pos - window) | (t < sinks)
                for h in range(self.Hq):
                    kh, vh, q = k[:, h // group], v[:, h // group], self.q[at:at + n, h].double()
                    # (Keys and values that a row does not see take no part, whatever they hold.)
                    s = q @ kh.nan_to_num(0, 0, 0).t().contiguous() * self.scale
                    s = torch.where(torch.isfinite(kh).all(1), s, float("nan")).masked_fill(~sees, float("-inf"))
                    p = torch.softmax(s, -1).masked_fill(~sees, 0.0)
                    p = p.masked_fill(~sees.any(-1, keepdim=True), 0.0)
                    clean = vh.nan_to_num(0, 0, 0)
                    o = p @ clean
                    dirty = (~torch.isfinite(vh)).any(1)
                    hit = (sees & dirty).any(-1)
                    size = p @ clean.abs()
                    score = ((q.abs() @ kh.nan_to_num(0, 0, 0).abs().t().contiguous()) * abs(self.scale)).masked_fill(
                        ~sees, 0.0).amax(-1, keepdim=True)
                    b = u * (size * 1.02 + o.abs()) + size * (4 * (D + 4) * 2.0 ** -24 * score + (c + 64) * 2.0 ** -23)
                    if self.q.dtype == HF:
                        b = b + 2.0 ** -25 * (sees.double() @ clean.abs() + 1)
                    out[at:at + n, h] = torch.where(hit[:, None], float("nan"), o)
                    bound[at:at + n, h] = b + 2.0 ** -130
            at += n
        return out, bound

    def check(self, got, window=0, sinks=0):
        want, bound = self.expected(window, sinks)
        assert got.shape == self.q.shape and got.dtype == self.q.dtype and got.is_contiguous()
        fine = torch.isfinite(want).all(-1)
        d = (got.double() - want).abs()
        assert (d[fine] <= bound[fine]).all(), ((d[fine] - bound[fine]).max().item(), d[fine].max().item())
        assert torch.isfinite(got[fine]).all()


TYPES = [(BF, BF), (HF, HF), (BF, U8), (HF, U8)]


@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{str(t[0])[6:]}-{str(t[1])[6:]}")
@pytest.mark.parametrize("D", [32, 64, 80, 96, 112, 120, 128, 192, 256])
def test_head_sizes_and_types(types, D):
    if D == 120 and types[1] == U8:
        pytest.skip("FP8 caches take head sizes that 16 divides")
    for bs in (8, 16, 32):
        b = Batch(D + bs, [1, 77, 200, 31], [1, 50, 3, 31], (4, 2), D, bs, *types)
        b.check(b.extend())
        b.check(b.extend(20, 5), 20, 5)
        b = Batch(D + bs + 1, [1, 5, 77, 300], [1] * 4, (4, 2), D, bs, *types)
        b.check(b.window(33, 3), 33, 3)
        b.check(b.extend())


@pytest.mark.parametrize("heads", [(1, 1), (32, 8), (28, 4), (6, 6), (16, 1), (20, 1), (40, 2), (9, 3), (64, 8)])
def test_head_groups(heads):
    b = Batch(1, [130, 1, 64, 65, 400], [130, 1, 33, 2, 70], heads)
    b.check(b.extend())
    b.check(b.extend(64, 4), 64, 4)
    b = Batch(2, [130, 1, 64, 65, 700], [1] * 5, heads)
    b.check(b.window(100, 4), 100, 4)
    b.check(b.extend())


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 3), (15, 0), (16, 16), (31, 1), (32, 33), (33, 64),
                                          (63, 0), (64, 65), (65, 4), (100, 500), (511, 7), (600, 0), (5000, 4)])
def test_windows_and_sinks(window, sinks):
    ctx = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 97, 128, 129, 500, 601]
    b = Batch(window, ctx, [1] * len(ctx), (4, 1), 64)
    b.check(b.window(window, sinks), window, sinks)
    b.check(b.extend(window, sinks), window, sinks)
    b = Batch(window + 1, ctx, [max(1, c - 3 * i) for i, c in enumerate(ctx)], (4, 2), 64, 8)
    b.check(b.extend(window, sinks), window, sinks)


@pytest.mark.parametrize("types", TYPES[:3], ids=lambda t: f"{str(t[0])[6:]}-{str(t[1])[6:]}")
def test_long_contexts_are_split(types):
    # Few sequences and long contexts: the length is split over workgroups and joined.
    b = Batch(3, [9000], [1], (8, 2), 128, 16, *types)
    b.check(b.window(9000))
    b.check(b.window(6000, 70), 6000, 70)
    b.check(b.extend())
    b = Batch(4, [7000, 40, 3333], [17, 40, 1], (8, 2), 128, 32, *types)
    b.check(b.extend())
    b.check(b.extend(2500, 9), 2500, 9)
    b = Batch(5, [20000, 3], [1, 1], (4, 1), 64, 8, *types)
    b.check(b.extend())


def test_rows_that_see_nothing_are_zero():
    b = Batch(6, [0, 40, 3, 90, 64], [2, 7, 5, 4, 4], (4, 2), 64)
    got = b.extend(max_seq_len=80, max_query_len=6)
    # No context; more rows than max_query_len; rows before position 0; a context beyond max_seq_len.
    want, bound = b.expected()
    for r in (range(0, 2), range(2, 9), range(9, 11), range(14, 18)):
        assert (got[list(r)] == 0).all()
    for r in (range(11, 14), range(18, 22)):
        assert ((got[list(r)].double() - want[list(r)]).abs() <= bound[list(r)]).all()
    b = Batch(7, [0, 40, 90], [1, 1, 1], (4, 2), 64)
    b.max_seq = 60
    got = b.window(10, 2)
    want, bound = b.expected(10, 2)
    assert (got[[0, 2]] == 0).all() and ((got[1].double() - want[1]).abs() <= bound[1]).all()


def test_query_ranges():
    # Sequences without queries, rows behind the last sequence, an empty batch.
    b = Batch(8, [30, 50, 0, 70], [0, 20, 0, 5], (4, 2), 64)
    b.check(b.extend())
    want, bound = b.expected()
    b.q = torch.cat([b.q, torch.full((19, 4, 64), 3.0, dtype=BF, device="cuda")])
    got = b.extend()
    assert (got[25:] == 0).all() and ((got[:25].double() - want).abs() <= bound).all()
    b = Batch(9, [30, 50, 0, 70], [0, 1, 0, 1], (4, 2), 64)
    want, bound = b.expected()
    b.q = torch.cat([b.q, torch.full((3, 4, 64), 3.0, dtype=BF, device="cuda")])
    got = b.extend()
    assert (got[2:] == 0).all() and ((got[:2].double() - want).abs() <= bound).all()
    assert b.extend(max_query_len=2).equal(got) or ((b.extend(max_query_len=2)[:2].double() - want).abs() <= bound).all()
    b = Batch(10, [], [], (4, 2), 64)
    b.q = torch.ones((5, 4, 64), dtype=BF, device="cuda")
    assert (b.extend() == 0).all() and (b.extend(max_query_len=4) == 0).all()
    b.q = b.q[:0]
    assert b.extend().shape == (0, 4, 64) and b.window(4).shape == (0, 4, 64)


def test_blocks_outside_the_pool_are_masked():
    for new in ([1, 1, 1], [60, 5, 1]):
        b = Batch(11, [100, 200, 33], new, (4, 2), 64)
        b.table[0, 2] = -1
        b.table[1, 5], b.table[1, 0] = b.k.shape[0], 2 ** 31 - 1
        b.table[2, :] = -7
        b.check(b.extend())
        b.check(b.extend(70, 9), 70, 9)
        assert (b.extend()[-1] == 0).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_unseen_tokens_do_not_reach_a_row(value):
    # What the cache holds behind the contexts.
    for new in ([1, 1], [90, 20]):
        b = Batch(12, [93, 61], new, (4, 2), 64)
        for i, c in enumerate(b.ctx):
            last = b.table[i, c // 16].item()
            b.k[last, :, :, c % 16:, :] = value
            b.v[last, :, :, c % 16:] = value
        b.k[0], b.v[0] = value, value
        b.check(b.extend())
        b.check(b.extend(30, 2), 30, 2)
    # A token inside a context: rows before it and rows whose window has left it are clean, the others are not.
    b = Batch(13, [200], [150], (4, 2), 128)
    blk = b.table[0, 100 // 16].item()
    b.v[blk, :, 5, 100 % 16] = value
    for window, sinks in ((0, 0), (20, 0), (20, 101)):
        got = b.extend(window, sinks)
        b.check(got, window, sinks)
        tok = torch.arange(50, 200)
        hit = (tok >= 100) & ((tok < 120) | (window == 0) | (sinks > 100))
        assert (~torch.isfinite(got[..., 5].cpu())).all(1).equal(hit)
        assert torch.isfinite(got[..., torch.arange(128) != 5]).all()
    b = Batch(14, [200], [1], (4, 2), 128)
    b.v[b.table[0, 3].item(), :, :, 2] = value
    assert torch.isfinite(b.window(140)).all() and not torch.isfinite(b.window(200)).any()
    b.k[b.table[0, 3].item(), :, :, 2] = value
    assert torch.isfinite(b.window(140)).all()


def test_extreme_scores():
    # One key far above the others, all far below zero, a negative scale, equal scores.
    b = Batch(15, [150, 64], [100, 64], (4, 2), 64, gain=40.0)
    b.check(b.extend())
    b.scale = -0.125
    b.check(b.extend())
    b.k.zero_()
    b.check(b.extend(9, 1), 9, 1)
    b = Batch(16, [900], [1], (4, 2), 64, gain=40.0)
    b.check(b.window(800))
    b.q.neg_()
    b.scale = -b.scale
    b.check(b.window(800))


def test_strides():
    b = Batch(17, [80, 33, 120], [40, 1, 7], (8, 2), 64, spread=3)
    assert not b.k.is_contiguous()
    b.check(b.extend())
    wide = torch.zeros(48, 20, 64, dtype=BF, device="cuda")
    wide[:, 4:12] = b.q
    want, b.q = b.extend(), wide[:, 4:12]
    assert b.extend().equal(want)
    odd = torch.zeros(48, 8 * 64 + 3, dtype=BF, device="cuda")
    odd[:, :512] = b.q.reshape(48, 512)
    b.q = odd[:, :512].unflatten(1, (8, 64))
    assert b.extend().equal(want)
    b.lens, b.table, b.start = b.lens.long(), b.table.long(), b.start.long()
    assert b.extend().equal(want)


def test_offsets_past_32_bits():
    # A pool of which the last blocks lie more than 2^31 elements (and 2^32 bytes) in.
    bs, H, D = 32, 8, 128
    nb = 2 ** 31 // (bs * H * D) + 64
    b = Batch(18, [300, 70], [64, 1], (16, 8), D, bs)
    used = b.k.shape[0]
    k = torch.empty((nb, H, D // 8, bs, 8), dtype=BF, device="cuda")
    v = torch.empty((nb, H, D, bs), dtype=BF, device="cuda")
    k[-used:], v[-used:] = b.k, b.v
    want = b.extend()
    one = Batch(18, [300, 70], [64, 1], (16, 8), D, bs)
    one.q, one.start, one.max_query = b.q[63:65].contiguous(), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), 1
    want1 = one.extend()
    for c in (b, one):
        c.k, c.v = k, v
        c.table = torch.where(c.table >= 0, c.table + (nb - used), c.table)
    assert b.extend().equal(want) and one.extend().equal(want1)


def test_same_bits_every_time_and_with_other_work():
    b = Batch(19, [5000, 777], [1, 1], (8, 2))
    c = Batch(20, [3000, 64], [30, 64], (8, 2))
    w, e = b.window(4000, 5), c.extend()
    for _ in range(5):
        assert c.extend().equal(e) and b.window(4000, 5).equal(w)
    # The decode entry points share the scratch of the stream.
    v1 = kernels.paged_attention_v1(b.q, b.k, b.v, b.table, b.lens, b.H, b.scale, b.bs, b.max_seq)
    assert b.window(4000, 5).equal(w)
    assert kernels.paged_attention_v1(b.q, b.k, b.v, b.table, b.lens, b.H, b.scale, b.bs, b.max_seq).equal(v1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [b.window(4000, 5) for _ in range(3)]
    again = [b.window(4000, 5) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(o.equal(w) for o in outs + again)


def test_whole_windows_agree_with_the_decode():
    b = Batch(21, [1000, 64, 3], [1, 1, 1], (8, 2))
    v1 = kernels.paged_attention_v1(b.q, b.k, b.v, b.table, b.lens, b.H, b.scale, b.bs, b.max_seq)
    want, bound = b.expected()
    for got in (b.window(1000), b.window(10 ** 9, 10 ** 9), b.extend(), b.extend(max_query_len=3)):
        assert ((got.double() - want).abs() <= bound).all()
        assert (got.double() - v1.double()).abs().max() <= 2 * bound.max()


def test_captured_replays():
    # Two graphs on one stream, replayed in turn with eager calls between, each with its own lengths.
    a = Batch(22, [3000, 900], [1, 1], (8, 2))
    b = Batch(23, [2500, 64], [20, 64], (8, 2))
    wa, wb = a.window(2000, 4), b.extend()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for call in (lambda: a.window(2000, 4), lambda: b.extend()):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(call())
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[0].replay()
            graphs[1].replay()
            graphs[0].replay()
        stream.synchronize()
        assert outs[0].equal(wa) and outs[1].equal(wb)
        assert a.window(2000, 4).equal(wa) and b.extend().equal(wb)
    # Shorter contexts in the same buffers.
    a.lens.fill_(70)
    a.ctx = [70, 70]
    torch.cuda.synchronize()
    graphs[0].replay()
    torch.cuda.synchronize()
    a.check(outs[0], 2000, 4)


def test_two_threads_on_one_stream():
    # Both calls split their row tiles and use the stream's one scratch.
    batches = [Batch(24, [5000], [40], (8, 2)), Batch(25, [4000, 1000], [33, 17], (8, 2))]
    want = [b.extend() for b in batches]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        for _ in range(100):
            got[i].append(batches[i].extend())

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert [len(g) for g in got] == [100, 100]
    assert all(o.equal(w) for g, w in zip(got, want) for o in g)


def test_windows_beyond_32_bits_see_the_whole_context():
    b = Batch(26, [300, 20], [1, 1], (8, 2))
    whole = b.window(300)
    assert b.window((1 << 32) + 5).equal(whole) and b.window(10 ** 20, 10 ** 20).equal(whole)
    e = Batch(27, [300, 90], [33, 9], (8, 2))
    whole = e.extend()
    for kw in (dict(window=(1 << 32) + 5), dict(window=300, sinks=(1 << 32) + 1), dict(max_query_len=(1 << 32) + 2)):
        assert e.extend(**kw).equal(whole)
