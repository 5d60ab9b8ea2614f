"""paged_attention_scaled against attention in 64 bits over code * scale."""

import numpy as np
import pytest
import torch

import pkv_scaled as ps
from sglang_mlx_amd import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"


class Case:
    """Sequences of `ctx` tokens with `new` query tokens each over one pool of scaled caches."""

    def __init__(self, seed, dtype, Hq, H, D, bs, ctx, new, powers=True, wide=6):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        rng = np.random.default_rng(seed)
        need = [-(-c // bs) for c in ctx]
        nb = sum(need) + 2
        ids = rng.permutation(nb)
        table = np.full((len(ctx), max(need + [1])), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = ids[at:at + n]
            at += n
        x = torch.randn((nb, H, D // 16, bs, 16), generator=g, device=DEV).mul_(60).clamp_(-240, 240)
        self.kc = x.to(torch.float8_e4m3fn).view(torch.uint8)
        x = torch.randn((nb, H, D, bs), generator=g, device=DEV).mul_(60).clamp_(-240, 240)
        self.vc = x.to(torch.float8_e4m3fn).view(torch.uint8)
        self.scales = torch.empty((nb, H, 2), device=DEV)
        self.scales[..., 0] = 2.0 ** torch.randint(-8, -5, (nb, H), generator=g, device=DEV)
        self.scales[..., 1] = 2.0 ** torch.randint(-6 - wide, -6 + wide, (nb, H), generator=g, device=DEV)
        if not powers:
            self.scales *= torch.rand((nb, H, 2), generator=g, device=DEV) + 0.5
        self.table = torch.from_numpy(table).to(DEV)
        self.ctx, self.new, self.bs, self.H = list(ctx), list(new), bs, H
        self.query = (torch.randn((sum(new), Hq, D), generator=g, device=DEV) * 1.5).to(dtype)
        self.scale = D ** -0.5

    def call(self, window=0, sinks=0, start=True, pad=0, max_seq_len=None, max_query_len=None, query=None):
        lens = torch.tensor(self.ctx, dtype=torch.int32, device=DEV)
        loc = None
        if start:
            loc = torch.tensor(np.concatenate([[0], np.cumsum(self.new)]), dtype=torch.int32, device=DEV)
        q = self.query if query is None else query
        if pad:
            q = torch.cat([q, q.new_full((pad,) + q.shape[1:], float("nan"))])
        return kernels.paged_attention_scaled(
            q, self.kc, self.vc, self.scales, self.table, lens, loc, self.H, self.scale, self.bs,
            self.table.shape[1] * self.bs if max_seq_len is None else max_seq_len,
            max(self.new + [1]) if max_query_len is None else max_query_len, window, sinks)

    def check(self, out, window=0, sinks=0, skip=()):
        at = 0
        assert out.dtype == self.query.dtype
        for i, (c, n) in enumerate(zip(self.ctx, self.new)):
            got = out[at:at + n].double()
            if n and (c == 0 or i in skip):
                assert (got == 0).all()
            elif n:
                k, v = ps.rows_of(self.kc, self.vc, self.scales, self.table[i], 0, c)
                want, off = ps.attend(self.query[at:at + n], k, v, c - n, self.scale, window, sinks)
                worst = ((got - want).abs() - off).max()
                assert worst <= 0, (i, c, n, float(worst))
            at += n
        assert (out[at:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,bs", [(128, 16), (32, 8), (64, 32), (80, 16), (96, 8), (112, 32), (128, 8), (192, 16),
                                  (256, 32), (256, 8)])
def test_single_tokens(dtype, D, bs):
    """Lengths around tile and block ends, from one token on, short and long together."""
    ctx = [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 129, 500, 1023]
    c = Case(D + bs, dtype, 8, 2, D, bs, ctx, [1] * len(ctx))
    c.check(c.call(start=False))
    c.check(c.call(start=True, pad=3))


@pytest.mark.parametrize("Hq,H", [(1, 1), (4, 4), (7, 1), (32, 2), (28, 4), (40, 1), (64, 8)])
def test_head_layouts(Hq, H):
    """One query head to a KV head, up to more than 16 (several row groups)."""
    ctx = [300, 1, 77, 2000]
    c = Case(Hq, torch.bfloat16, Hq, H, 64, 16, ctx, [1] * 4)
    c.check(c.call(start=False))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new", [(4, 4, 4, 4), (1, 3, 5, 2), (16, 1, 33, 8), (0, 5, 0, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3), (1, 0), (200, 33), (5, 64)])
def test_several_tokens(dtype, new, window, sinks):
    ctx = [39, 5, 700, 130]
    c = Case(sum(new), dtype, 12, 3, 128, 16, ctx, new)
    c.check(c.call(window, sinks), window, sinks)


@pytest.mark.parametrize("B", [1, 3, 40, 257, 600])
def test_schedule(B):
    """Items cut over workgroups, whole ones, several in one workgroup; sequences without tokens between them."""
    rng = np.random.default_rng(B)
    top = max(20, 24000 // B)
    ctx = [int(x) for x in rng.integers(1, top, B)]
    if B > 3:
        ctx[1], ctx[2] = 0, 0
    c = Case(B, torch.bfloat16, 8, 2, 64, 16, ctx, [1] * B)
    c.check(c.call(start=False, max_seq_len=max(ctx)))
    # The same sizes under a far larger bound.
    wide = torch.full((B, 4096), -1, dtype=torch.int32, device=DEV)
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide
    c.check(c.call(start=False))


@pytest.mark.parametrize("B,Hq,H", [(1, 8, 2), (5, 32, 8), (64, 32, 8), (65, 32, 8), (256, 4, 2), (257, 4, 2)])
@pytest.mark.parametrize("longest", [64, 512, 513])
def test_short_sequences(B, Hq, H, longest):
    """On both sides of the rule that gives each its own workgroups: their number, their longest."""
    ctx = [(37 * i + 5 * i * i) % (longest + 1) for i in range(B)]
    ctx[B // 2] = longest
    c = Case(31, torch.bfloat16, Hq, H, 64, 16, ctx, [1] * B)
    c.check(c.call(start=False))
    c.check(c.call(window=100, sinks=3), 100, 3)


def test_long_context():
    c = Case(3, torch.bfloat16, 8, 1, 128, 16, [70001, 5], [1, 1])
    c.check(c.call(start=False))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_of_any_size(dtype):
    """Scales that are no powers of two; V scales over 2^60; zeros; a float16 output within its range."""
    c = Case(11, dtype, 8, 2, 64, 16, [500, 33, 64], [1, 2, 1], powers=False)
    c.check(c.call())
    c.scales[..., 1] *= 2.0 ** -40
    c.scales[c.table[0, 3].long(), :, 1] = 2.0 ** -2
    c.scales[c.table[1, 0].long(), :, 1] = 0.0
    c.check(c.call())
    c.scales[..., 1] = 2.0 ** -120  # (outputs of 2^-113: zeros in float16, as the exact ones round)
    if dtype == torch.bfloat16:
        c.check(c.call())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_is_not_seen_does_not_matter(dtype):
    """NaN and inf codes behind the context, before the window, at positions that other rows see; huge scales there."""
    ctx, new, window, sinks = [45, 130], [3, 2], 20, 2
    c = Case(13, dtype, 8, 2, 64, 16, ctx, new)
    clean = c.call(window, sinks)
    c.check(clean, window, sinks)
    for i, (n, m) in enumerate(zip(ctx, new)):
        for t in list(range(n, c.table.shape[1] * 16)) + list(range(sinks, n - m - window + 1)):
            if t // 16 < -(-n // 16):
                b = c.table[i, t // 16].long()
                c.kc[b, :, :, t % 16] = 0x79
                c.vc[b, :, :, t % 16] = 0x78 if t % 2 else 0x79
    again = c.call(window, sinks)
    assert torch.equal(clean, again)
    # The last new token's value is NaN: the rows before it keep their outputs, its own row is NaN.
    b, t = c.table[0, 44 // 16].long(), 44 % 16
    c.vc[b, :, :, t] = 0x79
    out = c.call(window, sinks)
    assert torch.equal(out[:2], clean[:2]) and torch.equal(out[3:], clean[3:]) and out[2].isnan().all()


def test_rows_that_see_nothing():
    c = Case(17, torch.bfloat16, 8, 2, 64, 16, [50, 60, 70, 0, 2, 80], [1, 1, 1, 1, 4, 1])
    table = c.table.clone()
    c.table[1] = -1           # no block
    c.table[2, 1] = 10 ** 6   # one block outside the pool: its tokens are left out
    lens = c.ctx
    out = c.call(max_seq_len=79)  # the last context is beyond it
    got = out.double()
    assert (got[1] == 0).all() and (got[3] == 0).all() and (got[8] == 0).all()
    assert (got[4:6] == 0).all()  # sequence 4: rows before its first token
    k, v = ps.rows_of(c.kc, c.vc, c.scales, table[2], 0, 70)
    keep = torch.cat([torch.arange(16), torch.arange(32, 70)]).to(DEV)
    want, off = ps.attend(c.query[2:3], k[keep], v[keep], len(keep) - 1, c.scale)
    assert ((got[2:3] - want).abs() <= off).all()
    assert lens == [50, 60, 70, 0, 2, 80]
    # A sequence of more rows than max_query_len.
    assert (c.call(max_query_len=3)[4:8] == 0).all()


def test_repeats_bit_for_bit_and_strided_queries():
    c = Case(19, torch.float16, 16, 2, 128, 32, [4000, 900, 1, 2500], [1, 2, 1, 4])
    first = c.call()
    for _ in range(3):
        assert torch.equal(c.call(), first)
    wide = torch.zeros((c.query.shape[0], 40, 128), dtype=torch.float16, device=DEV)
    wide[:, 8:24] = c.query
    assert torch.equal(c.call(query=wide[:, 8:24]), first)


def test_strided_caches():
    """Caches that are views: blocks and heads further apart than they are long."""
    c = Case(23, torch.bfloat16, 8, 2, 64, 16, [100, 260], [1, 1])
    want = c.call(start=False)
    k = torch.zeros((c.kc.shape[0], 5) + c.kc.shape[2:], dtype=torch.uint8, device=DEV)
    v = torch.zeros((c.vc.shape[0], 3) + c.vc.shape[2:], dtype=torch.uint8, device=DEV)
    k[:, 1:5:2] = c.kc
    v[:, :2] = c.vc
    c.kc, c.vc = k[:, 1:5:2], v[:, :2]
    assert torch.equal(c.call(start=False), want)


def test_graph_replays():
    """A captured call serves lengths and tables that change between its replays."""
    c = Case(29, torch.bfloat16, 8, 2, 64, 16, [900, 40, 333], [1, 1, 1])
    lens = torch.tensor(c.ctx, dtype=torch.int32, device=DEV)
    args = (c.kc, c.vc, c.scales, c.table, lens, None, 2, c.scale, 16, 912)
    kernels.paged_attention_scaled(c.query, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.paged_attention_scaled(c.query, *args)
    for ctx in ([900, 40, 333], [1, 17, 900], [500, 0, 2], [900, 40, 333]):
        lens.copy_(torch.tensor(ctx, dtype=torch.int32))
        want = kernels.paged_attention_scaled(c.query, *args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
