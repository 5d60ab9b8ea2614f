"""paged_attention_scaled where the scales of V lie far apart: a block that a row sees but
gives no weight to takes no bits from the others, whatever its scale."""

import math

import pytest
import torch

import pkv_scaled as ps
from sglang_mlx_amd import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"


def attend(q, k, codes, vs, first, scale):
    """q [n, Hq, D] at positions first, ..; k [T, H, D], V's codes [T, H, D] and scales [T, H], float64.  The output
    and the most that a kernel may be off, both float64 [n, Hq, D].

    The bound, with u half a step of the type: each product of a weight and its scale is rounded to the type (u of
    it), the output once (u of it), e32 covers float32 scores, exponentials, sums and the division as in
    pkv_scaled.attend.  A float16 product below the type's normal range (2^-14) is off by at most 2^-25; the reference
    point is at most one above the log2 of the largest product, which is brought to 2^11 there and whose scale's
    significand is at least a half: the largest is stored as at least 2^9, so that every token's product is off by at
    most 2^-34 of the largest one, times its code.  An output below the type's normal range is a multiple of its
    smallest subnormal.

    Weights are float32 numbers relative to 2^m, m one of the row's scores (log2), and those below its normal range
    are zeros: s - m < -126, so that s is more than 126 below the largest.  Pieces of a row meet by factors 2^(m - M),
    which are zeros below 2^-126 too.  The whole of such tokens' share is allowed for (a score's own error, (D + 8)
    2^-24 of the sum of the sizes, is below 0.001 here)."""
    n, Hq, D = q.shape
    T, H = codes.shape[:2]
    u = torch.finfo(q.dtype).eps / 2
    least = u * torch.finfo(q.dtype).smallest_normal
    sees = torch.arange(T, device=DEV) <= torch.arange(first, first + n, device=DEV)[:, None]
    out = torch.zeros((n, Hq, D), dtype=torch.float64, device=DEV)
    off = torch.zeros_like(out)
    for h in range(Hq):
        g = h // (Hq // H)
        kh, qh = k[:, g].contiguous(), q[:, h].double()
        # (Not torch.softmax: over long rows its float64 form on the GPU takes float32 exponentials, zero below 2^-126.)
        p = ((qh @ kh.t().contiguous()) * scale).masked_fill(~sees, -math.inf)
        p = (p - p.amax(1, keepdim=True)).exp()
        p = p / p.sum(1, keepdim=True)
        w = p * vs[:, g]
        gone = torch.where(p < 1.001 * 2.0 ** -126 * p.amax(1, keepdim=True), w, 0.0)
        # (Scores' errors of the tokens that weigh: exp(error) of the others has no say.)
        size = (qh.abs() @ kh.abs().t().contiguous()) * abs(scale)
        e32 = 2 * (D + 8) * 2.0 ** -24 * torch.where(sees, size, 0.0).amax(1, keepdim=True) + 2.0 ** -20
        d = codes[:, g].abs().contiguous()
        o = w @ codes[:, g].contiguous()
        out[:, h] = o
        off[:, h] = ((u + e32) * (w @ d) + (u + e32) * o.abs() + least
                     + 2.0 ** -34 * w.amax(1, keepdim=True) * (sees.double() @ d) + gone @ d)
    return out, off


class Case:
    """Heavy blocks (of every head): V scale 2^high, keys that bring a score `nats` below the others' about 0.
    The others' V scales are 2^low."""

    def __init__(self, seed, dtype, Hq, H, D, bs, ctx, new, heavy, high, low, nats):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        need = [-(-c // bs) for c in ctx]
        nb = sum(need)
        self.table = torch.full((len(ctx), max(need)), -1, dtype=torch.int32)
        at = 0
        for i, m in enumerate(need):
            self.table[i, :m] = torch.arange(at, at + m)
            at += m
        self.table = self.table.to(DEV)
        codes = lambda s: torch.randn(s, generator=g, device=DEV).mul_(60).clamp_(-240, 240).to(  # noqa: E731
            torch.float8_e4m3fn)
        kc, vc = codes((nb, H, D // 16, bs, 16)), codes((nb, H, D, bs))
        self.scales = torch.empty((nb, H, 2), device=DEV)
        self.scales[..., 0], self.scales[..., 1] = 2.0 ** -8, 2.0 ** low
        # Dimension 0 of a query is 16; of a key 0, in heavy blocks -240 with a K scale to the score wanted.
        self.scale = D ** -0.5
        self.query = torch.randn((sum(new), Hq, D), generator=g, device=DEV)
        self.query[..., 0] = 16.0
        self.query = self.query.to(dtype)
        kc[:, :, 0, :, 0] = 0.0
        for i, blocks in enumerate(heavy):
            ids = [int(self.table[i, b]) for b in blocks]
            for b in ids:
                kc[b] = 0.0
                kc[b, :, 0, :, 0] = -240.0
                self.scales[b, :, 0] = nats / (16.0 * 240.0 * self.scale)
                self.scales[b, :, 1] = 2.0 ** high
        self.kc, self.vc = kc.view(torch.uint8), vc.view(torch.uint8)
        self.ctx, self.new, self.bs, self.H = ctx, new, bs, H

    def check(self):
        lens = torch.tensor(self.ctx, dtype=torch.int32, device=DEV)
        starts = [0]
        for n in self.new:
            starts.append(starts[-1] + n)
        out = kernels.paged_attention_scaled(
            self.query, self.kc, self.vc, self.scales, self.table, lens, torch.tensor(starts, dtype=torch.int32,
                                                                                     device=DEV),
            self.H, self.scale, self.bs, self.table.shape[1] * self.bs, max(self.new)).double()
        values = torch.from_numpy(ps.VALUES).to(DEV)
        for i, (c, n) in enumerate(zip(self.ctx, self.new)):
            k, _ = ps.rows_of(self.kc, self.vc, self.scales, self.table[i], 0, c)
            pos = torch.arange(c, device=DEV)
            block = self.table[i].long()[pos // self.bs]
            d = values[self.vc[block, :, :, pos % self.bs].long()]
            vs = self.scales.double()[block][:, :, 1]
            rows = slice(starts[i], starts[i + 1])
            want, off = attend(self.query[rows], k, d, vs, c - n, self.scale)
            worst = ((out[rows] - want).abs() / off).max()
            assert worst <= 1, (i, c, n, float(worst))


HEAVY = [[0], [3], [1, 7, 12], [20]]
CTX, NEW = [450, 97, 700, 5000], [1, 3, 4, 1]


@pytest.mark.parametrize("bs", [8, 16, 32])
@pytest.mark.parametrize("high,low,nats", [(0, 0, 42), (8, -14, 42), (12, -16, 42), (14, -16, 42), (15, -17, 42),
                                           (16, -18, 60), (100, -14, 80), (100, -18, 150), (121, -4, 86),
                                           (121, -14, 400)])
def test_float16(bs, high, low, nats):
    Case(high + bs, torch.float16, 8, 2, 64, bs, CTX, NEW, [[b for b in x if b * bs < c] for x, c in zip(HEAVY, CTX)],
         high, low, nats).check()


@pytest.mark.parametrize("bs", [8, 16, 32])
@pytest.mark.parametrize("high,low,nats", [(0, 0, 42), (60, -40, 100), (60, -60, 100), (70, -58, 100), (100, -36, 150),
                                           (120, -3, 86), (121, -100, 400)])
def test_bfloat16(bs, high, low, nats):
    Case(high + bs, torch.bfloat16, 8, 2, 128, bs, CTX, NEW,
         [[b for b in x if b * bs < c] for x, c in zip(HEAVY, CTX)], high, low, nats).check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nats", [1, 8, 20])
def test_blocks_that_weigh(dtype, nats):
    """The wide block's share of the output is large, small or between."""
    for high in (0, 6, 12):
        Case(5, dtype, 12, 3, 64, 16, CTX, NEW, HEAVY, high, -10, nats).check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_falling_and_rising_scores(dtype):
    """Every block's keys and V scale differ: scores over 120 nats, scales over 2^30, in both orders and mixed."""
    for order in (1, -1, 7):
        c = Case(9, dtype, 8, 2, 64, 16, [1500, 640], [2, 1], [[], []], 0, 0, 1)
        for i in range(2):
            ids = c.table[i][c.table[i] >= 0].long()
            m = len(ids)
            rank = torch.arange(m, device=DEV) * order % m
            kc = c.kc.view(torch.float8_e4m3fn)
            for j, b in enumerate(ids.tolist()):
                r = float(rank[j]) / (m - 1)
                kc[b] = 0.0
                kc[b, :, 0, :, 0] = -224.0 + 7 * torch.arange(16, device=DEV)  # tokens apart by up to 105 / 240
                c.scales[b, :, 0] = max(120.0 * r, 0.1) / (16.0 * 240.0 * c.scale)
                c.scales[b, :, 1] = 2.0 ** round(15 - 30 * (1 - r))
        c.check()
