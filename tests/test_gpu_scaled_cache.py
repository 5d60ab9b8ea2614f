"""quantize_and_cache and dequantize_cache: codes and scales bit for bit those of the rule
in plain form, rows back bit for bit code * scale rounded once."""

import numpy as np
import pytest
import torch

import pkv_scaled as ps
from sglang_mlx_amd import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"


class Pool:
    """Caches full of arbitrary codes, scales as a store writes them, and tables of disjoint blocks."""

    def __init__(self, seed, H, D, bs, lens, spare=3):
        self.rng = rng = np.random.default_rng(seed)
        need = [-(-int(c) // bs) for c in lens]
        self.nb = sum(need) + spare
        ids = rng.permutation(self.nb)
        self.tables = np.full((len(lens), max(need + [1])), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = ids[at:at + n]
            at += n
        codes = lambda shape: ((rng.integers(0, 0x78, shape) | (rng.integers(0, 2, shape) << 7)).astype(np.uint8))  # noqa: E731
        self.kc, self.vc = codes((self.nb, H, D // 16, bs, 16)), codes((self.nb, H, D, bs))
        self.scales = (2.0 ** rng.integers(-9, 1, (self.nb, H, 2))).astype(np.float32)
        self.H, self.D, self.bs = H, D, bs

    def check_store(self, key, value, ctx, start, stride_pad=0, tables=None):
        """key, value: tensors of the source type on the host."""
        tables = self.tables if tables is None else tables
        dev = [torch.from_numpy(x.copy()).to(DEV) for x in (self.kc, self.vc, self.scales)]
        if stride_pad:
            wide = torch.zeros((key.shape[0], 2 * self.H * self.D + stride_pad), dtype=key.dtype, device=DEV)
            k = wide[:, :self.H * self.D].unflatten(1, (self.H, self.D))
            v = wide[:, self.H * self.D:2 * self.H * self.D].unflatten(1, (self.H, self.D))
            k.copy_(key), v.copy_(value)
        else:
            k, v = key.to(DEV), value.to(DEV)
        ints = [torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV) for x in (tables, ctx, start)]
        out = kernels.quantize_and_cache(k, v, *dev, *ints)
        assert out[0] is dev[0] and out[1] is dev[1] and out[2] is dev[2]
        ps.store(key.float().numpy(), value.float().numpy(), self.kc, self.vc, self.scales, tables, ctx, start)
        for got, want in zip(dev, (self.kc, self.vc, self.scales)):
            assert np.array_equal(got.cpu().numpy().view(np.uint8), want.view(np.uint8))

    def source(self, n, dtype, spread=3.0):
        shape = (n, self.H, self.D)
        size = 2.0 ** self.rng.uniform(-spread, spread, (1, self.H, 1))
        k, v = (torch.from_numpy((self.rng.standard_normal(shape) * size).astype(np.float32)).to(dtype)
                for _ in range(2))
        return k, v


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,bs,H", [(128, 16, 2), (32, 8, 1), (64, 32, 3), (80, 16, 1), (96, 8, 2), (112, 32, 1),
                                    (192, 16, 1), (256, 32, 1), (256, 8, 2)])
def test_store_in_steps(dtype, D, bs, H):
    """A prefill, a chunk, single and several tokens: whole blocks, parts of blocks at either end, blocks that grow."""
    lens = np.array([0, 0, 0, 0, 0])
    pool = Pool(1, H, D, bs, [3 * bs + 7] * 5)
    for step, new in enumerate([(bs + 3, 2 * bs, 1, 0, 5), (2, 1, 1, 0, bs), (1, 1, 1, 1, 1), (bs + 1, 0, 3, 2 * bs, 1),
                                (1, 1, 1, 1, 1)]):
        lens = lens + np.array(new)
        n = sum(new)
        k, v = pool.source(n, dtype, spread=1.0 + step)
        pool.check_store(k, v, lens, np.concatenate([[0], np.cumsum(new)]), stride_pad=8 * (step % 2))


def test_store_a_token_at_a_time_is_a_store_at_once():
    """Codes of one block filled in 16 steps: as in one, but for codes that became subnormal on the way (rounded twice)."""
    H, D, bs = 2, 128, 16
    once, steps = Pool(5, H, D, bs, [bs]), Pool(5, H, D, bs, [bs])
    k, v = once.source(bs, torch.bfloat16, spread=0.0)
    k *= (2.0 ** torch.arange(-8, 8))[:, None, None]  # every token grows the scale
    once.check_store(k, v, [bs], [0, bs])
    for t in range(bs):
        steps.check_store(k[t:t + 1], v[t:t + 1], [t + 1], [0, 1])
    block = once.tables[0, 0]
    assert np.array_equal(once.scales[block], steps.scales[block])
    for a, b in ((once.kc, steps.kc), (once.vc, steps.vc)):
        x, y = ps.VALUES[a[block]], ps.VALUES[b[block]]
        normal = np.abs(x) >= 2.0 ** -6
        assert np.array_equal(x[normal], y[normal])
        assert np.abs(x - y).max() <= 2.0 ** -9  # two roundings of half a subnormal step each, one apart at most


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_store_special_values(dtype):
    """Zeros, subnormals, the largest and smallest values, inf and NaN; borders of the scale's rule."""
    pool = Pool(7, 1, 64, 16, [16] * 12)
    big = torch.finfo(dtype).max
    k, v = pool.source(16 * 12, dtype, spread=0.0)
    k[0:16] = 0.0
    v[16:32] *= torch.finfo(dtype).tiny
    k[32:48] *= torch.finfo(dtype).smallest_normal
    k[48, 0, 3], v[50, 0, 5], v[51, 0, 6] = float("inf"), float("-inf"), float("nan")
    k[64:80] = float("nan")
    v[80:96] = float("inf")
    k[96, 0, 0], v[97, 0, 1] = big, -big
    for i, a in enumerate((240.0, 241.0, 120.0, 0.9375, 0.94)):  # 240 is exactly on the border, 241 past it
        k[112 + 16 * i:128 + 16 * i] = k[112 + 16 * i:128 + 16 * i].clamp(-a / 2, a / 2)
        k[115 + 16 * i, 0, 9] = a
    pool.check_store(k, v, [16] * 12, np.arange(13) * 16)
    # A later token beside inf and NaN, beside zeros, beside the largest value.
    pool = Pool(8, 1, 64, 16, [16] * 4)
    k, v = pool.source(4 * 5, dtype, spread=0.0)
    k[0:5] = 0.0
    k[6, 0, 1], v[7, 0, 2], v[7, 0, 3] = float("inf"), float("nan"), float("-inf")
    k[10:15] = big
    pool.check_store(k, v, [5] * 4, np.arange(5) * 5)
    k, v = pool.source(4, dtype, spread=0.0)
    pool.check_store(k * 64, v * 64, [6] * 4, np.arange(5))


def test_store_scales_that_are_no_powers_of_two():
    """Scales that a calibration wrote: kept while they hold, replaced by a power of two when a token outgrows them."""
    pool = Pool(9, 2, 128, 16, [40, 40])
    pool.scales[:] = pool.rng.uniform(0.004, 0.02, pool.scales.shape)
    k, v = pool.source(8, torch.bfloat16, spread=2.0)
    pool.check_store(k, v, [19, 27], [0, 3, 8])


def test_store_what_goes_nowhere():
    H, D, bs = 2, 64, 16
    pool = Pool(11, H, D, bs, [40, 40, 40, 40, 40, 40])
    k, v = pool.source(64, torch.bfloat16)
    tables = pool.tables.copy()
    tables[0, 1], tables[1, 0] = -1, pool.nb  # blocks outside the cache
    # Sequence 2: no context; 3: beyond its table; 4: more rows than context; 5: ends past the rows at hand.
    pool.check_store(k, v, [40, 20, 0, 49, 5, 30], [0, 30, 33, 40, 44, 52, 70], tables=tables)
    # Rows behind the last sequence; sequences without rows; no sequence at all.
    pool.check_store(k, v, [33, 7], [0, 4, 4], tables=pool.tables[:2])
    pool.check_store(k[:0], v[:0], [33], [0, 0], tables=pool.tables[:1])
    pool.check_store(k, v, [], [0], tables=pool.tables[:0])


@pytest.mark.parametrize("B", [64, 65, 700, 5000])
def test_store_many_sequences(B):
    """The search for a work item's sequence, over one probe, two and three."""
    pool = Pool(13, 1, 32, 8, [12] * B)
    lens = 1 + np.arange(B) * 7 % 12
    new = np.minimum(lens, np.arange(B) * 5 % 4)
    k, v = pool.source(int(new.sum()) + 3, torch.float16)
    pool.check_store(k, v, lens, np.concatenate([[0], np.cumsum(new)]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,bs,H", [(128, 16, 2), (32, 8, 1), (64, 32, 3), (80, 16, 1), (96, 8, 2), (112, 32, 1),
                                    (192, 16, 1), (256, 32, 1), (256, 8, 2)])
def test_read(dtype, D, bs, H):
    lens = [1, 3 * bs + 5, 0, bs, 2 * bs - 1, 70]
    pool = Pool(17, H, D, bs, lens)
    pool.scales[:] = pool.rng.uniform(0.001, 0.1, pool.scales.shape)
    pool.kc.reshape(-1)[:256] = np.arange(256)  # every code
    pool.vc.reshape(-1)[:256] = np.arange(256)
    tables = pool.tables.copy()
    tables[1, 1] = -1
    tables[5, 0] = pool.nb + 5
    tables[3, 0], tables[0, 0] = 0, 0  # (a shared block, the one with every code)
    start = np.concatenate([[0], np.cumsum(lens)])
    extra = 9
    dev = [torch.from_numpy(x).to(DEV) for x in (pool.kc, pool.vc, pool.scales, tables)]
    k, v = kernels.dequantize_cache(*dev, torch.tensor(start, dtype=torch.int32, device=DEV), int(start[-1]) + extra,
                                    dtype)
    for got, cache, which in ((k, pool.kc.transpose(0, 3, 1, 2, 4).reshape(pool.nb, bs, H, D), 0),
                              (v, pool.vc.transpose(0, 3, 1, 2), 1)):
        want = np.zeros((int(start[-1]) + extra, H, D), np.float32)
        for s, n in enumerate(lens):
            for t in range(n):
                b = tables[s, t // bs]
                if 0 <= b < pool.nb:
                    want[start[s] + t] = ps.VALUES[cache[b, t % bs]].astype(np.float32) * pool.scales[b, :, which, None]
        want = torch.from_numpy(want).to(dtype)
        got = got.cpu()
        assert got.dtype == dtype and got.shape == want.shape
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(1.0), want.nan_to_num(1.0))


def test_read_past_a_table_and_cut_short():
    H, D, bs = 1, 64, 16
    pool = Pool(19, H, D, bs, [32, 32])
    dev = [torch.from_numpy(x).to(DEV) for x in (pool.kc, pool.vc, pool.scales, pool.tables)]
    whole = kernels.dequantize_cache(*dev, torch.tensor([0, 32, 64], dtype=torch.int32, device=DEV), 64, torch.float32)
    # 40 rows of a table of 32 tokens, then 40 of which 10 lie in the outputs.
    part = kernels.dequantize_cache(*dev, torch.tensor([0, 40, 80], dtype=torch.int32, device=DEV), 50, torch.float32)
    for a, b in zip(whole, part):
        assert torch.equal(b[:32], a[:32]) and (b[32:40] == 0).all() and torch.equal(b[40:], a[32:42])
    for n, start in ((5, [0]), (0, [0, 0, 0])):
        k, v = kernels.dequantize_cache(*dev[:3], dev[3][:len(start) - 1],
                                        torch.tensor(start, dtype=torch.int32, device=DEV), n)
        assert k.shape == v.shape == (n, H, D) and k.dtype == torch.bfloat16 and (k == 0).all() and (v == 0).all()


def test_index_types_and_other_stream():
    """int64 indexes and sources that need a copy take the general path; work runs on the current stream."""
    H, D, bs = 2, 64, 16
    pool = Pool(23, H, D, bs, [40, 21])
    key, value = pool.source(25, torch.float16)
    dev = [torch.from_numpy(x.copy()).to(DEV) for x in (pool.kc, pool.vc, pool.scales)]
    ref = [t.clone() for t in dev]
    i32 = [torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV) for x in (pool.tables, [40, 21], [0, 13, 25])]
    kernels.quantize_and_cache(key.to(DEV), value.to(DEV), *ref, *i32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k = key.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)  # (strided inside a row)
        kernels.quantize_and_cache(k, value.to(DEV), *dev, *[t.long() for t in i32])
        rows = kernels.dequantize_cache(*dev, i32[0].long(), torch.tensor([0, 40, 61], device=DEV), 61, torch.float16)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(dev, ref))
    want = kernels.dequantize_cache(*ref, i32[0], torch.tensor([0, 40, 61], dtype=torch.int32, device=DEV), 61,
                                    torch.float16)
    assert all(torch.equal(a, b) for a, b in zip(rows, want))
