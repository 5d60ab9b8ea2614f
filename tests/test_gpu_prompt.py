"""prompt_attention against attention in 64 bits."""

import numpy as np
import pytest
import torch

import pkv_scaled as ps
from sglang_mlx_amd import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def starts(lens):
    return ints(np.concatenate([[0], np.cumsum(lens)]))


class Case:
    def __init__(self, seed, dtype, Hq, H, D, new, ctx=None, gain=1.5):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.new, self.ctx = list(new), list(new if ctx is None else ctx)
        self.own = ctx is None
        make = lambda n, h: torch.randn((n, h, D), generator=g, device=DEV)  # noqa: E731
        self.q = (make(sum(new), Hq) * gain).to(dtype)
        self.k, self.v = (make(sum(self.ctx), H).to(dtype) for _ in range(2))
        self.scale = D ** -0.5

    def call(self, window=0, sinks=0, q=None, k=None, v=None, scale=None, max_query_len=None, max_key_len=None):
        more = {}
        if not self.own:
            more = dict(key_start_loc=starts(self.ctx), max_key_len=max_key_len or max(self.ctx + [1]))
        return kernels.prompt_attention(self.q if q is None else q, self.k if k is None else k,
                                        self.v if v is None else v, starts(self.new),
                                        self.scale if scale is None else scale, max_query_len or max(self.new + [1]),
                                        window=window, num_sinks=sinks, **more)

    def check(self, out, window=0, sinks=0, scale=None):
        a = b = 0
        for i, (n, c) in enumerate(zip(self.new, self.ctx)):
            if n and c:
                want, off = ps.attend(self.q[a:a + n], self.k[b:b + c].double(), self.v[b:b + c].double(), c - n,
                                      self.scale if scale is None else scale, window, sinks)
                worst = ((out[a:a + n].double() - want).abs() - off).max()
                assert worst <= 0, (i, n, c, float(worst))
            a, b = a + n, b + c
        assert (out[a:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 80, 96, 112, 120, 128, 192, 256])
def test_ragged_prompts(dtype, D):
    c = Case(D, dtype, 8, 2, D, [1, 2, 31, 32, 33, 63, 64, 65, 130, 5, 0, 257])
    c.check(c.call())


@pytest.mark.parametrize("Hq,H", [(1, 1), (4, 4), (7, 1), (32, 8), (28, 4), (40, 1), (3, 3)])
def test_head_layouts(Hq, H):
    c = Case(Hq, torch.bfloat16, Hq, H, 64, [77, 1, 190])
    c.check(c.call())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (33, 0), (64, 4), (100, 70), (5, 200), (2000, 3)])
def test_windows_and_contexts(dtype, window, sinks):
    c = Case(window, dtype, 8, 2, 128, [40, 1, 129, 300, 2], [40, 900, 500, 301, 64])
    c.check(c.call(window, sinks), window, sinks)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_few_rows_of_long_contexts(D):
    """Keys in several parts, merged by a second launch."""
    c = Case(D, torch.bfloat16, 8, 2, D, [30, 1, 60], [5000, 3000, 61])
    c.check(c.call())
    c.check(c.call(3000, 5), 3000, 5)
    # Hints that are too small or too large choose another cut and give the same rows.
    c.check(c.call(max_query_len=1, max_key_len=1))
    c.check(c.call(max_query_len=10 ** 12, max_key_len=10 ** 12))


def test_long_prompt():
    c = Case(5, torch.bfloat16, 4, 1, 128, [3333])
    c.check(c.call())
    c = Case(6, torch.float16, 4, 1, 64, [2222])
    c.check(c.call())


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0, 1e-30])
def test_scales(scale):
    c = Case(7, torch.bfloat16, 4, 2, 64, [100, 64])
    c.check(c.call(scale=scale), scale=scale)


def test_strided_rows():
    """Views of one projection, and rows that need a copy first."""
    c = Case(9, torch.bfloat16, 8, 2, 64, [50, 131])
    want = c.call()
    qkv = torch.cat([x.flatten(1) for x in (c.q, c.k, c.v)], 1)
    q, k, v = qkv.split([512, 128, 128], 1)
    assert torch.equal(c.call(q=q.unflatten(1, (8, 64)), k=k.unflatten(1, (2, 64)), v=v.unflatten(1, (2, 64))), want)
    k2 = c.k.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(c.call(k=k2), want)
    one = Case(10, torch.float16, 8, 2, 64, [1])
    one.check(one.call())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_is_not_seen_does_not_matter(dtype, D):
    """inf and NaN in later tokens, in the sequence behind, before a window."""
    c = Case(11, dtype, 8, 2, D, [100, 70, 40])
    clean, windowed = c.call(), c.call(20, 2)
    k, v = c.k.clone(), c.v.clone()
    k[90:100], v[90], v[95] = float("nan"), float("inf"), float("nan")   # tokens 90 .. 99 of sequence 0
    k[100], v[100:102] = float("inf"), float("-inf")                    # the first of sequence 1
    out = c.call(k=k, v=v)
    assert torch.equal(out[:90], clean[:90]) and torch.equal(out[170:], clean[170:])
    assert not out[90:170].isfinite().all(-1).any()
    k, v = c.k.clone(), c.v.clone()
    k[2:40], v[2:40] = float("nan"), float("nan")
    out = c.call(20, 2, k=k, v=v)
    assert torch.equal(out[:2], windowed[:2]) and torch.equal(out[59:], windowed[59:]) and out[2:59].isnan().all()


def test_rows_that_see_nothing():
    # More queries than keys, no keys, rows behind the last sequence.
    c = Case(13, torch.bfloat16, 4, 2, 64, [10, 5, 20], [4, 0, 40])
    out = c.call()
    assert (out[:6] == 0).all() and (out[10:15] == 0).all()
    want, off = ps.attend(c.q[6:10], c.k[:4].double(), c.v[:4].double(), 0, c.scale)
    assert ((out[6:10].double() - want).abs() <= off).all()
    want, off = ps.attend(c.q[15:], c.k[4:].double(), c.v[4:].double(), 20, c.scale)
    assert ((out[15:].double() - want).abs() <= off).all()
    d = Case(14, torch.bfloat16, 4, 2, 64, [30, 30])
    out = kernels.prompt_attention(d.q, d.k, d.v, ints([0, 30]), d.scale, 30)
    assert torch.equal(out[:30], d.call()[:30]) and (out[30:] == 0).all()
    assert (kernels.prompt_attention(d.q, d.k, d.v, ints([0]), d.scale, 30) == 0).all()
    assert kernels.prompt_attention(d.q[:0], d.k[:0], d.v[:0], ints([0, 0]), d.scale, 1).shape == (0, 4, 64)
    assert (kernels.prompt_attention(d.q, d.k[:0], d.v[:0], ints([0, 60]), d.scale, 60, ints([0, 0]), 1) == 0).all()


def test_many_sequences():
    lens = [1 + 13 * i % 29 for i in range(150)]
    c = Case(15, torch.float16, 4, 2, 64, lens)
    c.check(c.call())


def test_small_float16_weights():
    """Thousands of light tokens beside a heavy one keep their share (2^-22 each)."""
    c = Case(17, torch.float16, 1, 1, 64, [1], [8193], gain=0.0)
    c.q[:] = 0.0
    c.q[..., 0] = 1.0
    c.k[:] = 0.0
    c.k[0, 0, 0] = 22 * np.log(2) / c.scale
    c.v[:] = 0.0
    c.v[1:, 0, 0] = 1000.0
    c.check(c.call())


def test_repeats_and_graph_replays():
    c = Case(19, torch.bfloat16, 8, 2, 128, [60, 10], [2000, 700])
    first = c.call()
    args = (starts(c.new), c.scale, 60, starts(c.ctx), 2000)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.prompt_attention(c.q, c.k, c.v, *args)
    for _ in range(4):
        assert torch.equal(c.call(), first)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
