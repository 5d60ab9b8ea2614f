"""float16 queries over a context in which one token outweighs each of tens of
thousands of others: their weights are small beside the largest one, not beside the
sum, and must keep their bits.

All values of V are 1 but the heavy token's, 0, so that an output o is the light
tokens' share of the sum.  Bound: weights are rounded to 11 bits, u = 2^-11 of
each, and in float16's subnormals by half a step, 2^-25; they are scaled so that
the largest one is at least 2^11, so that this is at most 2^-36 of it for each of T
tokens.  The output is rounded, u o.  A score is off by at most (D + 4) 2^-24 of
its size in float32, which a weight and the sum take relatively, twice; sums
over T tokens and exponentials add at most (T + 64) 2^-23 o."""

import math

import pytest
import torch

from sglang_mlx_amd import kernels

pytestmark = pytest.mark.gpu

HF, U8 = torch.float16, torch.uint8
D, BS = 64, 16
U = 2.0 ** -11


def attend(cache, T, gap, new, seqs, where):
    """The outputs of `seqs` sequences over the same T tokens, of which token `where` has a score
    `gap` (of log2) above the others'."""
    blocks = T // BS
    x = 16 if cache == U8 else 8
    k = torch.zeros((blocks + 1, 1, D // x, BS, x), dtype=cache, device="cuda")
    v = torch.zeros((blocks + 1, 1, D, BS), dtype=cache, device="cuda")
    one = 0x38 if cache == U8 else 1.0
    v[:] = one
    v[where // BS, :, :, where % BS] = 0
    k[where // BS, :, :, where % BS] = one
    # Queries of 1 and D keys of 1: the score is D times the scale.
    scale = gap * math.log(2.0) / D
    table = torch.arange(blocks, dtype=torch.int32, device="cuda").repeat(seqs, 1)
    lens = torch.full((seqs,), T, dtype=torch.int32, device="cuda")
    start = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * new
    q = torch.ones((seqs * new, 2, D), dtype=HF, device="cuda")
    return kernels.paged_attention_extend(q, k, v, table, lens, start, 1, scale, BS, T, new), scale


@pytest.mark.parametrize("cache", [HF, U8], ids=["float16", "fp8"])
@pytest.mark.parametrize("gap", [12.4, 18.6, 20.3, 22.3, 23.4, 24.4, 25.5])
# Single tokens, few rows, row tiles; one sequence (split) and as many as fill the chip (not split).
@pytest.mark.parametrize("new,seqs", [(1, 1), (3, 2), (1, 600), (12, 1), (70, 1), (70, 300)])
def test_many_light_tokens(cache, gap, new, seqs):
    T = 32768
    for where in (0, 20000):  # (found first, or when most others have been summed)
        got, scale = attend(cache, T, gap, new, seqs, where)
        score = D * float(torch.tensor(scale, dtype=torch.float32))
        heavy = math.exp(score)
        # Row i of a sequence sees T - new + 1 + i tokens, the heavy one among them.
        light = torch.arange(T - new, T, dtype=torch.float64, device="cuda").repeat(seqs)
        want = light / (light + heavy)
        bound = want * (2.02 * U + 4 * (D + 4) * 2.0 ** -24 * score + (T + 64) * 2.0 ** -23) + 2.0 ** -36 * T + 2.0 ** -25
        error = (got.double() - want[:, None, None]).abs()
        assert (error <= bound[:, None, None]).all(), (where, (error / want[:, None, None]).max().item())
