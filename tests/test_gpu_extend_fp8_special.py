"""FP8 caches that hold codes of exponent 15 (infinities and NaN), which the
append stores for what overflows and stale blocks may hold: they decode to what
they stand for, they reach the rows that see them, and no other row.  Bounds as in
test_gpu_extend."""

import pytest
import torch

import test_gpu_extend
from test_gpu_extend import BF, HF, U8, Batch

pytestmark = pytest.mark.gpu

INF, MINUS_INF, NAN, MINUS_NAN, ODD_NAN = 0x78, 0xF8, 0x7F, 0xFF, 0x7A
CODES = [INF, MINUS_INF, NAN, MINUS_NAN, ODD_NAN]


@pytest.fixture(autouse=True)
def all_codes(monkeypatch):
    finite = test_gpu_extend.code_values

    def values():
        v = finite()
        for sign, at in ((1.0, 0), (-1.0, 128)):
            v[at + 0x78] = sign * float("inf")
            v[at + 0x79:at + 0x80] = float("nan")
        return v

    monkeypatch.setattr(test_gpu_extend, "code_values", values)


def batch(q, D, bs, ctx, new):
    return Batch(D + bs, ctx, new, (4, 2), D, bs, q, U8)


def spoil(b, cache, seq, token, code, d=None):
    """Sets a token's element d (all of them) of every KV head to the code."""
    blk, at = b.table[seq, token // b.bs].item(), token % b.bs
    if cache == "v":
        b.v[blk, :, slice(None) if d is None else d, at] = code
    elif d is None:
        b.k[blk, :, :, at] = code
    else:
        b.k[blk, :, d // 16, at, d % 16] = code


SHAPES = [(BF, 64, 32), (BF, 128, 16), (HF, 128, 8), (HF, 80, 16), (BF, 256, 16)]
IDS = [f"{str(q)[6:]}-{D}-{bs}" for q, D, bs in SHAPES]
NEW = [[1, 1], [4, 2], [90, 20]]  # single tokens, few rows, row tiles


@pytest.mark.parametrize("code", CODES, ids=hex)
@pytest.mark.parametrize("q,D,bs", SHAPES, ids=IDS)
def test_behind_the_contexts(q, D, bs, code):
    for new in NEW:
        b = batch(q, D, bs, [93, 61], new)
        want = [b.extend(), b.extend(30, 2)]
        for i, c in enumerate(b.ctx):
            blk = b.table[i, c // bs].item()
            b.k[blk, :, :, c % bs:], b.v[blk, :, :, c % bs:] = code, code
        b.k[0], b.v[0] = code, code  # (what missing blocks' loads read)
        assert b.extend().equal(want[0]) and b.extend(30, 2).equal(want[1])
        b.check(b.extend())


@pytest.mark.parametrize("code", CODES, ids=hex)
@pytest.mark.parametrize("q,D,bs", SHAPES, ids=IDS)
def test_inside_a_context(q, D, bs, code):
    # Token 100 of 200: seen by rows at its position and after, until a window leaves it.
    for new in ([150, 1], [104, 3], [3, 2]):
        for cache in "kv":
            b = batch(q, D, bs, [200, 40], new)
            first = 200 - new[0]
            spoil(b, cache, 0, 100, code, 5)
            for window, sinks in ((0, 0), (20, 0), (20, 101), (99, 0)):
                got = b.extend(window, sinks)
                b.check(got, window, sinks)
                pos = torch.arange(first, 200, device="cuda")
                hit = (pos >= 100) & ((pos < 100 + window) | (window == 0) | (sinks > 100))
                rows, other = got[:new[0]], torch.arange(D, device="cuda") != 5
                if cache == "v":
                    assert (~torch.isfinite(rows[..., 5])).all(1).equal(hit)
                    assert torch.isfinite(rows[..., other]).all()
                elif code not in (INF, MINUS_INF):
                    assert torch.isnan(rows[hit]).all() and torch.isfinite(rows[~hit]).all()
                assert torch.isfinite(got[new[0]:]).all()


@pytest.mark.parametrize("q", [BF, HF], ids=["bfloat16", "float16"])
def test_infinite_values_keep_their_sign(q):
    for new in NEW:
        for code, value in ((INF, float("inf")), (MINUS_INF, float("-inf"))):
            b = batch(q, 64, 16, [93, 61], new)
            spoil(b, "v", 0, 2, code, 7)
            got = b.extend()[:new[0]]
            sees = torch.arange(93 - new[0], 93, device="cuda") >= 2
            # (Where the weight is 0 in the product's type, 0 times an infinity is NaN: equal keys avoid it.)
            assert (~torch.isfinite(got[sees][..., 7])).all()
            b.k.zero_()
            got = b.extend()[:new[0]]
            assert (got[sees][..., 7] == value).all() and torch.isfinite(got[~sees]).all()


@pytest.mark.parametrize("q", [BF, HF], ids=["bfloat16", "float16"])
def test_a_key_of_minus_infinity_has_no_weight(q):
    # Its score is minus infinity where the query's element is positive: as if the token were not there.
    for new in NEW:
        b = batch(q, 64, 16, [93, 61], new)
        b.q[..., 9] = b.q[..., 9].abs() + 0.5
        spoil(b, "k", 0, 2, MINUS_INF, 9)
        got = b.extend()
        assert torch.isfinite(got).all()
        # A row of only such keys is zero, and the rows around it are not.
        first = 93 - new[0]
        if first < 3:
            continue
        for t in range(first + 1):
            spoil(b, "k", 0, t, MINUS_INF, 9)
        got = b.extend()
        assert (got[0] == 0).all() and torch.isfinite(got).all()


def test_long_split_contexts():
    for ctx, new in (([9000, 40], [1, 1]), ([7000, 40], [30, 2])):
        b = batch(BF, 128, 16, ctx, new)
        spoil(b, "v", 0, 3000, NAN, 5)
        for window, sinks in ((0, 0), (2000, 4), (2000, 3001)):
            got = b.extend(window, sinks)
            b.check(got, window, sinks)
            hit = window == 0 or sinks > 3000
            assert torch.isnan(got[:new[0], :, 5]).all() if hit else torch.isfinite(got).all()
