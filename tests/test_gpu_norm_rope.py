"""qk_norm_rope and qk_norm_rope_and_cache against the formula in 64 bits.

Bounds.  The kernel computes in float32 and rounds once.  With a, b the normed
pair, a rotated element is off by a few float32 roundings of |a cos| + |b sin| <=
|a| + |b|: the sum of D squares and its mean (a tree of sums of 8: at most 8 + 6
roundings, halved by the root), the division, the root and its reciprocal, two products
with them, and the rotation's three: below 24 in all, so 24 * 2^-24 (|a| + |b|),
taken twice.  Then half a step of the output type (and of its smallest
subnormal, 2^-25 for float16)."""

import numpy as np
import pytest
import torch

from oracle import pagedkv_oracle as orc
from sglang_mlx_amd import kernels
from sglang_mlx_amd.rotary import rotary_table

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
TINY = {BF: 2.0 ** -134, HF: 2.0 ** -25, FP: 2.0 ** -150}


def reference(x, weight, pos, cos_sin, eps, interleaved):
    """(value, |a| + |b|) in 64 bits."""
    x = x.double()
    P, rot = cos_sin.shape
    half = rot // 2
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    t = cos_sin.double()[pos.long().clamp(0, P - 1)][:, None]
    cos, sin = t[..., :half], t[..., half:]
    first = torch.arange(0, rot, 2) if interleaved else torch.arange(half)
    second = first + (1 if interleaved else half)
    y, size = x.clone(), x.abs()
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return y, size


def off(size):
    return 48 * 2.0 ** -24 * size


def assert_close(got, ref, size):
    step = torch.finfo(got.dtype).eps / 2 if got.dtype != FP else 2.0 ** -24
    err = off(size)
    assert ((got.double() - ref).abs() <= err + step * (ref.abs() + err) + TINY[got.dtype]).all()


def inputs(seed, N, Hq, H, D, rot, dtype, positions=4096, weights="both", weight_dtype=None, packed=True):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    qkv = torch.empty((N, (Hq + 2 * H) * D), device="cuda").normal_(generator=g).mul_(2).to(dtype)
    q, k, v = (t.view(N, -1, D) for t in qkv.split([Hq * D, H * D, H * D], 1))
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    w = [torch.empty(D, device="cuda").uniform_(0.3, 1.7, generator=g).to(weight_dtype or dtype) for _ in range(2)]
    qw, kw = (w[0] if weights in ("both", "q") else None), (w[1] if weights in ("both", "k") else None)
    pos = torch.randint(0, positions, (N,), device="cuda", dtype=torch.int32, generator=g)
    return q, k, v, pos, rotary_table(positions, rot, device="cuda"), qw, kw


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (64, 64), (64, 32), (80, 80), (80, 32), (96, 96), (112, 56),
                                   (120, 120), (120, 30), (256, 256), (192, 128), (32, 2), (8, 8), (8, 6), (256, 250),
                                   (240, 24)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_shapes(dtype, D, rot, interleaved):
    for N, Hq, H in ((1, 8, 2), (37, 5, 1)):
        q, k, v, pos, cs, qw, kw = inputs(D + rot + N, N, Hq, H, D, rot, dtype)
        qo, ko = kernels.qk_norm_rope(q, k, pos, cs, qw, kw, 1e-5, interleaved)
        assert qo.is_contiguous() and ko.is_contiguous() and qo.dtype == dtype
        assert_close(qo, *reference(q, qw, pos, cs, 1e-5, interleaved))
        assert_close(ko, *reference(k, kw, pos, cs, 1e-5, interleaved))


@pytest.mark.parametrize("weights,weight_dtype", [("none", None), ("q", None), ("k", FP), ("both", FP)])
@pytest.mark.parametrize("heads", [(32, 8), (28, 4), (1, 1), (14, 2), (3, 3), (64, 8)])
def test_weights_and_heads(weights, weight_dtype, heads):
    q, k, v, pos, cs, qw, kw = inputs(5, 23, *heads, 128, 128, BF, weights=weights, weight_dtype=weight_dtype)
    qo, ko = kernels.qk_norm_rope(q, k, pos, cs, qw, kw)
    assert_close(qo, *reference(q, qw, pos, cs, 1e-6, False))
    assert_close(ko, *reference(k, kw, pos, cs, 1e-6, False))


def test_without_norm_and_at_position_zero_the_bits_stay():
    q, k, v, pos, cs, _, _ = inputs(6, 40, 8, 2, 128, 64, BF, weights="none")
    qo, ko = kernels.qk_norm_rope(q, k, torch.zeros_like(pos), cs)
    assert torch.equal(qo, q) and torch.equal(ko, k)
    qo, ko = kernels.qk_norm_rope(q, k, pos, cs)
    assert torch.equal(qo[..., 64:], q[..., 64:]) and not torch.equal(qo[..., :64], q[..., :64])


def test_positions_outside_the_table_and_index_types():
    q, k, v, pos, cs, qw, kw = inputs(7, 9, 4, 2, 64, 64, HF, positions=50)
    pos = torch.tensor([-1, -2 ** 31, 0, 49, 50, 2 ** 31 - 1, 7, 8, 9], device="cuda")
    for p in (pos.int(), pos, pos.int()[:, None].expand(-1, 2)[:, 0]):
        qo, ko = kernels.qk_norm_rope(q, k, p, cs, qw, kw)
        assert_close(qo, *reference(q, qw, pos, cs, 1e-6, False))
        assert_close(ko, *reference(k, kw, pos, cs, 1e-6, False))


def test_strides_and_alignment():
    # Rows that are not 16-byte aligned, heads out of order, a misaligned table and weights: copies, the same result.
    q, k, v, pos, cs, qw, kw = inputs(8, 21, 6, 3, 64, 64, BF, packed=False)
    want = kernels.qk_norm_rope(q, k, pos, cs, qw, kw)
    buf = torch.zeros(21 * 6 * 64 + 1, dtype=BF, device="cuda")
    q1 = buf[1:].view(21, 6, 64).copy_(q)
    wide = torch.zeros(21, 3 * 64 + 3, dtype=BF, device="cuda")
    k1 = wide[:, :192].unflatten(1, (3, 64)).copy_(k)
    q2 = q.transpose(0, 1).contiguous().transpose(0, 1)
    cs1 = torch.zeros(cs.numel() + 1, device="cuda")[1:].view_as(cs).copy_(cs)
    w1 = torch.zeros(65, dtype=BF, device="cuda")[1:].copy_(qw)
    for a in ((q1, k, pos, cs, qw, kw), (q, k1, pos, cs, qw, kw), (q2, k, pos, cs, qw, kw), (q, k, pos, cs1, w1, kw)):
        got = kernels.qk_norm_rope(*a)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_zero_tokens_and_special_values():
    q, k, v, pos, cs, qw, kw = inputs(9, 4, 4, 2, 64, 64, BF)
    qo, ko = kernels.qk_norm_rope(q[:0], k[:0], pos[:0], cs, qw, kw)
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)
    q = q.clone()
    q[1, 2, 5] = float("inf")
    q[2, 3] = 0
    qo, _ = kernels.qk_norm_rope(q, k, pos, cs, qw, kw)
    assert qo[1, 2].isnan().any() and (qo[2, 3] == 0).all()
    # The other heads and tokens are untouched by it.
    ref, size = reference(q, qw, pos, cs, 1e-6, False)
    keep = torch.ones(4, 4, dtype=torch.bool, device="cuda")
    keep[1, 2] = False
    assert_close(qo[keep], ref[keep], size[keep])


# ---- with the append -----------------------------------------------------------------


def slots_of(kind, rng, N, nb, bs):
    """Slots that fill blocks in order at ragged prompts, scattered ones, or a mix with skipped tokens."""
    if kind == "scatter":
        return rng.permutation(nb * bs)[:N]
    ids, out, at = rng.permutation(nb), [], 0
    while len(out) < N:
        n = int(rng.integers(1, 4 * bs))
        t = np.arange(n)
        need = -(-n // bs)
        if at + need > nb:
            break
        out += (ids[at + t // bs] * bs + t % bs).tolist()
        at += need
    out = np.array((out + [-1] * N)[:N])
    if kind == "skips":
        out[rng.random(N) < 0.1] = -1
        out[rng.random(N) < 0.05] = nb * bs + 3
    return out


PAIRS = [(BF, BF), (HF, HF), (FP, FP), (FP, BF), (FP, HF), (BF, torch.uint8), (HF, torch.uint8), (FP, torch.uint8)]


def caches(kind, nb, bs, H, D, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = 16 // torch.empty(0, dtype=dtype).element_size()
    shapes = {"paged": ((nb, H, D // x, bs, x), (nb, H, D, bs)), "rows": ((nb * bs, H, D),) * 2,
              "flash": ((nb, bs, H, D),) * 2}[kind]
    make = lambda s: (torch.randint(0, 100, s, device="cuda", dtype=torch.uint8, generator=g) if dtype == torch.uint8
                      else torch.empty(s, device="cuda").normal_(generator=g).to(dtype))
    return make(shapes[0]), make(shapes[1])


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{str(p[0])[6:]}-{str(p[1])[6:]}")
@pytest.mark.parametrize("kind,bs", [("paged", 8), ("paged", 16), ("paged", 32), ("rows", 1), ("flash", 16)])
@pytest.mark.parametrize("slots", ["prompts", "scatter", "skips"])
def test_cache_holds_what_the_append_would_store(pair, kind, bs, slots):
    # The append of the rotated keys, computed in float32 so that they are rounded once, gives the same caches: the
    # float32 kernel's keys are within the bounds above, and where the two kernels' roundings part, the codes are
    # those of neighbouring values.
    dtype, cdtype = pair
    rng = np.random.default_rng(3)
    for N, Hq, H, D, rot in ((133, 8, 2, 128, 128), (3, 5, 5, 64, 32), (70, 4, 1, 80, 80)):
        nb = max(2, 4 * N // bs)
        q, k, v, pos, cs, qw, kw = inputs(N, N, Hq, H, D, rot, dtype)
        slot = torch.tensor(slots_of(slots, rng, N, nb, bs), dtype=torch.int32, device="cuda")
        kc, vc = caches(kind, nb, bs, H, D, cdtype, N)
        rk, rv = kc.clone(), vc.clone()
        scales = dict(k_scale=0.1, v_scale=0.03) if cdtype == torch.uint8 else {}
        qo, k2, v2 = kernels.qk_norm_rope_and_cache(q, k, v, pos, cs, kc, vc, slot, qw, kw, **scales)
        assert k2 is kc and v2 is vc
        assert_close(qo, *reference(q, qw, pos, cs, 1e-6, False))
        view = (lambda t: t.view(-1, H, D)) if kind == "flash" else (lambda t: t)
        key, size = reference(k, kw, pos, cs, 1e-6, False)
        kernels.reshape_and_cache(key.float() if cdtype == torch.uint8 or dtype == FP else key.to(dtype),
                                  v.float() if cdtype == torch.uint8 or dtype == FP else v, view(rk), view(rv), slot,
                                  **scales)
        assert torch.equal(vc, rv)
        if cdtype == torch.uint8:
            got, want = kc.cpu().numpy(), rk.cpu().numpy()
            # One rounding apart at most, and rarely: magnitudes are ordered as their codes.
            place = lambda c: np.where(c & 0x80, -(c & 0x7f).astype(np.int64), c & 0x7f)
            assert np.abs(place(got) - place(want)).max() <= 1
            assert (got != want).mean() < 1e-3
        else:
            # Two values within the float32 bound of each other round to the same element or to neighbours.
            step = torch.finfo(cdtype).eps
            ref = rk.double()
            assert ((kc.double() - ref).abs() <= step * ref.abs() + 2 * off(size.max()) + TINY[cdtype] * 2).all()
        # What no token names is as it was.
        named = torch.zeros(nb * bs, dtype=torch.bool, device="cuda")
        ok = (slot >= 0) & (slot < nb * bs)
        named[slot[ok].long()] = True
        k0, _ = caches(kind, nb, bs, H, D, cdtype, N)
        if kind == "paged":
            rows = lambda t: t.permute(0, 3, 1, 2, 4).reshape(nb * bs, -1)
        else:
            rows = lambda t: t.reshape(nb * bs, -1)
        assert torch.equal(rows(kc)[~named], rows(k0)[~named])


def test_values_keep_their_bits():
    q, k, v, pos, cs, qw, kw = inputs(11, 48, 4, 2, 64, 64, BF)
    bits = torch.randint(-2 ** 15, 2 ** 15, v.shape, dtype=torch.int16, device="cuda")
    v = bits.view(BF)
    for kind, bs in (("paged", 16), ("rows", 1)):
        kc, vc = caches(kind, 8 if kind == "paged" else 128, bs, 2, 64, BF, 1)
        slot = torch.arange(16, 64, dtype=torch.int32, device="cuda")
        kernels.qk_norm_rope_and_cache(q, k, v, pos, cs, kc, vc, slot, qw, kw)
        rows = vc.permute(0, 3, 1, 2).reshape(-1, 2, 64) if kind == "paged" else vc
        assert torch.equal(rows.view(torch.int16)[16:64], bits)


def test_fp8_codes_against_the_encoder():
    # Each code is the encoder's of some value within the bounds of the formula.
    q, k, v, pos, cs, qw, kw = inputs(12, 64, 4, 2, 128, 128, BF)
    kc, vc = caches("rows", 64, 1, 2, 128, torch.uint8, 2)
    kernels.qk_norm_rope_and_cache(q, k, v, pos, cs, kc, vc, torch.arange(64, dtype=torch.int32, device="cuda"), qw, kw,
                                   k_scale=0.02, v_scale=0.02)
    ref, size = reference(k, kw, pos, cs, 1e-6, False)
    err = off(size) + ref.abs() * 2.0 ** -23
    lo, hi = ((ref + e).float().div(0.02).cpu().numpy() for e in (-err, err))
    got = kc.cpu().numpy()
    assert ((got == orc.fp8_e4m3_encode(lo)) | (got == orc.fp8_e4m3_encode(hi))).all()


def test_other_streams_and_captured_replays():
    N = 50
    q, k, v, pos, cs, qw, kw = inputs(13, N, 8, 2, 128, 128, BF, packed=False)
    kc, vc = caches("paged", 20, 16, 2, 128, BF, 3)
    slot = torch.arange(N, dtype=torch.int32, device="cuda") + 5
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        qo, _, _ = kernels.qk_norm_rope_and_cache(q, k, v, pos, cs, kc, vc, slot, qw, kw)
    for seed in (14, 15, 16):
        a = inputs(seed, N, 8, 2, 128, 128, BF, packed=False)
        for dst, src in zip((q, k, v, pos), a):
            dst.copy_(src)
        ek, ev = caches("paged", 20, 16, 2, 128, BF, 3)
        kc.copy_(ek), vc.copy_(ev)
        torch.cuda.synchronize()
        graph.replay()
        want, ek, ev = kernels.qk_norm_rope_and_cache(*a[:5], ek, ev, slot, qw, kw)
        torch.cuda.synchronize()
        assert torch.equal(qo, want) and torch.equal(kc, ek) and torch.equal(vc, ev)
    with torch.cuda.stream(stream):
        again = kernels.qk_norm_rope(q, k, pos, cs, qw, kw)
    stream.synchronize()
    assert torch.equal(again[0], want)
