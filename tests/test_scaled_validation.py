"""Argument checks of the caches with a scale per block and head, of attention over them
and of attention of packed prompts, on CPU tensors and at the C ABI: nothing here reaches a
launch.  The plain forms that the GPU tests compare with are checked here too."""

import math

import numpy as np
import pytest
import torch

import pkv_scaled as ps
from sglang_mlx_amd import _lib, kernels

I32, BF, U8 = torch.int32, torch.bfloat16, torch.uint8
P = 4096  # an aligned address that no accepted call is made with


def caches(nb=4, H=2, D=64, bs=16):
    return dict(key_cache=torch.zeros(nb, H, D // 16, bs, 16, dtype=U8), value_cache=torch.zeros(nb, H, D, bs, dtype=U8),
                kv_scales=torch.zeros(nb, H, 2))


def store_args(**kw):
    a = dict(key=torch.zeros(5, 2, 64, dtype=BF), value=torch.zeros(5, 2, 64, dtype=BF), **caches(),
             block_tables=torch.zeros(2, 3, dtype=I32), context_lens=torch.tensor([20, 7], dtype=I32),
             query_start_loc=torch.tensor([0, 3, 5], dtype=I32))
    a.update(kw)
    return a


def read_args(**kw):
    a = dict(**caches(), block_tables=torch.zeros(2, 3, dtype=I32), start_loc=torch.tensor([0, 20, 27], dtype=I32),
             num_tokens=27)
    a.update(kw)
    return a


def attend_args(**kw):
    a = dict(query=torch.zeros(5, 8, 64, dtype=BF), **caches(), block_tables=torch.zeros(2, 3, dtype=I32),
             context_lens=torch.tensor([20, 7], dtype=I32), query_start_loc=torch.tensor([0, 3, 5], dtype=I32),
             num_kv_heads=2, scale=0.1, block_size=16, max_seq_len=48, max_query_len=3)
    a.update(kw)
    return a


def prompt_args(**kw):
    a = dict(query=torch.zeros(5, 8, 64, dtype=BF), key=torch.zeros(5, 2, 64, dtype=BF),
             value=torch.zeros(5, 2, 64, dtype=BF), query_start_loc=torch.tensor([0, 3, 5], dtype=I32), scale=0.1,
             max_query_len=3)
    a.update(kw)
    return a


CACHES = [  # what the calls over these caches refuse alike
    (dict(key_cache=torch.zeros(4, 2, 4, 16, 16, dtype=BF)), ValueError, "must be uint8"),
    (dict(value_cache=torch.zeros(4, 2, 64, 16, dtype=torch.int8)), ValueError, "must be uint8"),
    (dict(key_cache=torch.zeros(4, 2, 8, 16, 8, dtype=U8)), ValueError, "key_cache must have shape"),
    (dict(value_cache=torch.zeros(4, 2, 64, 8, dtype=U8)), ValueError, "value_cache must have shape"),
    (dict(value_cache=torch.zeros(4, 16, 2, 64, 1, dtype=U8)), ValueError, "paged layout"),
    (caches(bs=64), ValueError, "Unsupported head_size/block_size"),
    (caches(nb=0), ValueError, "Unsupported head_size/block_size"),
    (dict(kv_scales=torch.zeros(4, 2, 2, dtype=torch.float64)), ValueError, "kv_scales must be"),
    (dict(kv_scales=torch.zeros(4, 2)), ValueError, "kv_scales must be"),
    (dict(kv_scales=torch.zeros(4, 2, 4)[..., ::2]), ValueError, "kv_scales must be"),
    (dict(kv_scales=None), TypeError, "Expected torch.Tensor"),
    (dict(block_tables=torch.zeros(6, dtype=I32)), ValueError, "2D"),
    (dict(block_tables=torch.zeros(2, 3)), ValueError, "integer dtype"),
    (dict(), RuntimeError, "GPU-only"),
]


@pytest.mark.parametrize("kw,err,msg", CACHES + [
    (dict(key=torch.zeros(5, 128, dtype=BF)), ValueError, "key and value must have shape"),
    (dict(value=torch.zeros(4, 2, 64, dtype=BF)), ValueError, "key and value must have shape"),
    (dict(value=torch.zeros(5, 2, 64)), ValueError, "dtypes differ"),
    (dict(key=torch.zeros(5, 2, 64, dtype=torch.float64), value=torch.zeros(5, 2, 64, dtype=torch.float64)), ValueError,
     "dtype"),
    (dict(key=torch.zeros(5, 2, 72, dtype=BF), value=torch.zeros(5, 2, 72, dtype=BF)), ValueError, "key_cache must have"),
    (dict(context_lens=torch.zeros(3, dtype=I32)), ValueError, "of the same sequences"),
    (dict(context_lens=torch.zeros(2)), ValueError, "integer dtype"),
    (dict(query_start_loc=torch.zeros(2, dtype=I32)), ValueError, "query_start_loc must have shape"),
    (dict(query_start_loc=None), TypeError, "Expected torch.Tensor"),
    (dict(block_tables=torch.zeros(2, 0, dtype=I32)), ValueError, "must have a column"),
    (dict(key_cache=torch.zeros(8, 2, 4, 16, 16, dtype=U8)[::2]), ValueError, "must be contiguous"),
])
def test_store_checks(kw, err, msg):
    with pytest.raises(err, match=msg):
        kernels.quantize_and_cache(**store_args(**kw))


@pytest.mark.parametrize("kw,err,msg", CACHES + [
    (dict(start_loc=torch.zeros(2, dtype=I32)), ValueError, "start_loc must have shape"),
    (dict(start_loc=torch.zeros(3)), ValueError, "integer dtype"),
    (dict(dtype=torch.float64), ValueError, "Unsupported dtype"),
    (dict(num_tokens=-1), ValueError, "num_tokens must be"),
    (dict(num_tokens=1 << 31), ValueError, "num_tokens must be"),
    (dict(block_tables=torch.zeros(2, 0, dtype=I32)), ValueError, "must have a column"),
    (dict(value_cache=torch.zeros(8, 2, 64, 16, dtype=U8)[::2]), ValueError, "must be contiguous"),
])
def test_read_checks(kw, err, msg):
    with pytest.raises(err, match=msg):
        kernels.dequantize_cache(**read_args(**kw))


@pytest.mark.parametrize("kw,err,msg", CACHES + [
    (dict(query=torch.zeros(5, 512, dtype=BF)), ValueError, "query must have shape"),
    (dict(query=torch.zeros(5, 7, 64, dtype=BF)), ValueError, "divisible"),
    (dict(num_kv_heads=0), ValueError, "divisible"),
    (dict(query=torch.zeros(5, 8, 64)), ValueError, "Unsupported query dtype"),
    (dict(query=torch.zeros(5, 8, 120, dtype=BF)), ValueError, "key_cache must have shape"),
    (dict(context_lens=torch.zeros(3, dtype=I32)), ValueError, "sequence counts differ"),
    (dict(query_start_loc=None), ValueError, "sequence counts differ"),
    (dict(query_start_loc=None, query=torch.zeros(2, 8, 64, dtype=BF)), ValueError, "one token per sequence"),
    (dict(query_start_loc=torch.zeros(4, dtype=I32)), ValueError, "query_start_loc must have shape"),
    (dict(query_start_loc=torch.zeros(3)), ValueError, "integer dtype"),
    (dict(block_size=8), ValueError, "do not match block_size"),
    (dict(value_cache=torch.zeros(4, 2, 16, 64, dtype=U8).transpose(2, 3)), ValueError, "contiguous within"),
    (dict(max_seq_len=0), ValueError, "max_seq_len must be positive"),
    (dict(max_seq_len=49), ValueError, "block table capacity"),
    (dict(max_query_len=0), ValueError, "max_query_len must be positive"),
    (dict(window=-1), ValueError, "non-negative"),
    (dict(num_sinks=-1), ValueError, "non-negative"),
    (dict(scale=math.nan), ValueError, "scale must be finite"),
    (dict(scale=-math.inf), ValueError, "scale must be finite"),
])
def test_attention_checks(kw, err, msg):
    with pytest.raises(err, match=msg):
        kernels.paged_attention_scaled(**attend_args(**kw))


@pytest.mark.parametrize("kw,err,msg", [
    (dict(query=torch.zeros(5, 512, dtype=BF)), ValueError, "query must have shape"),
    (dict(key=torch.zeros(5, 128, dtype=BF)), ValueError, "key and value must have shape"),
    (dict(value=torch.zeros(5, 1, 64, dtype=BF)), ValueError, "key and value must have shape"),
    (dict(query=torch.zeros(5, 8, 128, dtype=BF)), ValueError, "head sizes differ"),
    (dict(query=torch.zeros(5, 7, 64, dtype=BF)), ValueError, "divisible"),
    (dict(query=torch.zeros(5, 8, 64)), ValueError, "Unsupported dtype"),
    (dict(key=torch.zeros(5, 2, 64, dtype=torch.float16)), ValueError, "dtypes differ"),
    (dict(value=torch.zeros(5, 2, 64)), ValueError, "dtypes differ"),
    (dict(query=torch.zeros(5, 8, 72, dtype=BF), key=torch.zeros(5, 2, 72, dtype=BF),
          value=torch.zeros(5, 2, 72, dtype=BF)), ValueError, "Unsupported head_size"),
    (dict(query_start_loc=torch.zeros(0, dtype=I32)), ValueError, "query_start_loc must have shape"),
    (dict(query_start_loc=torch.zeros(3, 1, dtype=I32)), ValueError, "query_start_loc must have shape"),
    (dict(query_start_loc=torch.zeros(3)), ValueError, "integer dtype"),
    (dict(key=torch.zeros(6, 2, 64, dtype=BF), value=torch.zeros(6, 2, 64, dtype=BF)), ValueError, "as many keys"),
    (dict(max_key_len=4), ValueError, "max_key_len is max_query_len"),
    (dict(key_start_loc=torch.zeros(3, dtype=I32)), ValueError, "needs max_key_len"),
    (dict(key_start_loc=torch.zeros(2, dtype=I32), max_key_len=4), ValueError, "key_start_loc must have shape"),
    (dict(key_start_loc=torch.zeros(3), max_key_len=4), ValueError, "integer dtype"),
    (dict(key_start_loc=torch.zeros(3, dtype=I32), max_key_len=0), ValueError, "must be positive"),
    (dict(key_start_loc=[0, 3, 5], max_key_len=4), TypeError, "Expected torch.Tensor"),
    (dict(max_query_len=0), ValueError, "must be positive"),
    (dict(window=-1), ValueError, "non-negative"),
    (dict(num_sinks=-1), ValueError, "non-negative"),
    (dict(scale=math.inf), ValueError, "scale must be finite"),
    (dict(query=None), TypeError, "Expected torch.Tensor"),
    (dict(), RuntimeError, "GPU-only"),
])
def test_prompt_checks(kw, err, msg):
    with pytest.raises(err, match=msg):
        kernels.prompt_attention(**prompt_args(**kw))


def refusals(name, base, cases):
    lib = _lib.lib()
    for kw, code, msg in cases:
        assert set(kw) <= set(base), kw
        st = getattr(lib, name)(*{**base, **kw}.values())
        assert st == code and msg in lib.pkv_last_error().decode(), (kw, st, lib.pkv_last_error())


BIG = (1 << 31) - 1
PAGES = [
    (dict(N=-1), 1, "non-negative"), (dict(B=-1), 1, "non-negative"), (dict(H=0), 1, "num_kv_heads"),
    (dict(D=120), 2, "Unsupported head_size"), (dict(D=48), 2, "Unsupported head_size"),
    (dict(bs=64), 2, "Unsupported head_size"), (dict(W=0), 1, "block"), (dict(nb=0), 1, "num_blocks"),
    (dict(dt=_lib.PKV_FP8_E4M3), 1, "dtype"), (dict(dt=77), 1, "dtype"),
    (dict(kc=None), 1, "null buffer"), (dict(vc=None), 1, "null buffer"), (dict(sc=None), 1, "null buffer"),
    (dict(bt=None), 1, "null buffer"), (dict(start=None), 1, "null buffer"),
    (dict(kc=P + 8), 1, "aligned"), (dict(vc=P + 8), 1, "aligned"), (dict(sc=P + 4), 1, "aligned"),
    (dict(N=BIG, B=BIG, H=BIG), 2, "launch"),
]


def test_store_abi_refusals():
    base = dict(k=P, v=P, kc=P, vc=P, sc=P, bt=P, ctx=P, start=P, N=5, B=2, H=2, D=64, bs=16, W=3, nb=4, ks=128, vs=128,
                dt=_lib.PKV_BF16, stream=None)
    refusals("pkv_quantize_and_cache", base, PAGES + [
        (dict(k=None), 1, "null buffer"), (dict(v=None), 1, "null buffer"), (dict(ctx=None), 1, "null buffer"),
        (dict(ks=127), 1, "rows must be"), (dict(vs=120), 1, "rows must be"), (dict(ks=132), 1, "rows must be"),
        (dict(k=P + 8), 1, "rows must be"), (dict(v=P + 2), 1, "rows must be"),
        (dict(vs=130, dt=_lib.PKV_F32), 1, "rows must be"),
    ])
    lib = _lib.lib()
    assert lib.pkv_quantize_and_cache(*{**base, "N": 0}.values()) == 0
    assert lib.pkv_quantize_and_cache(*{**base, "B": 0}.values()) == 0


def test_read_abi_refusals():
    base = dict(ko=P, vo=P, kc=P, vc=P, sc=P, bt=P, start=P, N=27, B=2, H=2, D=64, bs=16, W=3, nb=4, dt=_lib.PKV_BF16,
                stream=None)
    refusals("pkv_dequantize_cache", base, PAGES + [
        (dict(ko=None), 1, "null buffer"), (dict(vo=None), 1, "null buffer"),
        (dict(ko=P + 8), 1, "16-byte aligned"), (dict(vo=P + 2), 1, "16-byte aligned"),
    ])
    assert _lib.lib().pkv_dequantize_cache(*{**base, "N": 0}.values()) == 0


def test_attention_abi_refusals():
    base = dict(out=P, q=P, kc=P, vc=P, sc=P, bt=P, ctx=P, start=P, N=5, B=2, Hq=8, H=2, D=64, bs=16, W=3, max_seq=48,
                max_query=3, window=0, sinks=0, nb=4, scale=0.1, qs=512, kbs=2048, khs=1024, vbs=2048, vhs=1024, ws=P,
                wsb=1 << 30, dt=_lib.PKV_BF16, stream=None)
    refusals("pkv_paged_attention_scaled", base, [
        (dict(N=-1), 1, "non-negative"), (dict(B=-1), 1, "non-negative"), (dict(H=3), 1, "divisible"),
        (dict(H=0), 1, "divisible"), (dict(Hq=0), 1, "divisible"), (dict(max_seq=0), 1, "max_seq_len must be positive"),
        (dict(max_seq=(1 << 30) + 1), 2, "at most 2^30"), (dict(max_query=0), 1, "max_query_len"),
        (dict(window=-1), 1, "window"), (dict(sinks=-1), 1, "window"), (dict(start=None), 1, "one token per sequence"),
        (dict(start=None, N=2), 1, "one token per sequence"), (dict(D=120), 2, "Unsupported head_size"),
        (dict(D=100), 2, "Unsupported head_size"), (dict(bs=64), 2, "Unsupported head_size"),
        (dict(max_seq=49), 1, "capacity"), (dict(W=0), 1, "capacity"), (dict(dt=_lib.PKV_F32), 2, "query dtype"),
        (dict(scale=math.nan), 1, "scale must be finite"), (dict(scale=3e38), 1, "scale must be finite"),
        (dict(nb=0), 1, "num_blocks"), (dict(N=1 << 28), 2, "launch"),
        (dict(B=BIG, N=BIG >> 4, W=1 << 25, max_seq=1 << 29), 2, "launch"), (dict(max_query=BIG), 2, "launch"),
        (dict(max_query=BIG, Hq=1 << 27, H=1, N=3, qs=1 << 33), 2, "launch"),
        (dict(out=None), 1, "null buffer"), (dict(q=None), 1, "null buffer"), (dict(kc=None), 1, "null buffer"),
        (dict(vc=None), 1, "null buffer"), (dict(sc=None), 1, "null buffer"), (dict(bt=None), 1, "null buffer"),
        (dict(ctx=None), 1, "null buffer"), (dict(out=P + 8), 1, "out must be"), (dict(qs=511), 1, "query rows"),
        (dict(q=P + 2), 1, "query rows"), (dict(qs=516), 1, "query rows"), (dict(kc=P + 8), 1, "not aligned"),
        (dict(vc=P + 8), 1, "not aligned"), (dict(kbs=2056), 1, "not aligned"), (dict(khs=1032), 1, "not aligned"),
        (dict(vbs=2056), 1, "not aligned"), (dict(vhs=1032), 1, "not aligned"), (dict(sc=P + 4), 1, "not aligned"),
        (dict(ws=None), 1, "workspace is smaller"), (dict(wsb=100), 1, "workspace is smaller"),
        (dict(ws=P + 4), 1, "16-byte aligned"),
    ])
    lib = _lib.lib()
    assert lib.pkv_paged_attention_scaled(*{**base, "N": 0}.values()) == 0
    size = lib.pkv_paged_attention_scaled_workspace_size
    assert size(2, 8, 2, 64, 48, 3, 0, 0) >= _lib.PKV_COUNTER_BYTES
    for bad in [(-1, 8, 2, 64, 48, 3, 0, 0), (2, 8, 3, 64, 48, 3, 0, 0), (2, 8, 2, 0, 48, 3, 0, 0),
                (2, 8, 2, 64, 0, 3, 0, 0), (2, 8, 2, 64, 48, 0, 0, 0), (2, 8, 2, 64, 48, 3, -1, 0),
                (2, 8, 2, 64, 48, 3, 0, -1), (2, 8, 2, 64, (1 << 30) + 1, 3, 0, 0)]:
        assert size(*bad) == 0


def test_attention_workspace_is_that_of_the_arguments():
    """Also where max_query_len exceeds the call's tokens: fewer, longer crews need less room than many short ones."""
    lib = _lib.lib()
    need = lib.pkv_paged_attention_scaled_workspace_size(64, 64, 8, 128, 4096, 600, 0, 0)
    a = [P, P, P, P, P, P, P, P, 64, 64, 64, 8, 128, 16, 256, 4096, 600, 0, 0, 4, 0.1, 8192, 16384, 2048, 16384, 2048,
         P + 4, need, _lib.PKV_BF16, None]
    assert lib.pkv_paged_attention_scaled(*a) == 1 and b"16-byte aligned" in lib.pkv_last_error()
    a[27] = need - 1
    assert lib.pkv_paged_attention_scaled(*a) == 1 and b"workspace is smaller" in lib.pkv_last_error()


def test_prompt_abi_refusals():
    base = dict(out=P, q=P, k=P, v=P, start=P, kstart=None, N=5, T=5, B=2, Hq=8, H=2, D=64, max_query=3, max_key=3,
                window=0, sinks=0, scale=0.1, qs=512, ks=128, vs=128, ws=P, wsb=1 << 30, dt=_lib.PKV_BF16, stream=None)
    refusals("pkv_prompt_attention", base, [
        (dict(N=-1), 1, "non-negative"), (dict(T=-1), 1, "non-negative"), (dict(B=-1), 1, "non-negative"),
        (dict(Hq=0), 1, "divisible"), (dict(H=0), 1, "divisible"), (dict(H=3), 1, "divisible"),
        (dict(max_query=0), 1, "must be positive"), (dict(max_key=0), 1, "must be positive"),
        (dict(T=(1 << 30) + 1), 2, "at most 2^30"), (dict(window=-1), 1, "window"), (dict(sinks=-1), 1, "window"),
        (dict(T=6), 1, "as many keys"), (dict(D=72), 2, "Unsupported head_size"), (dict(dt=_lib.PKV_F32), 2, "dtype"),
        (dict(scale=math.inf), 1, "scale must be finite"), (dict(scale=3e38), 1, "scale must be finite"),
        (dict(qs=511), 1, "smaller than a row"), (dict(ks=127), 1, "smaller than a row"),
        (dict(vs=0), 1, "smaller than a row"), (dict(ks=(1 << 24) + 8), 2, "at most 2^24"),
        (dict(vs=1 << 25), 2, "at most 2^24"), (dict(N=1 << 28, T=1 << 28), 2, "grid limit"),
        (dict(B=BIG, Hq=BIG, H=BIG, D=32, qs=BIG * 32, ks=BIG * 32, vs=BIG * 32), 2, "2^24"),
        (dict(B=BIG), 2, "grid limit"),
        (dict(out=None), 1, "null buffer"), (dict(q=None), 1, "null buffer"), (dict(k=None), 1, "null buffer"),
        (dict(v=None), 1, "null buffer"), (dict(start=None), 1, "null buffer"), (dict(out=P + 8), 1, "aligned"),
        (dict(q=P + 2), 1, "aligned"), (dict(k=P + 8), 1, "aligned"), (dict(v=P + 4), 1, "aligned"),
        (dict(qs=516), 1, "aligned"), (dict(ks=132), 1, "aligned"), (dict(vs=130), 1, "aligned"),
        (dict(ws=None), 1, "workspace is smaller"), (dict(wsb=16), 1, "workspace is smaller"),
        (dict(ws=P + 4), 1, "16-byte aligned"),
    ])
    lib = _lib.lib()
    assert lib.pkv_prompt_attention(*{**base, "N": 0, "T": 0}.values()) == 0
    size = lib.pkv_prompt_attention_workspace_size
    assert size(5, 2, 8, 2, 64, 3, 3, 0, 0) >= _lib.PKV_COUNTER_BYTES
    # A few rows behind a long context are split: their states need room.
    assert size(4, 1, 28, 4, 128, 4, 32768, 0, 0) > _lib.PKV_COUNTER_BYTES + 4 * 28 * 2 * 130 * 4
    for bad in [(-1, 2, 8, 2, 64, 3, 3, 0, 0), (5, -1, 8, 2, 64, 3, 3, 0, 0), (5, 2, 8, 3, 64, 3, 3, 0, 0),
                (5, 2, 8, 2, 0, 3, 3, 0, 0), (5, 2, 8, 2, 64, 0, 3, 0, 0), (5, 2, 8, 2, 64, 3, 0, 0, 0),
                (5, 2, 8, 2, 64, 3, 3, -1, 0), (5, 2, 8, 2, 64, 3, 3, 0, -1)]:
        assert size(*bad) == 0


# ---- the plain forms ------------------------------------------------------------------


def test_codes_are_those_of_the_format():
    want = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    values = torch.from_numpy(ps.VALUES)
    finite = values.isfinite()
    # Below exponent 15 the codes are those of torch's type of 4 exponent bits.
    assert torch.equal(want.view(torch.float8_e4m3fn).double()[finite], values[finite])
    assert np.array_equal(ps.encode(ps.VALUES[finite.numpy()]), want.numpy()[finite.numpy()])


def test_encoding_takes_the_nearest_and_the_even_one():
    x = np.concatenate([np.linspace(-240, 240, 20001), 2.0 ** np.linspace(-14, 7, 5001)])
    finite = np.sort(np.unique(ps.VALUES[np.isfinite(ps.VALUES)]))
    got = ps.VALUES[ps.encode(x)]
    best = np.abs(finite[None] - x[:, None]).min(1)
    assert (np.abs(got - x) == best).all()
    assert np.array_equal(ps.encode([17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10]), ps.encode([16.0, 20.0, 0.0, 2.0 ** -8]))


def test_scale_rule():
    for a, want in [(0.0, 2.0 ** -126), (240.0, 1.0), (241.0, 2.0), (120.0, 0.5), (1e-40, 2.0 ** -126),
                    (3.3895313892515355e38, 2.0 ** 121)]:
        assert ps.scale_for(a) == want


def test_plain_attention_is_attention():
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(9, h, 16, generator=g, dtype=torch.float64).to(BF) for h in (4, 2, 2))
    out, off = ps.attend(q, k.double(), v.double(), 0, 0.25, window=4, sinks=1)
    want = torch.nn.functional.scaled_dot_product_attention(
        q.double().transpose(0, 1), k.double().transpose(0, 1).repeat_interleave(2, 0),
        v.double().transpose(0, 1).repeat_interleave(2, 0), scale=0.25,
        attn_mask=torch.tensor([[j <= i and (j > i - 4 or j < 1) for j in range(9)] for i in range(9)]))
    assert (out - want.transpose(0, 1)).abs().max() < 1e-14 and (off > 0).all() and off.max() < 0.05
