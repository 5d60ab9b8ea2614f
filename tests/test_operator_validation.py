"""Argument checks of the operators around the cache (step tables, norm and
rotation, window decode, attention of new tokens) on CPU tensors and at the C
ABI: nothing here reaches a launch.  The rotary tables and the host side of
RequestBlocks, which need no GPU, are tested here too."""

import ctypes
import math

import numpy as np
import pytest
import torch

from sglang_mlx_amd import _lib, kernels
from sglang_mlx_amd.rotary import rotary_frequencies, rotary_table
from sglang_mlx_amd.srt.mem_cache import BlockAllocator, RequestBlocks

I32 = torch.int32


def tables_args(**kw):
    a = dict(request_blocks=torch.full((4, 8), -1, dtype=I32), rows=torch.tensor([0, 2], dtype=I32),
             context_lens=torch.tensor([5, 3], dtype=I32), query_lens=torch.tensor([1, 3], dtype=I32),
             new_blocks=torch.tensor([7, 9], dtype=I32), block_size=16, num_tokens=4)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,err,msg", [
    (dict(request_blocks=torch.zeros(8, dtype=I32)), ValueError, "request_blocks must have shape"),
    (dict(context_lens=torch.zeros(3, dtype=I32)), ValueError, "rows, context_lens and query_lens"),
    (dict(rows=torch.zeros(2, 1, dtype=I32)), ValueError, "rows, context_lens and query_lens"),
    (dict(new_blocks=torch.zeros(2, 1, dtype=I32)), ValueError, "new_blocks must be 1-D"),
    (dict(request_blocks=torch.zeros(4, 8, dtype=torch.int64)), ValueError, "contiguous int32"),
    (dict(request_blocks=torch.zeros(8, 4, dtype=I32).t()), ValueError, "contiguous int32"),
    (dict(request_blocks=torch.zeros(4, 0, dtype=I32)), ValueError, "must be positive"),
    (dict(block_size=0), ValueError, "must be positive"),
    (dict(num_tokens=-1), ValueError, "non-negative"),
    (dict(num_tokens=(1 << 32) + 4), ValueError, "below 2"),
    (dict(block_size=(1 << 32) + 16), ValueError, "below 2"),
    (dict(query_lens=torch.zeros(2)), ValueError, "integer dtype"),
    (dict(rows=[0, 1]), TypeError, "Expected torch.Tensor"),
    (dict(rows=torch.zeros(4097, dtype=I32), context_lens=torch.zeros(4097, dtype=I32),
          query_lens=torch.zeros(4097, dtype=I32)), ValueError, "at most 4096"),
    (dict(), RuntimeError, "GPU-only"),
])
def test_step_tables_checks(kw, err, msg):
    with pytest.raises(err, match=msg):
        kernels.build_step_tables(**tables_args(**kw))


def rope_args(cache=True, **kw):
    bf = torch.bfloat16
    a = dict(query=torch.zeros(3, 8, 64, dtype=bf), key=torch.zeros(3, 2, 64, dtype=bf),
             positions=torch.zeros(3, dtype=I32), cos_sin=torch.zeros(10, 64), q_weight=None, k_weight=None)
    if cache:
        a.update(value=torch.zeros(3, 2, 64, dtype=bf), key_cache=torch.zeros(4, 2, 8, 16, 8, dtype=bf),
                 value_cache=torch.zeros(4, 2, 64, 16, dtype=bf), slot_mapping=torch.zeros(3, dtype=I32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(query=torch.zeros(3, 512, dtype=torch.bfloat16)), "query and key must have shapes"),
    (dict(key=torch.zeros(2, 2, 64, dtype=torch.bfloat16)), "query and key must have shapes"),
    (dict(key=torch.zeros(3, 2, 32, dtype=torch.bfloat16)), "query and key must have shapes"),
    (dict(key=torch.zeros(3, 2, 64)), "dtypes differ"),
    (dict(query=torch.zeros(3, 8, 64, dtype=torch.float64), key=torch.zeros(3, 2, 64, dtype=torch.float64)),
     "Unsupported dtype"),
    (dict(query=torch.zeros(3, 8, 60, dtype=torch.bfloat16), key=torch.zeros(3, 2, 60, dtype=torch.bfloat16)),
     "multiple of 8"),
    (dict(query=torch.zeros(3, 8, 264, dtype=torch.bfloat16), key=torch.zeros(3, 2, 264, dtype=torch.bfloat16)),
     "multiple of 8"),
    (dict(positions=torch.zeros(4, dtype=I32)), "positions must have shape"),
    (dict(positions=torch.zeros(3)), "integer dtype"),
    (dict(cos_sin=torch.zeros(10, 64, dtype=torch.bfloat16)), "cos_sin must be a float32"),
    (dict(cos_sin=torch.zeros(0, 64)), "cos_sin must be a float32"),
    (dict(cos_sin=torch.zeros(10, 66)), "rotary_dim must be even"),
    (dict(cos_sin=torch.zeros(10, 7)), "rotary_dim must be even"),
    (dict(q_weight=torch.zeros(32, dtype=torch.bfloat16)), "norm weights must have shape"),
    (dict(q_weight=torch.zeros(64, dtype=torch.float16)), "norm weights must be of"),
    (dict(q_weight=torch.zeros(64), k_weight=torch.zeros(64, dtype=torch.bfloat16)), "norm weights must be of"),
    (dict(q_weight=torch.zeros(64), eps=math.inf), "eps must be finite"),
    (dict(k_weight=torch.zeros(64), eps=-1.0), "eps must be finite"),
])
def test_norm_rope_checks(kw, msg):
    with pytest.raises(ValueError, match=msg):
        kernels.qk_norm_rope(**rope_args(False, **kw))
    with pytest.raises(ValueError, match=msg):
        kernels.qk_norm_rope_and_cache(**rope_args(True, **kw))


@pytest.mark.parametrize("kw,msg", [
    (dict(value=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), "key and value must have shape"),
    (dict(value=torch.zeros(3, 2, 64)), "dtypes differ"),
    (dict(slot_mapping=torch.zeros(2, dtype=I32)), "slot_mapping must have shape"),
    (dict(slot_mapping=torch.zeros(3)), "integer dtype"),
    (dict(value_cache=torch.zeros(4, 2, 64, 16)), "dtypes differ"),
    (dict(key_cache=torch.zeros(4, 2, 8, 16, 8, dtype=torch.float16),
          value_cache=torch.zeros(4, 2, 64, 16, dtype=torch.float16)), "Unsupported key/cache dtype pair"),
    (dict(key_cache=torch.zeros(4, 2, 16, 16, 4, dtype=torch.bfloat16)), "key_cache must have shape"),
    (dict(value_cache=torch.zeros(4, 2, 32, 16, dtype=torch.bfloat16)), "value_cache must have shape"),
    (dict(key_cache=torch.zeros(4, 2, 8, 4, 8, dtype=torch.bfloat16),
          value_cache=torch.zeros(4, 2, 64, 4, dtype=torch.bfloat16)), "block_size must be 8, 16 or 32"),
    (dict(key_cache=torch.zeros(9, 4, 64, dtype=torch.bfloat16),
          value_cache=torch.zeros(9, 4, 64, dtype=torch.bfloat16)), "token-major caches must have shape"),
    (dict(key_cache=torch.zeros(9, 64, dtype=torch.bfloat16)), "paged or token-major layout"),
    (dict(key_cache=torch.zeros(4, 2, 4, 16, 16, dtype=torch.uint8),
          value_cache=torch.zeros(4, 2, 64, 16, dtype=torch.uint8), v_scale=0.0), "finite and nonzero"),
    (dict(key_cache=torch.zeros(8, 2, 8, 16, 8, dtype=torch.bfloat16)[::2]), "must be contiguous"),
])
def test_norm_rope_cache_checks(kw, msg):
    with pytest.raises(ValueError, match=msg):
        kernels.qk_norm_rope_and_cache(**rope_args(True, **kw))


def test_norm_rope_is_gpu_only():
    with pytest.raises(RuntimeError, match="GPU-only"):
        kernels.qk_norm_rope(**rope_args(False))
    with pytest.raises(RuntimeError, match="GPU-only"):
        kernels.qk_norm_rope_and_cache(**rope_args())
    with pytest.raises(TypeError, match="Expected torch.Tensor"):
        kernels.qk_norm_rope(**rope_args(False, positions=[0, 1, 2]))


def attn_args(extend, **kw):
    f = torch.float16
    a = dict(query=torch.zeros(2, 8, 64, dtype=f), key_cache=torch.zeros(6, 2, 8, 16, 8, dtype=f),
             value_cache=torch.zeros(6, 2, 64, 16, dtype=f), block_tables=torch.zeros(2, 4, dtype=I32),
             context_lens=torch.ones(2, dtype=I32), num_kv_heads=2, scale=0.125, block_size=16, max_seq_len=64,
             window=32, num_sinks=4)
    if extend:
        a.update(query=torch.zeros(5, 8, 64, dtype=f), query_start_loc=torch.tensor([0, 2, 5], dtype=I32),
                 max_query_len=3)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(query=torch.zeros(2, 512, dtype=torch.float16)), "query must have shape"),
    (dict(block_tables=torch.zeros(3, 4, dtype=I32)), "sequence counts differ"),
    (dict(block_tables=torch.zeros(2, dtype=I32)), "block_tables must be 2D"),
    (dict(num_kv_heads=3), "num_heads must be divisible"),
    (dict(num_kv_heads=4), "cache KV-head count"),
    (dict(value_cache=torch.zeros(6, 2, 32, 16, dtype=torch.float16)), "cache head size"),
    (dict(block_size=8), "cache block dimensions"),
    (dict(max_seq_len=0), "max_seq_len must be positive"),
    (dict(max_seq_len=65), "exceeds block table capacity"),
    (dict(window=-1), "window"),
    (dict(num_sinks=-1), "non-negative"),
    (dict(query=torch.zeros(2, 8, 64)), "Unsupported query/cache dtype pair"),
    (dict(query=torch.zeros(2, 8, 64, dtype=torch.bfloat16)), "Unsupported query/cache dtype pair"),
    (dict(block_tables=torch.zeros(2, 4)), "integer dtype"),
    (dict(key_cache=torch.zeros(96, 2, 64, dtype=torch.float16),
          value_cache=torch.zeros(96, 2, 64, dtype=torch.float16), block_size=1,
          block_tables=torch.zeros(2, 64, dtype=I32)), "reads the paged 5-D layout"),
    (dict(key_cache=torch.zeros(6, 2, 4, 16, 16, dtype=torch.uint8),
          value_cache=torch.zeros(6, 2, 64, 16, dtype=torch.uint8), k_scale=0.0), "finite and nonzero"),
    (dict(key_cache=torch.zeros(6, 2, 16, 8, 8, dtype=torch.float16).transpose(2, 3)),
     "key_cache must be contiguous within each"),
])
def test_attention_checks(kw, msg):
    with pytest.raises(ValueError, match=msg):
        kernels.paged_attention_window(**attn_args(False, **kw))
    if "query" not in kw:
        with pytest.raises(ValueError, match=msg):
            kernels.paged_attention_extend(**attn_args(True, **kw))


def test_attention_checks_of_one_call():
    with pytest.raises(ValueError, match="window must be positive"):
        kernels.paged_attention_window(**attn_args(False, window=0))
    with pytest.raises(ValueError, match="sequence counts differ"):
        kernels.paged_attention_window(**attn_args(False, query=torch.zeros(3, 8, 64, dtype=torch.float16)))
    with pytest.raises(ValueError, match="query_start_loc must have shape"):
        kernels.paged_attention_extend(**attn_args(True, query_start_loc=torch.zeros(2, dtype=I32)))
    with pytest.raises(ValueError, match="max_query_len must be positive"):
        kernels.paged_attention_extend(**attn_args(True, max_query_len=0))
    with pytest.raises(TypeError, match="Expected torch.Tensor"):
        kernels.paged_attention_extend(**attn_args(True, query_start_loc=None))
    with pytest.raises(RuntimeError, match="GPU-only"):
        kernels.paged_attention_window(**attn_args(False))
    with pytest.raises(RuntimeError, match="GPU-only"):
        kernels.paged_attention_extend(**attn_args(True))


# ---- C ABI ----------------------------------------------------------------------------

BUF = np.zeros(256, dtype=np.uint8)
P = (BUF.ctypes.data + 63) // 64 * 64  # a non-null, aligned address that no rejected call reads


def test_extend_abi_refusals():
    lib = _lib.lib()
    base = dict(out=P, q=P, kc=P, vc=P, bt=P, ctx=P, start=P, N=5, B=2, Hq=8, Hkv=2, D=128, bs=16, max_blocks=4,
                max_seq=64, max_query=3, window=0, sinks=0, nb=10, scale=1.0, qs=1024, kbs=4096, khs=2048, vbs=4096,
                vhs=2048, ws=P, wsb=1 << 40, qd=_lib.PKV_BF16, cd=_lib.PKV_BF16, k_scale=1.0, v_scale=1.0, stream=None)
    for kw, code, msg in [
        (dict(N=-1), 1, "non-negative"), (dict(Hkv=3), 1, "divisible"), (dict(max_seq=0), 1, "max_seq_len"),
        (dict(max_seq=(1 << 30) + 1, max_blocks=1 << 28), 2, "at most 2^30"),
        (dict(max_query=0), 1, "max_query_len"), (dict(window=-1), 1, "window"), (dict(sinks=-1), 1, "window"),
        (dict(start=None), 1, "one token per sequence"), (dict(start=None, N=2), 1, "one token per sequence"),
        (dict(D=100), 2, "Unsupported head_size"), (dict(bs=64), 2, "Unsupported head_size"),
        (dict(max_seq=65), 1, "capacity"), (dict(qd=_lib.PKV_F32, cd=_lib.PKV_F32), 2, "dtype pair"),
        (dict(qd=_lib.PKV_F16), 2, "dtype pair"), (dict(cd=_lib.PKV_FP8_E4M3, D=120), 2, "multiple of 16"),
        (dict(cd=_lib.PKV_FP8_E4M3, v_scale=math.nan), 1, "finite and nonzero"), (dict(nb=0), 1, "num_blocks"),
        (dict(N=1 << 28), 2, "grid limit"), (dict(out=None), 1, "null buffer"), (dict(bt=None), 1, "null buffer"),
        (dict(out=P + 8), 1, "out must be"), (dict(qs=1023), 1, "query rows"), (dict(q=P + 2), 1, "query rows"),
        (dict(kbs=4097), 1, "not aligned"), (dict(vc=P + 8), 1, "not aligned"), (dict(vhs=2052), 1, "not aligned"),
        (dict(ws=None), 1, "workspace is smaller"), (dict(wsb=100), 1, "workspace is smaller"),
        (dict(ws=P + 4), 1, "16-byte aligned"),
    ]:
        st = lib.pkv_paged_attention_extend(*{**base, **kw}.values())
        assert st == code and msg in lib.pkv_last_error().decode(), (kw, st, lib.pkv_last_error())
    assert lib.pkv_paged_attention_extend(*{**base, "N": 0}.values()) == 0
    size = lib.pkv_paged_attention_extend_workspace_size
    assert size(5, 2, 8, 2, 128, 64, 3, 0, 0) >= _lib.PKV_COUNTER_BYTES
    # Split rows need their states: one sequence of 32768 tokens.
    assert size(1, 1, 28, 4, 128, 32768, 1, 0, 0) > _lib.PKV_COUNTER_BYTES + 28 * 2 * 130 * 4
    for bad in [(-1, 2, 8, 2, 128, 64, 3, 0, 0), (5, 2, 8, 3, 128, 64, 3, 0, 0), (5, 2, 8, 2, 0, 64, 3, 0, 0),
                (5, 2, 8, 2, 128, 0, 3, 0, 0), (5, 2, 8, 2, 128, 64, 0, 0, 0), (5, 2, 8, 2, 128, 64, 3, -1, 0)]:
        assert size(*bad) == 0


def test_attention_refuses_a_scale_that_is_not_finite():
    for scale in (math.nan, math.inf, -math.inf):
        for extend, call in ((False, kernels.paged_attention_window), (True, kernels.paged_attention_extend)):
            with pytest.raises(ValueError, match="scale must be finite"):
                call(**attn_args(extend, scale=scale))
    lib = _lib.lib()
    args = lambda scale, cd, k_scale: (P, P, P, P, P, P, P, 5, 2, 8, 2, 128, 16, 4, 64, 3, 0, 0, 10, scale, 1024, 4096,  # noqa: E731
                                       2048, 4096, 2048, None, 0, _lib.PKV_BF16, cd, k_scale, 1.0, None)
    for scale, cd, k_scale in ((math.nan, _lib.PKV_BF16, 1.0), (math.inf, _lib.PKV_BF16, 1.0),
                               (3e38, _lib.PKV_BF16, 1.0), (1e30, _lib.PKV_FP8_E4M3, 1e30)):
        assert lib.pkv_paged_attention_extend(*args(scale, cd, k_scale)) == 1
        assert b"scale must be finite" in lib.pkv_last_error()
    # (An FP8 scale does not count for other caches; the next check is the workspace's.)
    assert lib.pkv_paged_attention_extend(*args(1e30, _lib.PKV_BF16, 1e30)) == 1
    assert b"workspace" in lib.pkv_last_error()


def test_norm_rope_abi_refusals():
    lib = _lib.lib()
    base = dict(qo=P, q=P, k=P, v=P, pos=P, cs=P, qw=None, kw=None, kc=P, vc=P, slots=P, N=3, Hq=8, Hkv=2, D=64,
                rot=64, P=10, qs=512, ks=128, vs=128, eps=1e-6, inter=0, wd=_lib.PKV_BF16,
                layout=_lib.PKV_LAYOUT_PAGED5D, bs=16, x=8, num_slots=64, dt=_lib.PKV_BF16, cd=_lib.PKV_BF16,
                k_scale=1.0, v_scale=1.0, stream=None)
    for kw, code, msg in [
        (dict(N=-1), 1, "non-negative"), (dict(Hq=0), 1, "must be positive"), (dict(D=60), 2, "multiple of 8"),
        (dict(D=512, rot=64), 2, "multiple of 8"), (dict(rot=66), 1, "rotary_dim"), (dict(rot=3), 1, "rotary_dim"),
        (dict(rot=0), 1, "rotary_dim"), (dict(P=0), 1, "num_positions"), (dict(dt=5), 1, "Unsupported dtype"),
        (dict(cd=_lib.PKV_F16), 2, "dtype pair"), (dict(qw=P, wd=_lib.PKV_F16), 2, "weights"),
        (dict(kw=P, eps=-1.0), 1, "eps"), (dict(bs=4), 2, "block_size must be"), (dict(x=4), 1, "last dimension"),
        (dict(num_slots=65), 1, "multiple of block_size"), (dict(layout=3), 1, "layout"),
        (dict(qs=511), 1, "smaller than a row"), (dict(ks=132), 1, "16-byte aligned"), (dict(q=P + 8), 1, "aligned"),
        (dict(cs=P + 4), 1, "aligned"), (dict(v=None), 1, "null buffer"), (dict(slots=None), 1, "null buffer"),
        (dict(vs=100), 1, "value rows"), (dict(kc=P + 8), 1, "value rows"), (dict(pos=None), 1, "null buffer"),
        (dict(cd=_lib.PKV_FP8_E4M3, x=16, k_scale=math.inf), 1, "finite and nonzero"),
    ]:
        st = lib.pkv_qk_norm_rope_and_cache(*{**base, **kw}.values())
        assert st == code and msg in lib.pkv_last_error().decode(), (kw, st, lib.pkv_last_error())
    assert lib.pkv_qk_norm_rope_and_cache(*{**base, "N": 0}.values()) == 0
    plain = (P, None, P, P, P, P, None, None, 3, 8, 2, 64, 64, 10, 512, 128, 1e-6, 0, 2, 2, None)
    assert lib.pkv_qk_norm_rope(*plain) == 1 and b"k_out" in lib.pkv_last_error()
    # More lane groups than a launch holds.
    big = {**base, "N": 1 << 31}
    assert lib.pkv_qk_norm_rope_and_cache(*big.values()) == 2 and b"grid limit" in lib.pkv_last_error()


def test_step_tables_abi_refusals():
    lib = _lib.lib()
    base = dict(rb=P, rows=P, ctx=P, ql=P, nbk=P, bt=P, slots=P, pos=P, start=P, R=4, B=2, W=8, nn=2, N=4, bs=16,
                stream=None)
    for kw, code, msg in [(dict(B=-1), 1, "non-negative"), (dict(N=-1), 1, "non-negative"), (dict(W=0), 1, "positive"),
                          (dict(bs=0), 1, "positive"), (dict(B=4097), 2, "at most 4096"), (dict(start=None), 1, "null"),
                          (dict(slots=None), 1, "null"), (dict(rows=None), 1, "null"), (dict(nbk=None), 1, "null"),
                          (dict(rb=None), 1, "null")]:
        st = lib.pkv_build_step_tables(*{**base, **kw}.values())
        assert st == code and msg in lib.pkv_last_error().decode(), (kw, st)


# ---- rotary tables --------------------------------------------------------------------


def test_rotary_table_values():
    t = rotary_table(2000, 8, base=100.0)
    assert t.dtype == torch.float32 and t.shape == (2000, 8)
    for p in (0, 1, 1999):
        for i in range(4):
            a = p * 100.0 ** (-2 * i / 8)
            # Half a float32 step of the value, and as much of the angle's own 64-bit rounding.
            assert abs(t[p, i].item() - math.cos(a)) <= 2.0 ** -24 and abs(t[p, 4 + i].item() - math.sin(a)) <= 2.0 ** -24


def test_rotary_far_positions_keep_their_angle():
    t = rotary_table(1 << 20, 2, base=10000.0)
    a = float((1 << 20) - 1)
    assert abs(t[-1, 0].item() - math.cos(a)) <= 2.0 ** -24


def test_rotary_scalings():
    plain, one = rotary_frequencies(64, 10000.0)
    assert one == 1.0
    linear, _ = rotary_frequencies(64, 10000.0, {"type": "linear", "factor": 4.0})
    assert torch.allclose(linear * 4, plain, rtol=1e-15, atol=0)
    ntk, _ = rotary_frequencies(64, 10000.0, {"type": "ntk", "factor": 8.0})
    assert ntk[0] == plain[0] and abs(ntk[-1] / plain[-1] * 8 - 1) < 1e-12
    rule = {"type": "yarn", "factor": 16.0, "original_max_position": 4096}
    yarn, f = rotary_frequencies(128, 10000.0, rule)
    plain, _ = rotary_frequencies(128, 10000.0)
    assert abs(f - (0.1 * math.log(16.0) + 1)) < 1e-15
    turns = 4096 * plain / (2 * math.pi)
    # The fast pairs are untouched, the slow ones slowed 16 times, the ratio falls in between.
    ratio = yarn / plain
    assert (ratio[turns > 40] == 1).all() and torch.allclose(ratio[turns < 0.8] * 16, torch.ones(1).double())
    assert (ratio[1:] <= ratio[:-1] + 1e-15).all()
    assert rotary_frequencies(128, 10000.0, {**rule, "attention_factor": 1.0})[1] == 1.0
    rule = {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
            "original_max_position": 8192}
    bands, f = rotary_frequencies(128, 500000.0, rule)
    plain, _ = rotary_frequencies(128, 500000.0)
    turns = 8192 * plain / (2 * math.pi)
    assert f == 1.0 and (bands[turns >= 4] == plain[turns >= 4]).all()
    assert torch.allclose(bands[turns <= 1] * 8, plain[turns <= 1], rtol=1e-15, atol=0)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and ((bands[mid] < plain[mid]) & (bands[mid] > plain[mid] / 8)).all()


@pytest.mark.parametrize("args,msg", [
    ((0, 8), "max_positions"), ((4, 7), "rotary_dim"), ((4, 0), "rotary_dim"), ((4, 8, 0.0), "base"),
    ((4, 8, 1e4, {"type": "other"}), "Unknown rotary scaling"), ((4, 8, 1e4, {"type": "linear"}), "needs 'factor'"),
    ((4, 8, 1e4, {"type": "linear", "factor": -1}), "must be positive"),
    ((4, 2, 1e4, {"type": "ntk", "factor": 2}), "above 2"),
    ((4, 8, 1.0, {"type": "yarn", "factor": 2, "original_max_position": 8}), "above 1"),
    ((4, 8, 1e4, {"type": "llama3", "factor": 2, "low_freq_factor": 4, "high_freq_factor": 1,
                  "original_max_position": 8}), "must exceed"),
])
def test_rotary_refusals(args, msg):
    with pytest.raises(ValueError, match=msg):
        rotary_table(*args)


def test_rotary_scaling_without_a_type_is_refused():
    # (A rule under another name for its type must not become an unscaled table.)
    for rule in ({}, {"factor": 8.0}, {"type": None, "factor": 8.0}, {"rope_type": "linear", "factor": 8.0}):
        with pytest.raises(ValueError, match="Unknown rotary scaling None"):
            rotary_table(4, 8, 1e4, rule)


# ---- the host side of RequestBlocks ---------------------------------------------------


def test_request_blocks_host_state():
    alloc = BlockAllocator(10)
    shared = alloc.alloc(2)
    rb = RequestBlocks(2, 4, 16, alloc, "cpu")
    a = rb.open(shared)
    b = rb.open()
    assert rb.num_tokens(a) == 32 and rb.blocks(a) == shared and alloc.refcount(shared[0]) == 2
    assert rb.table[a].tolist() == shared + [-1, -1]
    with pytest.raises(MemoryError, match="every row"):
        rb.open()
    for rows, new, kw, msg in [([a], [1, 2], {}, "same length"), ([a, a], [1, 1], {}, "once"), ([7], [1], {}, "not open"),
                               ([a], [-1], {}, "non-negative"), ([a], [33], {}, "max_blocks"),
                               ([a, b], [1, 1], {"num_seqs": 1}, "must hold"), ([a], [5], {"num_tokens": 4}, "must hold")]:
        with pytest.raises(ValueError, match=msg):
            rb.step(rows, new, **kw)
    # A step that cannot run leaves blocks, lengths and the allocator as they were.
    free = alloc.available_size
    with pytest.raises(RuntimeError, match="GPU-only"):
        rb.step([a, b], [3, 20])
    assert alloc.available_size == free and rb.num_tokens(b) == 0 and rb.blocks(a) == shared
    taken = alloc.alloc(free)
    with pytest.raises(MemoryError):
        rb.step([b], [1])
    alloc.free(taken)
    rb.close(a)
    assert alloc.refcount(shared[0]) == 1
    with pytest.raises(ValueError, match="not open"):
        rb.close(a)
    with pytest.raises(ValueError, match="prefix blocks exceed"):
        rb.open([1] * 5)
    assert rb.open() == a
