"""The native call path of the step-table, rotation and new-token attention entry
points against the Python path: plain calls are taken and give the same bytes,
other forms are handed back and give the Python path's result, refusals keep
their messages."""

import pytest
import torch

from sglang_mlx_amd import _ext, kernels
from sglang_mlx_amd.rotary import rotary_table

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
I32, BF = torch.int32, torch.bfloat16


def ints(*a):
    return torch.tensor(a, dtype=I32, device=DEV)


def table_args():
    return [torch.arange(40, dtype=I32, device=DEV).view(5, 8), ints(3, 0, -1), ints(40, 17, 0), ints(9, 17, 0),
            ints(90, 91, 92, 93), 16, 30]


def rope_args(cache=True, dtype=BF, cdtype=BF, layout="paged"):
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    qkv = torch.randn(21, 12 * 64, device=DEV, generator=g).to(dtype)
    q, k, v = (t.view(21, -1, 64) for t in qkv.split([512, 128, 128], 1))
    a = dict(query=q, key=k, positions=torch.arange(21, dtype=I32, device=DEV), cos_sin=rotary_table(30, 64, device=DEV),
             q_weight=torch.rand(64, device=DEV, generator=g).to(dtype), k_weight=torch.rand(64, device=DEV, generator=g)
             .to(dtype), eps=1e-5, interleaved=False)
    if cache:
        x = 16 // torch.empty((), dtype=cdtype).element_size()
        shapes = [(4, 2, 64 // x, 16, x), (4, 2, 64, 16)] if layout == "paged" else [(64, 2, 64)] * 2
        a.update(value=v, key_cache=torch.zeros(shapes[0], dtype=cdtype, device=DEV),
                 value_cache=torch.zeros(shapes[1], dtype=cdtype, device=DEV),
                 slot_mapping=torch.arange(5, 26, dtype=I32, device=DEV), k_scale=1.0, v_scale=1.0)
    return a


def attn_args(extend, dtype=BF):
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    kc, vc = (torch.randn(s, device=DEV, generator=g).to(dtype) for s in ((12, 2, 8, 16, 8), (12, 2, 64, 16)))
    a = dict(query=torch.randn(7 if extend else 2, 8, 64, device=DEV, generator=g).to(dtype), key_cache=kc,
             value_cache=vc, block_tables=torch.arange(12, dtype=I32, device=DEV).view(2, 6), seq_lens=ints(70, 96))
    if extend:
        a.update(query_start_loc=ints(0, 5, 7))
    a.update(num_kv_heads=2, scale=0.125, block_size=16, max_seq_len=96)
    if extend:
        a.update(max_query_len=5)
    a.update(window=30, num_sinks=2, k_scale=1.0, v_scale=1.0)
    return a


def same(a, b):
    for x, y in zip(a if isinstance(a, (list, tuple)) else [a], b if isinstance(b, (list, tuple)) else [b]):
        assert x.dtype == y.dtype and torch.equal(x, y)


def both(monkeypatch, fn, make, taken):
    """Runs fn natively and by the Python path on equal inputs; taken: whether the native path is to answer."""
    calls = []
    real = _ext._done

    def done(result):
        calls.append(result is not None and type(result) is not int)
        return real(result)

    monkeypatch.setattr(_ext, "_done", done)
    fn(make())  # (the first decode of a stream allocates its scratch on the Python path)
    calls.clear()
    got = fn(make())
    assert calls == [taken], calls
    monkeypatch.setattr(_ext, "_native", None)
    same(got, fn(make()))


@pytest.mark.parametrize("make,fn", [
    (table_args, lambda a: (*kernels.build_step_tables(*a), a[0])),
    (lambda: rope_args(False), lambda a: kernels.qk_norm_rope(**a)),
    (lambda: {**rope_args(False), "q_weight": None, "interleaved": True}, lambda a: kernels.qk_norm_rope(**a)),
    (rope_args, lambda a: kernels.qk_norm_rope_and_cache(**a)),
    (lambda: rope_args(layout="rows"), lambda a: kernels.qk_norm_rope_and_cache(**a)),
    (lambda: rope_args(dtype=torch.float32, cdtype=torch.uint8), lambda a: kernels.qk_norm_rope_and_cache(**a)),
    (lambda: attn_args(False), lambda a: _ext.paged_attention_window(**a)),
    (lambda: attn_args(True), lambda a: _ext.paged_attention_extend(**a)),
    (lambda: attn_args(True, torch.float16), lambda a: _ext.paged_attention_extend(**a)),
])
def test_plain_calls_are_taken_and_equal(monkeypatch, make, fn):
    both(monkeypatch, fn, make, True)


@pytest.mark.parametrize("make,fn", [
    (lambda: [t.long() if i in (1, 2, 3, 4) else t for i, t in enumerate(table_args())],
     lambda a: (*kernels.build_step_tables(*a), a[0])),
    (lambda: {**rope_args(), "positions": torch.arange(21, device=DEV)}, lambda a: kernels.qk_norm_rope_and_cache(**a)),
    (lambda: {**rope_args(), "eps": 0}, lambda a: kernels.qk_norm_rope_and_cache(**a)),
    (lambda: {**rope_args(False), "query": rope_args(False)["query"].transpose(0, 1).contiguous().transpose(0, 1)},
     lambda a: kernels.qk_norm_rope(**a)),
    (lambda: {**attn_args(True), "seq_lens": attn_args(True)["seq_lens"].long()},
     lambda a: _ext.paged_attention_extend(**a)),
    (lambda: {**attn_args(False), "scale": 1}, lambda a: _ext.paged_attention_window(**a)),
])
def test_other_forms_go_to_the_python_path(monkeypatch, make, fn):
    both(monkeypatch, fn, make, False)


def test_refusals_keep_their_messages():
    a = table_args()
    with pytest.raises(ValueError, match="must be positive"):
        kernels.build_step_tables(*a[:5], 0, 4)
    with pytest.raises(ValueError, match="rotary_dim must be even"):
        kernels.qk_norm_rope(**{**rope_args(False), "cos_sin": rotary_table(4, 66, device=DEV)})
    with pytest.raises(ValueError, match="slot_mapping must have shape"):
        kernels.qk_norm_rope_and_cache(**{**rope_args(), "slot_mapping": ints(1, 2)})
    with pytest.raises(RuntimeError, match="GPU-only"):
        kernels.qk_norm_rope_and_cache(**{**rope_args(), "slot_mapping": torch.zeros(21, dtype=I32)})
    with pytest.raises(ValueError, match="exceeds block table capacity"):
        _ext.paged_attention_extend(**{**attn_args(True), "max_seq_len": 97})
    with pytest.raises(ValueError, match="window must be positive"):
        _ext.paged_attention_window(**{**attn_args(False), "window": 0})
    with pytest.raises(ValueError, match="Unsupported head_size"):
        b = attn_args(False)
        _ext.paged_attention_window(**{**b, "query": b["query"][..., :40].contiguous(),
                                       "key_cache": b["key_cache"][:, :, :5].contiguous(),
                                       "value_cache": b["value_cache"][:, :, :40].contiguous()})
