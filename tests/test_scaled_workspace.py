"""The workspace of attention over caches with a scale per block and head: states for the
pieces that a call can leave, on the CPU by the C ABI's sizes, on the GPU by what it writes."""

import numpy as np
import pytest
import torch

import pkv_scaled as ps
from sglang_mlx_amd import _lib

DEV = "cuda"


def size(B, Hq, H, D, max_seq, max_query, window=0, sinks=0):
    return _lib.lib().pkv_paged_attention_scaled_workspace_size(B, Hq, H, D, max_seq, max_query, window, sinks)


@pytest.mark.parametrize("Hq,H,D", [(32, 8, 128), (64, 8, 256), (28, 4, 128), (8, 1, 64), (16, 16, 32)])
def test_size_stays_bounded(Hq, H, D):
    """Sequences are cut where two crews or more share at most 512 workgroups, each with two states of 16 rows."""
    most = _lib.PKV_COUNTER_BYTES + 512 * 2 * 16 * (D + 2) * 4
    for max_query in (1, 4, 5, 16, 33, 64, 512, 513, 1000, 8192, 1 << 20):
        for B, max_seq in ((1, 500), (4, 1 << 20), (64, 4096), (600, 100)):
            units = H * -(-max_query * (Hq // H) // 16)
            need = size(B, Hq, H, D, max_seq, max_query)
            assert _lib.PKV_COUNTER_BYTES <= need <= most, (B, max_seq, max_query, need)
            if units > 256:  # a single crew: nothing is cut
                assert need == _lib.PKV_COUNTER_BYTES


@pytest.mark.gpu
def test_a_single_crew_writes_no_states():
    """70 rows of 64 heads over 8 are 280 units: one crew, whole sequences; what lies behind the counters stays."""
    Hq, H, D, bs, B = 64, 8, 64, 16, 3
    new, ctx = [70, 1, 30], [300, 1000, 45]
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    need_blocks = [-(-c // bs) for c in ctx]
    nb = sum(need_blocks)
    table = torch.full((B, max(need_blocks)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need_blocks):
        table[i, :n] = torch.arange(at, at + n)
        at += n
    table = table.to(DEV)
    kc, vc = (torch.randn(s, generator=g, device=DEV).mul_(60).clamp_(-240, 240).to(torch.float8_e4m3fn).view(torch.uint8)
              for s in ((nb, H, D // 16, bs, 16), (nb, H, D, bs)))
    scales = torch.full((nb, H, 2), 2.0 ** -7, device=DEV)
    q = torch.randn((sum(new), Hq, D), generator=g, device=DEV).bfloat16()
    lens = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    loc = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=DEV)
    max_seq = table.shape[1] * bs
    need = size(B, Hq, H, D, max_seq, max(new))
    assert need == _lib.PKV_COUNTER_BYTES
    room = torch.zeros(need + (1 << 20), dtype=torch.uint8, device=DEV)
    room[need:] = 0x55
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    _lib.check(_lib.lib().pkv_paged_attention_scaled(
        out.data_ptr(), q.data_ptr(), kc.data_ptr(), vc.data_ptr(), scales.data_ptr(), table.data_ptr(),
        lens.data_ptr(), loc.data_ptr(), sum(new), B, Hq, H, D, bs, table.shape[1], max_seq, max(new), 0, 0, nb,
        D ** -0.5, q.stride(0), kc.stride(0), kc.stride(1), vc.stride(0), vc.stride(1), room.data_ptr(), need,
        _lib.PKV_BF16, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert (room[:need] == 0).all() and (room[need:] == 0x55).all()
    a = 0
    for i, (c, n) in enumerate(zip(ctx, new)):
        k, v = ps.rows_of(kc, vc, scales, table[i], 0, c)
        want, off = ps.attend(q[a:a + n], k, v, c - n, D ** -0.5)
        assert ((out[a:a + n].double() - want).abs() <= off).all()
        a += n
