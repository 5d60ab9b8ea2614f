"""The operators together, as a server runs a layer: requests open (one on a
cached prefix), a prefill in two chunks, then decode steps with a window; tables
from RequestBlocks, keys and values through qk_norm_rope_and_cache, attention by
paged_attention_extend and paged_attention_window.  Every step's output is
compared with attention in 64 bits over the sequence's whole history of rotated
keys and values, kept apart from the cache."""

import numpy as np
import pytest
import torch

from sglang_mlx_amd import kernels
from sglang_mlx_amd.rotary import rotary_table
from sglang_mlx_amd.srt.mem_cache import BlockAllocator, RequestBlocks

pytestmark = pytest.mark.gpu

Hq, H, D, BS, NB = 8, 2, 64, 16, 80


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_prefill_and_decode(dtype, window, sinks):
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    cos_sin = rotary_table(512, D, scaling={"type": "linear", "factor": 2.0}, device="cuda")
    qw, kw = (torch.empty(D, device="cuda").uniform_(0.5, 1.5, generator=g).to(dtype) for _ in range(2))
    kc = torch.full((NB, H, D // 8, BS, 8), float("nan"), dtype=dtype, device="cuda")
    vc = torch.full((NB, H, D, BS), float("nan"), dtype=dtype, device="cuda")
    alloc = BlockAllocator(NB)
    rb = RequestBlocks(6, 12, BS, alloc, "cuda")
    history = {}  # row -> (keys [t, H, D], values)
    u = torch.finfo(dtype).eps / 2

    def step(rows, new, pad_seqs=0, pad_tokens=0):
        n = sum(new)
        st = rb.step(rows, new, len(rows) + pad_seqs, n + pad_tokens)
        qkv = torch.empty((n + pad_tokens, (Hq + 2 * H) * D), device="cuda").normal_(generator=g).to(dtype)
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, H * D, H * D], 1))
        q2, k2 = kernels.qk_norm_rope(q, k, st.positions, cos_sin, qw, kw)
        q1, _, _ = kernels.qk_norm_rope_and_cache(q, k, v, st.positions, cos_sin, kc, vc, st.slot_mapping, qw, kw)
        assert torch.equal(q1, q2)
        args = (q1, kc, vc, st.block_tables, st.context_lens)
        if st.max_query_len == 1 and window and pad_tokens == 0:
            out = kernels.paged_attention_window(*args, H, D ** -0.5, BS, st.max_seq_len, window, sinks)
        else:
            out = kernels.paged_attention_extend(*args, st.query_start_loc, H, D ** -0.5, BS, st.max_seq_len,
                                                 st.max_query_len, window, sinks)
        at = 0
        for r, m in zip(rows, new):
            hk, hv = history.get(r, (k2[:0], v[:0]))
            hk, hv = torch.cat([hk, k2[at:at + m]]), torch.cat([hv, v[at:at + m]])
            history[r] = hk, hv
            T = hk.shape[0]
            assert T == rb.num_tokens(r)
            t, pos = torch.arange(T, device="cuda"), torch.arange(T - m, T, device="cuda")[:, None]
            sees = t <= pos
            if window:
                sees &= (t > pos - window) | (t < sinks)
            for h in range(Hq):
                kh, vh = hk[:, h // 4].double(), hv[:, h // 4].double()
                s = (q2[at:at + m, h].double() @ kh.t().contiguous() * D ** -0.5).masked_fill(~sees, float("-inf"))
                p = torch.softmax(s, -1)
                # Weights and output are rounded to the type (half a step each), keys that rounded to another
                # neighbour in the two kernels' float32 would show as more; float32's own part is far below.
                bound = 1.1 * u * (p @ vh.abs() + (p @ vh).abs()) + 1e-5
                assert ((out[at:at + m, h].double() - p @ vh).abs() <= bound).all()
            at += m
        assert (out[at:] == 0).all()
        return out

    a, b = rb.open(), rb.open()
    step([a, b], [70, 16])                       # ragged prefill
    step([b, a], [33, 5], pad_seqs=2, pad_tokens=3)  # chunks behind cached tokens, a padded batch
    c = rb.open(rb.blocks(a)[:3])                # 48 tokens of request a as a shared prefix
    history[c] = tuple(x[:48] for x in history[a])
    step([c, b], [9, 1])
    for _ in range(3):
        step([a, b, c], [1, 1, 1])
    rb.close(b)
    d = rb.open()
    history.pop(b)
    step([d, a, c], [40, 1, 4])                  # a prefill beside single and drafted tokens
    for _ in range(2):
        step([c, d, a], [1, 1, 1], pad_seqs=1, pad_tokens=1)
    for r in (a, c, d):
        rb.close(r)
    assert alloc.available_size == NB - 1
