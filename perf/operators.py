"""Performance cases of the operators around the paged KV cache.

Kinds, each one call of a serving program on tensors that it already holds:

  tables   block tables, slots and positions of a step, from request lengths
  rope     per-head norm of queries and keys, position rotation, and the append
           of the rotated keys and the values to the cache (or, with cache
           "none", the rotated queries and keys alone)
  window   decode attention over a sliding window and a few first tokens
  extend   causal attention of several new tokens per sequence (a prefill, a
           chunk of one, a verification of drafted tokens), whole or windowed

With `own` false a pass is the operator written in elementary tensor operations,
in 32 bits, rounded once at the end; with `own` true it is the package's call.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.uint8}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1}
# Scales of FP8 caches: codes hold K / k_scale and V / v_scale.
K_SCALE, V_SCALE = 0.05, 0.02
# Queries are this much wider than unit normal, so that a softmax row has the
# peaks that attention over a real context has.
Q_GAIN = 2.0
EPS = 1e-6

# The most that a drawn case costs: bytes of a decode, floating-point
# operations of an extend, tokens of a rope or tables call.
DRAW_BYTES = 5.0e8
DRAW_FLOPS = 1.0e12
DRAW_TOKENS = 8192
# Score elements of one step of the plain extend (its memory, not its result).
PLAIN_SCORES = 1 << 28


def listed():
    return [
        # A loaded server's decode step: 64 requests, one new token each.
        dict(name="tables_decode_b64", kind="tables", batch=64, lo=512, hi=4096, new_lo=1, new_hi=1, block_size=16,
             pad=0, requests=256),
        # A chunked prefill of 16K tokens packed from 211 requests of very
        # different lengths, padded to fixed sizes.
        dict(name="tables_prefill_16k", kind="tables", batch=211, lo=40, hi=8000, new_lo=1, new_hi=153,
             block_size=16, pad=45, requests=512),
        # One user's decode step (32 query heads, 8 KV heads of 128): latency.
        dict(name="rope_b1", kind="rope", q="bf16", cache="bf16", layout="paged", tokens=1, heads=32, kv_heads=8,
             head_size=128, rot=128, block_size=16, lo=1, hi=1, pattern="scatter", norm=True, interleaved=False),
        # A loaded server's decode step into the token pool: half of each head
        # rotates, neighbouring elements in pairs.
        dict(name="rope_pool_b200", kind="rope", q="f16", cache="f16", layout="token", tokens=200, heads=32,
             kv_heads=8, head_size=128, rot=64, block_size=1, lo=1, hi=1, pattern="scatter", norm=False,
             interleaved=True),
        # Prefill of ragged prompts, 8K tokens, into paged caches.
        dict(name="rope_prefill_8k", kind="rope", q="bf16", cache="bf16", layout="paged", tokens=8192, heads=32,
             kv_heads=8, head_size=128, rot=128, block_size=16, lo=97, hi=927, pattern="prompts", norm=True,
             interleaved=False),
        # Queries and keys alone, float32 activations, an odd number of tokens
        # of 28 and 4 heads.
        dict(name="rope_f32_1999", kind="rope", q="f32", cache="none", layout="none", tokens=1999, heads=28,
             kv_heads=4, head_size=128, rot=128, block_size=1, lo=1, hi=1, pattern="scatter", norm=True,
             interleaved=False),
        # One user with a long context, of which 4096 tokens and 4 first ones
        # are read.
        dict(name="window_b1_32k", kind="window", q="bf16", cache="bf16", batch=1, heads=32, kv_heads=8,
             head_size=128, block_size=16, lo=32000, hi=32000, window=4096, sinks=4),
        # A loaded server over FP8 caches, a window of 1024.
        dict(name="window_fp8_b64", kind="window", q="bf16", cache="fp8", batch=64, heads=32, kv_heads=8,
             head_size=128, block_size=16, lo=700, hi=9001, window=1024, sinks=16),
        # A large batch of long chats, most of them past the window.
        dict(name="window_f16_b128", kind="window", q="f16", cache="f16", batch=128, heads=28, kv_heads=4,
             head_size=128, block_size=32, lo=333, hi=6007, window=4000, sinks=1),
        # Verification of 5 drafted tokens in each of 16 requests.
        dict(name="extend_draft_b16", kind="extend", q="bf16", cache="bf16", batch=16, heads=32, kv_heads=8,
             head_size=128, block_size=16, lo=300, hi=4000, new_lo=5, new_hi=5, window=0, sinks=0),
        # Ragged prompts of a small model (head size 64), behind cached
        # prefixes, with a window, over FP8 caches.
        dict(name="extend_fp8_window", kind="extend", q="bf16", cache="fp8", batch=13, heads=32, kv_heads=8,
             head_size=64, block_size=32, lo=200, hi=5000, new_lo=1, new_hi=1700, window=1024, sinks=4),
        # One long prompt, the second half of it: 8K tokens behind 8K.
        dict(name="extend_8k_of_16k", kind="extend", q="bf16", cache="bf16", batch=1, heads=32, kv_heads=8,
             head_size=128, block_size=16, lo=16384, hi=16384, new_lo=8192, new_hi=8192, window=0, sinks=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables"] * 2 + ["rope"] * 3 + ["window"] * 3 + ["extend"] * 4)
    if kind == "tables":
        batch = _log_int(rng, 1, 512)
        new_lo = rng.choice([1, 1, _log_int(rng, 1, 100)])
        new_hi = max(new_lo, min(2 * DRAW_TOKENS // batch, rng.choice([1, 1, _log_int(rng, 1, 1000)])))
        if batch * (new_lo + new_hi) > 4 * DRAW_TOKENS:
            new_lo = new_hi = 1
        lo = max(new_hi, _log_int(rng, 1, 4000))
        return dict(kind=kind, batch=batch, lo=lo, hi=min(8192, lo + _log_int(rng, 1, 4000)), new_lo=new_lo,
                    new_hi=new_hi, block_size=rng.choice([1, 8, 16, 16, 32]), pad=rng.choice([0, 0, 3, 40]),
                    requests=batch + rng.choice([0, 64, 300]))
    heads = rng.choice([(32, 8), (32, 8), (28, 4), (14, 2), (8, 1), (16, 16), (64, 8)])
    if kind == "rope":
        head_size = rng.choice([64, 80, 128, 128, 128, 256])
        q, cache = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
        layout = rng.choice(["paged", "paged", "token", "none"])
        row = (heads[0] + 2 * heads[1]) * head_size * BYTES[q]
        tokens = min(_log_int(rng, 1, DRAW_TOKENS), DRAW_TOKENS * 6144 * 2 // row)
        lo = _log_int(rng, 1, min(tokens, 2048))
        return dict(kind=kind, q=q, cache="none" if layout == "none" else cache, layout=layout, tokens=tokens,
                    heads=heads[0], kv_heads=heads[1], head_size=head_size,
                    rot=rng.choice([head_size, head_size, head_size // 2, 32]),
                    block_size=rng.choice([8, 16, 16, 32]) if layout == "paged" else 1, lo=lo, hi=min(4 * lo, 8192),
                    pattern=rng.choice(["prompts", "scatter"]) if layout == "paged" else "scatter",
                    norm=rng.random() < 0.6, interleaved=rng.random() < 0.35)
    q, cache = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "fp8"), ("f16", "fp8")])
    head_size = rng.choice([64, 80, 128, 128, 128, 256])
    case = dict(kind=kind, q=q, cache=cache, heads=heads[0], kv_heads=heads[1], head_size=head_size,
                block_size=rng.choice([8, 16, 16, 32]))
    if kind == "window":
        window = _log_int(rng, 16, 8192)
        mean = _log_int(rng, 32, 30000)
        per_seq = 2 * heads[1] * head_size * BYTES[cache] * min(2 * mean, window + 32)
        batch = min(_log_int(rng, 1, 256), max(1, int(DRAW_BYTES / per_seq)))
        # (The cache holds whole contexts, the call reads their windows.)
        batch = min(batch, max(1, int(8e9 / (2 * heads[1] * head_size * BYTES[cache] * mean))))
        lo = max(1, int(mean * rng.uniform(0.05, 1.0)))
        case.update(batch=batch, lo=lo, hi=max(lo, 2 * mean - lo), window=window,
                    sinks=rng.choice([0, 1, 4, 4, 16, 33]))
        return case
    new_hi = _log_int(rng, 1, 8192)
    new_lo = max(1, int(new_hi * rng.uniform(0.0, 1.0)))
    lo = new_hi + rng.choice([0, 0, _log_int(rng, 1, 8192)])
    hi = lo + rng.choice([0, _log_int(rng, 1, 4000)])
    per_seq = 4.0 * heads[0] * head_size * (new_lo + new_hi) / 2 * hi
    if per_seq > DRAW_FLOPS:
        new_hi = max(1, int(new_hi * DRAW_FLOPS / per_seq))
        new_lo = min(new_lo, new_hi)
        per_seq = 4.0 * heads[0] * head_size * (new_lo + new_hi) / 2 * hi
    batch = min(_log_int(rng, 1, 64), max(1, int(DRAW_FLOPS / per_seq)))
    batch = min(batch, max(1, int(DRAW_BYTES / (2 * heads[1] * head_size * BYTES[cache] * hi))))
    window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
    case.update(batch=batch, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi, window=window,
                sinks=rng.choice([0, 4, 33]) if window else 0)
    return case


# ---- inputs ---------------------------------------------------------------------


def _lengths(lo, hi, n):
    """n lengths spread evenly over [lo, hi]."""
    return np.array([lo + int((hi - lo) * (i + 0.5) / n + 0.5) for i in range(n)], dtype=np.int64)


def _batch_lengths(case, rng=None):
    """Contexts and new tokens of a batch, paired by a fixed rule; the seed
    draws the order of the sequences."""
    B = case["batch"]
    ctx = _lengths(case["lo"], case["hi"], B)
    new = np.ones(B, dtype=np.int64)
    if "new_lo" in case:
        new = np.minimum(_lengths(case["new_lo"], case["new_hi"], B)[np.arange(B) * 7919 % B], ctx)
    order = np.arange(B) if rng is None else rng.permutation(B)
    return ctx[order], new[order]


def _prompts(case):
    """Lengths of the prompts that a prefill of case["tokens"] tokens packs."""
    out, left, i = [], case["tokens"], 0
    while left > 0:
        n = min(left, case["lo"] + (case["hi"] - case["lo"]) * (i % 5) // 4)
        out.append(n)
        left -= n
        i += 1
    return out


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _values(shape, dtype, gen):
    """Cache contents: unit normal, as codes of x / scale for FP8 (below
    exponent 15, where the format's finite values end)."""
    if dtype == "fp8":
        x = torch.empty(shape, dtype=torch.float16, device=DEV).normal_(generator=gen)
        return x.mul_(20.0).clamp_(-240.0, 240.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.empty(shape, dtype=TORCH[dtype], device=DEV).normal_(generator=gen)


def _paged_caches(nb, case, gen):
    H, D, bs = case["kv_heads"], case["head_size"], case["block_size"]
    x = 16 // BYTES[case["cache"]]
    return _values((nb, H, D // x, bs, x), case["cache"], gen), _values((nb, H, D, bs), case["cache"], gen)


def _rotation(positions, rot, base=500000.0):
    """[positions, rot] float32: rot / 2 cosines, then rot / 2 sines."""
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "tables":
        return _prepare_tables(case, s, rng)
    if case["kind"] == "rope":
        return _prepare_rope(case, s, rng, gen)
    B, D, bs = case["batch"], case["head_size"], case["block_size"]
    ctx, new = _batch_lengths(case, rng)
    need = -(-ctx // bs)
    used = int(need.sum())
    nb = used + used // 10 + 2
    ids = rng.permutation(nb - 1)[:used] + 1
    table = np.full((B, int(need.max())), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    s["table"], s["ctx"] = _ints(table), _ints(ctx)
    s["max_seq_len"], s["max_query_len"] = int(ctx.max()), int(new.max())
    s["start"] = _ints(np.concatenate([[0], np.cumsum(new)]))
    # The plain form's loop over sequences knows the lengths on the host.
    s["host"] = [(int(c), int(n)) for c, n in zip(ctx, new)]
    s["scale"] = 1.0 / math.sqrt(D)
    s["scales"] = {"k_scale": K_SCALE, "v_scale": V_SCALE} if case["cache"] == "fp8" else {}
    s["k"], s["v"] = _paged_caches(nb, case, gen)
    shape = (int(new.sum()), case["heads"], D)
    s["query"] = (torch.empty(shape, dtype=torch.float32, device=DEV).normal_(generator=gen)
                  * Q_GAIN).to(TORCH[case["q"]])
    if case["cache"] == "fp8":
        s["codes"] = _code_values().float()
    return s


def _prepare_tables(case, s, rng):
    B, bs, R = case["batch"], case["block_size"], case["requests"]
    ctx, new = _batch_lengths(case, rng)
    width = -(-case["hi"] // bs) + 1
    have, need = -(-(ctx - new) // bs), -(-ctx // bs)
    total = int(need.sum())
    ids = rng.permutation(total + total // 10) + 1
    rows = rng.permutation(R)[:B]
    pool = np.full((R, width), -1, dtype=np.int32)
    at = 0
    for r, n in zip(rows, have):
        pool[r, :n] = ids[at:at + n]
        at += n
    count = int((need - have).sum())
    s["new_blocks"] = _ints(ids[at:at + count + 1])
    s["pool"] = _ints(pool)
    # A padded batch ends in sequences of no request and no tokens.
    pad = case["pad"]
    s["rows"] = _ints(np.concatenate([rows, np.full(pad, -1)]))
    s["ctx"] = _ints(np.concatenate([ctx, np.zeros(pad)]))
    s["new"] = _ints(np.concatenate([new, np.zeros(pad)]))
    s["tokens"] = int(new.sum()) + 7 * pad
    return s


def _prepare_rope(case, s, rng, gen):
    N, Hq, H, D, bs = case["tokens"], case["heads"], case["kv_heads"], case["head_size"], case["block_size"]
    dt = TORCH[case["q"]]
    # Queries, keys and values are views of one projection's output.
    qkv = torch.empty((N, (Hq + 2 * H) * D), dtype=dt, device=DEV).normal_(generator=gen)
    s["query"] = qkv[:, :Hq * D].view(N, Hq, D)
    s["key"] = qkv[:, Hq * D:(Hq + H) * D].view(N, H, D)
    s["value"] = qkv[:, (Hq + H) * D:].view(N, H, D)
    s["weights"] = {}
    if case["norm"]:
        for name in ("q_weight", "k_weight"):
            s["weights"][name] = torch.empty(D, dtype=dt, device=DEV).uniform_(0.5, 1.5, generator=gen)
    s["cos_sin"] = _rotation(8192, case["rot"])
    if case["pattern"] == "prompts":
        # Each prompt starts at position 0 and fills fresh blocks from offset 0.
        lens = _prompts(case)
        pos = np.concatenate([np.arange(n) % 8192 for n in lens])
        need = [-(-n // bs) for n in lens]
        nb = sum(need) + sum(need) // 10 + 2
        ids = rng.permutation(nb - 1)[:sum(need)].astype(np.int64) + 1
        slots, at = [], 0
        for n, b in zip(lens, need):
            t = np.arange(n)
            slots.append(ids[at + t // bs] * bs + t % bs)
            at += b
        slots = np.concatenate(slots)
        num_slots = nb * bs
    else:
        # One new token of each of many sequences.
        pos = rng.integers(0, 8192, N)
        nb = 4 * N // bs + 2
        num_slots = nb * bs
        slots = rng.permutation(num_slots - bs)[:N] + bs
    s["positions"], s["slots"] = _ints(pos), _ints(slots)
    if case["layout"] == "paged":
        s["k"], s["v"] = _paged_caches(nb, case, gen)
    elif case["layout"] == "token":
        shape = (num_slots, H, D)
        s["k"], s["v"] = _values(shape, case["cache"], gen), _values(shape, case["cache"], gen)
    return s


# ---- one pass -------------------------------------------------------------------


def _kernels():
    """The package (one level below the repository's root), only where `own` is true."""
    root = os.path.abspath("sglang-mlx_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from sglang_mlx_amd import kernels
    return kernels


def run(s):
    case = s["case"]
    return {"tables": _run_tables, "rope": _run_rope, "window": _run_window, "extend": _run_extend}[case["kind"]](s)


def _run_tables(s):
    bs = s["case"]["block_size"]
    if own:
        out = _kernels().build_step_tables(s["pool"], s["rows"], s["ctx"], s["new"], s["new_blocks"], bs,
                                             s["tokens"])
        return (*out, s["pool"])
    pool, W = s["pool"], s["pool"].shape[1]
    live = s["rows"] >= 0
    row = s["rows"].clamp(min=0).long()
    ctx = torch.where(live, s["ctx"], 0).long()
    new = torch.where(live, s["new"], 0).long()
    have, need = (ctx - new + bs - 1) // bs, (ctx + bs - 1) // bs
    taken = torch.cumsum(need - have, 0)
    start = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(new, 0)])
    cols = torch.arange(W, device=DEV)
    fresh = (cols >= have[:, None]) & (cols < need[:, None])
    which = (taken - (need - have))[:, None] + cols - have[:, None]
    which = which.clamp(0, s["new_blocks"].numel() - 1)
    table = torch.where(fresh, s["new_blocks"][which], torch.where(cols < have[:, None], pool[row], -1))
    at = torch.where(fresh & live[:, None], row[:, None] * W + cols, pool.numel())
    flat = torch.cat([pool.view(-1), pool.new_zeros(1)])
    flat[at.view(-1)] = table.view(-1)
    pool.copy_(flat[:-1].view_as(pool))
    t = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(start[1:], t, right=True)
    real = seq < row.numel()
    seq = seq.clamp(max=row.numel() - 1)
    pos = torch.where(real, (ctx - new)[seq] + t - start[seq], 0)
    slot = torch.where(real, table[seq, (pos // bs).clamp(max=W - 1)].long() * bs + pos % bs, -1)
    return table, slot.int(), pos.int(), start.int(), pool


def _norm_rotate(x, weight, cos, sin, rot, interleaved):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    turn, rest = x[..., :rot], x[..., rot:]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if interleaved else turn.split(rot // 2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    turn = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turn, rest], -1)


def _run_rope(s):
    case = s["case"]
    if own:
        k = _kernels()
        more = dict(s["weights"], eps=EPS, interleaved=case["interleaved"])
        if case["layout"] == "none":
            return k.qk_norm_rope(s["query"], s["key"], s["positions"], s["cos_sin"], **more)
        return k.qk_norm_rope_and_cache(s["query"], s["key"], s["value"], s["positions"], s["cos_sin"], s["k"],
                                        s["v"], s["slots"], **more)
    rot, D = case["rot"], case["head_size"]
    cs = s["cos_sin"][s["positions"]][:, None]
    cos, sin = cs[..., :rot // 2], cs[..., rot // 2:]
    q = _norm_rotate(s["query"], s["weights"].get("q_weight"), cos, sin, rot, case["interleaved"])
    k = _norm_rotate(s["key"], s["weights"].get("k_weight"), cos, sin, rot, case["interleaved"])
    q = q.to(s["query"].dtype)
    if case["layout"] == "none":
        return q, k.to(s["key"].dtype)
    k, v = k.to(s["k"].dtype), s["value"].to(s["v"].dtype)
    if case["layout"] == "token":
        s["k"][s["slots"]] = k
        s["v"][s["slots"]] = v
        return q, s["k"], s["v"]
    blk, off = s["slots"] // case["block_size"], s["slots"] % case["block_size"]
    x = s["k"].shape[4]
    s["k"][blk, :, :, off, :] = k.view(-1, case["kv_heads"], D // x, x)
    s["v"][blk, :, :, off] = v
    return q, s["k"], s["v"]


def _code_values():
    """The 256 E4M3 codes (bias 7; exponent 15 is not used) as float64."""
    c = torch.arange(256, dtype=torch.int64, device=DEV)
    e, m = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e.double() - 7))
    return torch.where(c >= 128, -mag, mag)


def _keys_values(s, i, lo, hi):
    """K and V of tokens [lo, hi) of sequence i: [H, D, T] and [H, T, D] in 32 bits."""
    case = s["case"]
    H, D, bs = case["kv_heads"], case["head_size"], case["block_size"]
    ids = s["table"][i, lo // bs:-(-hi // bs)]
    k, v = s["k"][ids], s["v"][ids]
    if case["cache"] == "fp8":
        k, v = s["codes"][k.int()] * K_SCALE, s["codes"][v.int()] * V_SCALE
    at = lo - lo // bs * bs
    k = k.float().permute(1, 2, 4, 0, 3).reshape(H, D, -1)[..., at:at + hi - lo]
    v = v.float().permute(1, 0, 3, 2).reshape(H, -1, D)[:, at:at + hi - lo]
    return k, v


def _attend(s, i, q, first, ctx):
    """Queries q [n, Hq, D] at positions first, first + 1, ... of sequence i."""
    case = s["case"]
    H, D, window, sinks = case["kv_heads"], case["head_size"], case["window"], case["sinks"]
    n, group = q.shape[0], case["heads"] // H
    lo = 0
    if window:
        lo = max(0, first - window + 1)
    lead = min(sinks, lo) if window else 0
    k, v = _keys_values(s, i, lo, min(ctx, first + n))
    key_pos = torch.arange(lo, min(ctx, first + n), device=DEV)
    if lead:
        k0, v0 = _keys_values(s, i, 0, lead)
        k, v = torch.cat([k0, k], 2), torch.cat([v0, v], 1)
        key_pos = torch.cat([torch.arange(lead, device=DEV), key_pos])
    pos = torch.arange(first, first + n, device=DEV)[:, None]
    seen = key_pos <= pos
    if window:
        seen &= (key_pos > pos - window) | (key_pos < sinks)
    out = torch.empty((n, case["heads"], D), dtype=q.dtype, device=DEV)
    step = max(1, PLAIN_SCORES // (n * key_pos.numel() * group))
    for h in range(0, H, step):
        hs = min(step, H - h)
        qh = q[:, h * group:(h + hs) * group].float().view(n, hs, group, D).permute(1, 2, 0, 3)
        sc = torch.matmul(qh.reshape(hs, group * n, D), k[h:h + hs].contiguous()).view(hs, group, n, -1)
        sc = (sc * s["scale"]).masked_fill(~seen, float("-inf"))
        p = torch.exp(sc - sc.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(hs, group * n, -1), v[h:h + hs].contiguous()).view(hs, group, n, D)
        out[:, h * group:(h + hs) * group] = o.permute(2, 0, 1, 3).reshape(n, hs * group, D).to(q.dtype)
    return out


def _run_window(s):
    case = s["case"]
    if own:
        return _kernels().paged_attention_window(s["query"], s["k"], s["v"], s["table"], s["ctx"],
                                                   case["kv_heads"], s["scale"], case["block_size"],
                                                   s["max_seq_len"], case["window"], case["sinks"], **s["scales"])
    return torch.cat([_attend(s, i, s["query"][i:i + 1], c - 1, c) for i, (c, _) in enumerate(s["host"])])


def _run_extend(s):
    case = s["case"]
    if own:
        return _kernels().paged_attention_extend(s["query"], s["k"], s["v"], s["table"], s["ctx"], s["start"],
                                                   case["kv_heads"], s["scale"], case["block_size"],
                                                   s["max_seq_len"], s["max_query_len"], case["window"],
                                                   case["sinks"], **s["scales"])
    group = case["heads"] // case["kv_heads"]
    out, at = [], 0
    for i, (c, n) in enumerate(s["host"]):
        step = max(1, PLAIN_SCORES // (c * group))
        for j in range(0, n, step):
            m = min(step, n - j)
            out.append(_attend(s, i, s["query"][at + j:at + j + m], c - n + j, c))
        at += n
    return torch.cat(out)


# ---- what a pass cannot do without ------------------------------------------------


def work(case):
    if case["kind"] == "tables":
        ctx, new = _batch_lengths(case)
        bs, pad = case["block_size"], case["pad"]
        width = -(-case["hi"] // bs) + 1
        held, total = int((-(-(ctx - new) // bs)).sum()), int((-(-ctx // bs)).sum())
        rows, tokens = case["batch"] + pad, int(new.sum()) + 7 * pad
        read = held + (total - held) + 3 * rows
        return {"bytes": 4 * (read + rows * width + (total - held) + 2 * tokens + rows + 1), "flops": 0}
    Hq, H, D = case["heads"], case["kv_heads"], case["head_size"]
    if case["kind"] == "rope":
        N, qb = case["tokens"], BYTES[case["q"]]
        nbytes = 2 * N * Hq * D * qb + N * (case["rot"] * 4 + 4)
        if case["layout"] == "none":
            nbytes += 2 * N * H * D * qb
        else:
            nbytes += 2 * N * H * D * (qb + BYTES[case["cache"]]) + 4 * N
        return {"bytes": nbytes, "flops": N * (Hq + H) * (3 * case["rot"] + 4 * D)}
    ctx, new = _batch_lengths(case)
    window, sinks, cb = case["window"], case["sinks"], BYTES[case["cache"]]
    pairs = read = 0
    for c, n in zip(ctx.tolist(), new.tolist()):
        first = np.arange(c - n, c, dtype=np.int64)
        if window:
            lo = np.maximum(0, first - window + 1)
            pairs += int((first + 1 - lo + np.minimum(sinks, lo)).sum())
            read += c - int(lo[0]) + min(sinks, int(lo[0]))
        else:
            pairs += int((first + 1).sum())
            read += c
    nbytes = 2 * read * H * D * cb + 2 * int(new.sum()) * Hq * D * BYTES[case["q"]]
    nbytes += 4 * read // case["block_size"] + 8 * case["batch"]
    return {"bytes": nbytes, "flops": 4 * pairs * Hq * D}


# ---- the same in 64 bits ----------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_rope(case, s) if case["kind"] == "rope" else _exact_attention(case, s)


def _exact_rope(case, s):
    rot = case["rot"]
    half = rot // 2
    turn = s["cos_sin"].double()[s["positions"].long()]
    factor = torch.complex(turn[:, :half], turn[:, half:])[:, None, :]

    def whole(x, weight):
        y = x.double().clone()
        if weight is not None:
            y /= (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt()
            y *= weight.double()
        first = torch.arange(0, rot, 2, device=DEV) if case["interleaved"] else torch.arange(half, device=DEV)
        second = first + (1 if case["interleaved"] else half)
        z = torch.complex(y[..., first], y[..., second]) * factor
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q = whole(s["query"], s["weights"].get("q_weight"))
    k = whole(s["key"], s["weights"].get("k_weight"))
    if case["layout"] == "none":
        return q, k
    kc, vc, slots = s["k"].double(), s["v"].double(), s["slots"].long()
    if case["layout"] == "token":
        kc.index_copy_(0, slots, k)
        vc.index_copy_(0, slots, s["value"].double())
        return q, kc, vc
    bs = case["block_size"]
    nb, H, chunks, _, x = kc.shape
    rows = kc.permute(0, 3, 1, 2, 4).reshape(nb * bs, H, chunks * x).contiguous()
    rows.index_copy_(0, slots, k)
    kc = rows.view(nb, bs, H, chunks, x).permute(0, 2, 3, 1, 4).contiguous()
    rows = vc.permute(0, 3, 1, 2).reshape(nb * bs, H, -1).contiguous()
    rows.index_copy_(0, slots, s["value"].double())
    return q, kc, rows.view(nb, bs, H, -1).permute(0, 2, 3, 1).contiguous()


def _exact_attention(case, s):
    if work(case)["flops"] > 2.5e12:
        return None
    H, D, bs = case["kv_heads"], case["head_size"], case["block_size"]
    group, window, sinks = case["heads"] // H, case["window"], case["sinks"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    codes = _code_values()
    at = 0
    for i, (c, n) in enumerate(s["host"]):
        pos = torch.arange(c, device=DEV)
        ids = s["table"][i].long()[pos // bs]
        keep = pos >= 0
        if window:
            keep = (pos > c - n - window) | (pos < sinks)
        pos, ids = pos[keep], ids[keep]
        for h in range(H):
            k = s["k"][ids, h, :, pos % bs, :].reshape(-1, D)
            v = s["v"][ids, h, :, pos % bs]
            if case["cache"] == "fp8":
                k, v = codes[k.long()] * K_SCALE, codes[v.long()] * V_SCALE
            k, v = k.double(), v.double()
            step = max(1, (1 << 26) // (group * pos.numel()))
            for j in range(0, n, step):
                m = min(step, n - j)
                rows = s["query"][at + j:at + j + m, h * group:(h + 1) * group].double()
                mine = (torch.arange(j, j + m, device=DEV) + c - n)[:, None]
                hidden = pos[None] > mine
                if window:
                    hidden |= (pos[None] <= mine - window) & (pos[None] >= sinks)
                sc = (rows.reshape(m * group, D) @ k.t().contiguous()).view(m, group, -1) * s["scale"]
                sc.masked_fill_(hidden[:, None], -math.inf)
                p = torch.softmax(sc, -1).view(m * group, -1)
                out[at + j:at + j + m, h * group:(h + 1) * group] = (p @ v).view(m, group, D)
        at += n
    return out
