"""Performance cases of a KV cache held in 8 bits, with a scale for each block of
tokens and KV head, and of the attention beside it.

Kinds, each one call of a serving program on tensors that it already holds:

  store    the newest keys and values of each sequence, quantised into the cache
           with the scales of the blocks that they touch
  read     the first tokens of each sequence, back from the cache in 16 or 32 bits
  scaled   attention of single and drafted tokens over that cache
  prompt   causal attention of packed prompts over their keys and values as they
           left the projection (or, behind a context, as `read` gives them)

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
F8 = torch.float8_e4m3fn  # what a code below exponent 15 stands for, without its scale
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MOST = 240.0  # the largest value of a code
# Queries are this much wider than unit normal, so that a softmax row has the
# peaks that attention over a real context has.
Q_GAIN = 2.0

# The most that a drawn case costs: tokens of a store or a read, cache bytes of a
# scaled call, score elements and operations of a prompt.
DRAW_TOKENS = 16384
DRAW_BYTES = 3.0e8
DRAW_SCORES = 32 * 8192 * 8192
DRAW_FLOPS = 5.4e11


def listed():
    return [
        # One user's decode step: one token of 8 KV heads of 128, latency.
        dict(name="store_b1", kind="store", src="bf16", batch=1, kv_heads=8, head_size=128, block_size=16, lo=1500,
             hi=1500, new_lo=1, new_hi=1),
        # A loaded server's decode step, one token each into blocks of 32.
        dict(name="store_decode_b200", kind="store", src="f16", batch=200, kv_heads=4, head_size=128, block_size=32,
             lo=40, hi=700, new_lo=1, new_hi=1),
        # A prefill of ragged prompts and chunks, 16K tokens, most of them beginning inside a block.
        dict(name="store_prefill_16k", kind="store", src="bf16", batch=23, kv_heads=8, head_size=128, block_size=16,
             lo=100, hi=2600, new_lo=95, new_hi=1329),
        # A request that continues a cached prefix of 1001 tokens of a small model.
        dict(name="read_b1_1k", kind="read", out="f16", batch=1, kv_heads=2, head_size=64, block_size=16, lo=1001,
             hi=1001),
        # Contexts of 11 chunked prefills, 32K tokens, into the form that their attention reads.
        dict(name="read_32k", kind="read", out="bf16", batch=11, kv_heads=8, head_size=128, block_size=16, lo=700,
             hi=5258),
        # One user with a context of 8K: latency.
        dict(name="scaled_b1_8k", kind="scaled", q="bf16", batch=1, heads=32, kv_heads=8, head_size=128,
             block_size=16, lo=8190, hi=8190, new=1, window=0, sinks=0),
        # A loaded server's decode step: 64 requests of 533 to 4097 tokens.
        dict(name="scaled_b64", kind="scaled", q="bf16", batch=64, heads=32, kv_heads=8, head_size=128,
             block_size=16, lo=533, hi=4097, new=1, window=0, sinks=0),
        # Verification of 4 drafted tokens in each of 24 requests, blocks of 32.
        dict(name="scaled_draft_b24", kind="scaled", q="f16", batch=24, heads=32, kv_heads=8, head_size=128,
             block_size=32, lo=301, hi=7000, new=4, window=0, sinks=0),
        # Three long documents, 7 query heads to a KV head.
        dict(name="scaled_b3_long", kind="scaled", q="bf16", batch=3, heads=28, kv_heads=4, head_size=128,
             block_size=16, lo=40001, hi=130000, new=1, window=0, sinks=0),
        # One short prompt: latency.
        dict(name="prompt_b1_177", kind="prompt", q="bf16", batch=1, heads=32, kv_heads=8, head_size=128, lo=177,
             hi=177, ctx_lo=0, ctx_hi=0, window=0, sinks=0),
        # 9 ragged prompts of a model with 14 query heads of 64, 8K tokens.
        dict(name="prompt_ragged_8k", kind="prompt", q="f16", batch=9, heads=14, kv_heads=2, head_size=64, lo=61,
             hi=1759, ctx_lo=0, ctx_hi=0, window=0, sinks=0),
        # One long prompt of 8K tokens.
        dict(name="prompt_b1_8k", kind="prompt", q="bf16", batch=1, heads=32, kv_heads=8, head_size=128, lo=8192,
             hi=8192, ctx_lo=0, ctx_hi=0, window=0, sinks=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store"] * 3 + ["read"] * 2 + ["scaled"] * 4 + ["prompt"] * 4)
    Hq, H = rng.choice([(32, 8), (32, 8), (28, 4), (14, 2), (8, 1), (16, 16), (64, 8)])
    if kind in ("store", "read"):
        D = rng.choice([64, 96, 128, 128, 128, 256])
        case = dict(kind=kind, kv_heads=H, head_size=D, block_size=rng.choice([8, 16, 16, 32]))
        most = max(64, DRAW_TOKENS * 1024 // max(1024, H * D))
        if kind == "read":
            tokens = _log_int(rng, 1, 2 * most)
            case["out"] = rng.choice(["bf16", "bf16", "f16", "f32"])
            if case["out"] == "f32":
                tokens = max(1, tokens // 2)
            batch = min(tokens, _log_int(rng, 1, 64))
            lo = max(1, int(tokens / batch * rng.uniform(0.1, 1.0)))
            return dict(case, batch=batch, lo=lo, hi=max(lo, 2 * (tokens // batch) - lo))
        case["src"] = rng.choice(["bf16", "bf16", "f16", "f32"])
        tokens = _log_int(rng, 1, most // (2 if case["src"] == "f32" else 1))
        batch = min(tokens, _log_int(rng, 1, 256))
        new_lo = max(1, int(tokens / batch * rng.uniform(0.1, 1.0)))
        new_hi = max(new_lo, 2 * (tokens // batch) - new_lo)
        lo = rng.choice([new_hi, new_hi + 3, new_hi + _log_int(rng, 1, 500)])
        return dict(case, batch=batch, lo=lo, hi=lo + rng.choice([0, _log_int(rng, 1, 500)]), new_lo=new_lo,
                    new_hi=new_hi)
    q = rng.choice(["bf16", "bf16", "f16"])
    window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
    sinks = rng.choice([0, 4, 33]) if window else 0
    if kind == "scaled":
        D = rng.choice([64, 96, 128, 128, 128, 256])
        mean = _log_int(rng, 16, min(60000, int(DRAW_BYTES / (2 * H * D))))
        batch = min(_log_int(rng, 1, 256), int(DRAW_BYTES / (2 * H * D * mean)))
        new = rng.choice([1, 1, 1, 2, 4, 5])
        lo = max(new, int(mean * rng.uniform(0.1, 1.0)))
        return dict(kind=kind, q=q, batch=batch, heads=Hq, kv_heads=H, head_size=D,
                    block_size=rng.choice([8, 16, 16, 32]), lo=lo, hi=max(lo, 2 * mean - lo), new=new, window=window,
                    sinks=sinks)
    D = rng.choice([64, 80, 128, 128, 128, 256])
    hi = _log_int(rng, 1, 8192)
    ctx_hi = rng.choice([0, 0, _log_int(rng, 1, 8192)])
    if 4 * Hq * D * hi * (hi / 2 + ctx_hi) > DRAW_FLOPS:
        hi, ctx_hi = hi // 3 + 1, ctx_hi // 3
    most = min(DRAW_SCORES / (Hq * hi * (hi + ctx_hi)), DRAW_FLOPS / (4 * Hq * D * hi * (hi / 2 + ctx_hi + 1)))
    batch = max(1, min(_log_int(rng, 1, 64), int(most)))
    return dict(kind=kind, q=q, batch=batch, heads=Hq, kv_heads=H, head_size=D,
                lo=max(1, int(hi * rng.uniform(0.02, 1.0))), hi=hi, ctx_lo=int(ctx_hi * rng.uniform(0.0, 1.0)),
                ctx_hi=ctx_hi, window=window, sinks=sinks)


# ---- inputs ---------------------------------------------------------------------


def _spread(lo, hi, n):
    """n lengths spread evenly over [lo, hi]."""
    return np.array([lo + int((hi - lo) * (i + 0.5) / n + 0.5) for i in range(n)], dtype=np.int64)


def _lengths(case):
    """(context, new tokens) of each sequence, by a fixed rule."""
    B = case["batch"]
    pair = np.arange(B) * 7919 % B
    if case["kind"] == "prompt":
        new = _spread(case["lo"], case["hi"], B)
        return new + _spread(case["ctx_lo"], case["ctx_hi"], B)[pair], new
    ctx = _spread(case["lo"], case["hi"], B)
    if case["kind"] == "store":
        return ctx, np.minimum(_spread(case["new_lo"], case["new_hi"], B)[pair], ctx)
    return ctx, ctx if case["kind"] == "read" else np.full(B, case["new"])


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _starts(lens):
    return _ints(np.concatenate([[0], np.cumsum(lens)]))


def _codes(shape, gen):
    """Codes of normal values whose largest in a block comes near the largest code."""
    x = torch.empty(shape, dtype=torch.float16, device=DEV).normal_(generator=gen)
    return x.mul_(55.0).clamp_(-MOST, MOST).to(F8).view(torch.uint8)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": case}
    ctx, new = _lengths(case)
    order = rng.permutation(case["batch"])  # the seed draws the order of the sequences
    ctx, new = ctx[order], new[order]
    D, H = case["head_size"], case["kv_heads"]
    s["start"] = _starts(new)
    s["max_new"], s["max_ctx"], s["tokens"] = int(new.max()), int(ctx.max()), int(new.sum())
    if case["kind"] == "prompt":
        dt, Hq, scale = TORCH[case["q"]], case["heads"], 1.0 / math.sqrt(D)
        if case["ctx_hi"]:
            # Queries of a chunk; keys and values of its context and of itself.
            s["query"] = torch.empty((s["tokens"], Hq, D), device=DEV).normal_(generator=gen).mul_(Q_GAIN).to(dt)
            s["key"], s["value"] = (torch.empty((int(ctx.sum()), H, D), dtype=dt, device=DEV).normal_(generator=gen)
                                    for _ in range(2))
        else:
            # Queries, keys and values are views of one projection's output.
            qkv = torch.empty((s["tokens"], (Hq + 2 * H) * D), device=DEV).normal_(generator=gen)
            qkv[:, :Hq * D] *= Q_GAIN
            qkv = qkv.to(dt)
            s["query"] = qkv[:, :Hq * D].unflatten(1, (Hq, D))
            s["key"] = qkv[:, Hq * D:(Hq + H) * D].unflatten(1, (H, D))
            s["value"] = qkv[:, (Hq + H) * D:].unflatten(1, (H, D))
        s["key_start"], s["scale"] = _starts(ctx), scale
        return s
    bs = case["block_size"]
    need = -(-ctx // bs)
    used = int(need.sum())
    nb = used + used // 10 + 2
    ids = rng.permutation(nb - 1)[:used] + 1
    table = np.full((case["batch"], int(need.max())), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    s["table"], s["ctx"] = _ints(table), _ints(ctx)
    s["k"], s["v"] = _codes((nb, H, D // 16, bs, 16), gen), _codes((nb, H, D, bs), gen)
    # Scales as the store writes them, powers of two, so that values are about unit normal.
    exponent = torch.randint(-7, -4, (nb, H, 2), generator=gen, device=DEV)
    s["scales"] = torch.ldexp(torch.ones((), device=DEV), exponent)
    if case["kind"] == "store":
        # Keys and values: views of one projection's output; a few heads are wider than the others.
        kv = torch.empty((s["tokens"], 2 * H * D), device=DEV).normal_(generator=gen)
        kv *= torch.empty(2 * H, device=DEV).uniform_(0.5, 3.0, generator=gen).repeat_interleave(D)
        kv = kv.to(TORCH[case["src"]])
        s["key"], s["value"] = (x.unflatten(1, (H, D)) for x in kv.split(H * D, 1))
    elif case["kind"] == "scaled":
        s["query"] = torch.empty((s["tokens"], case["heads"], D), device=DEV).normal_(generator=gen).mul_(Q_GAIN).to(
            TORCH[case["q"]])
        s["scale"] = 1.0 / math.sqrt(D)
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
    return {"store": _run_store, "read": _run_read, "scaled": _run_scaled, "prompt": _run_prompt}[s["case"]["kind"]](s)


def _places(s, start, first):
    """Sequence, position, block and offset of each token of a packed batch; `first`: each sequence's first position."""
    bs = s["case"]["block_size"]
    t = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(start[1:], t, right=True)
    pos = first[seq] + t - start[seq]
    return seq, pos, s["table"][seq, pos // bs].long(), pos % bs


def _scale_of(amax):
    """The least power of two that brings amax to at most MOST."""
    m, e = torch.frexp(amax)  # MOST is 0.9375 * 2^8
    e = torch.where(amax == 0, -126, torch.where(m > 0.9375, e - 7, e - 8)).clamp(min=-126)
    return torch.ldexp(torch.ones((), device=DEV), e)


def _run_store(s):
    case = s["case"]
    if own:
        _kernels().quantize_and_cache(s["key"], s["value"], s["k"], s["v"], s["scales"], s["table"], s["ctx"],
                                      s["start"])
        return s["k"].view(F8), s["v"].view(F8), s["scales"]
    H, D, bs, nb = case["kv_heads"], case["head_size"], case["block_size"], s["k"].shape[0]
    start, first = s["start"].long(), (s["ctx"] - (s["start"][1:] - s["start"][:-1])).long()
    _, _, block, off = _places(s, start, first)
    k, v = s["key"].float(), s["value"].float()
    amax = torch.stack([k.abs().amax(-1), v.abs().amax(-1)], -1)
    amax = torch.zeros((nb, H, 2), device=DEV).index_reduce_(0, block, amax, "amax")
    touched = torch.zeros(nb, dtype=torch.bool, device=DEV).index_fill_(0, block, True)[:, None, None]
    # A sequence's first block may hold earlier tokens; every other one begins anew.
    head, held = s["table"].gather(1, (first // bs)[:, None])[:, 0].long(), first % bs
    old = torch.zeros_like(s["scales"]).index_copy_(0, head, s["scales"][head] * (held > 0)[:, None, None])
    new = torch.maximum(old, _scale_of(amax))
    shrink = (old / new)[head]
    mine = torch.arange(bs, device=DEV) < held[:, None]
    kc, vc = s["k"][head], s["v"][head]
    ks = (kc.view(F8).float() * shrink[:, :, 0, None, None, None]).to(F8).view(torch.uint8)
    vs = (vc.view(F8).float() * shrink[:, :, 1, None, None]).to(F8).view(torch.uint8)
    s["k"][head] = torch.where(mine[:, None, None, :, None], ks, kc)
    s["v"][head] = torch.where(mine[:, None, None, :], vs, vc)
    k = (k / new[block][:, :, 0, None]).to(F8).view(torch.uint8)
    v = (v / new[block][:, :, 1, None]).to(F8).view(torch.uint8)
    s["k"][block, :, :, off, :] = k.view(-1, H, D // 16, 16)
    s["v"][block, :, :, off] = v
    s["scales"].copy_(torch.where(touched, new, s["scales"]))
    return s["k"].view(F8), s["v"].view(F8), s["scales"]


def _rows(s, block, off):
    """Keys and values of the tokens at (block, off), in 32 bits: [..., H, D]."""
    scale = s["scales"][block]
    k = s["k"].permute(0, 3, 1, 2, 4)[block, off].flatten(-2).view(F8).float() * scale[..., 0, None]
    v = s["v"].permute(0, 3, 1, 2)[block, off].view(F8).float() * scale[..., 1, None]
    return k, v


def _run_read(s):
    dt = TORCH[s["case"]["out"]]
    if own:
        return _kernels().dequantize_cache(s["k"], s["v"], s["scales"], s["table"], s["start"], s["tokens"], dt)
    start = s["start"].long()
    _, _, block, off = _places(s, start, torch.zeros_like(start))
    k, v = _rows(s, block, off)
    return k.to(dt), v.to(dt)


def _attend(q, k, v, hidden, scale):
    """q [B, n, Hq, D], k and v [B, T, H, D], hidden [B, n, T]: [B, n, Hq, D] in 32 bits."""
    B, n, Hq, D = q.shape
    T, H = k.shape[1:3]
    q = q.unflatten(2, (H, Hq // H)).permute(0, 2, 3, 1, 4).reshape(B * H, -1, D)
    k = k.permute(0, 2, 3, 1).reshape(B * H, D, T)
    v = v.permute(0, 2, 1, 3).reshape(B * H, T, D)
    p = torch.bmm(q, k).mul_(scale).view(B, Hq, n, T)
    p.masked_fill_(hidden[:, None], float("-inf"))
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    return torch.bmm(p.view(B * H, -1, T), v).view(B, Hq, n, D).transpose(1, 2)


def _run_scaled(s):
    case = s["case"]
    H, bs, n, window, sinks = case["kv_heads"], case["block_size"], case["new"], case["window"], case["sinks"]
    if own:
        return _kernels().paged_attention_scaled(
            s["query"], s["k"], s["v"], s["scales"], s["table"], s["ctx"], s["start"] if n > 1 else None, H,
            s["scale"], bs, s["max_ctx"], n, window, sinks)
    first = s["ctx"].long()[:, None] - n
    # The keys that a sequence's queries may see: the window's, and the first ones before it.
    low = (first - window + 1).clamp(min=0) if window else torch.zeros_like(first)
    count = min(s["max_ctx"], window + n - 1) if window else s["max_ctx"]
    lead = torch.arange(min(sinks, s["max_ctx"]), device=DEV).expand(case["batch"], -1)
    pos = torch.cat([lead, low + torch.arange(count, device=DEV)], 1)
    gone = torch.cat([lead >= low, pos[:, lead.shape[1]:] >= first + n], 1)
    at = torch.where(gone, 0, pos)
    k, v = _rows(s, s["table"].gather(1, at // bs).long(), at % bs)
    mine = (first + torch.arange(n, device=DEV))[:, :, None]
    pos = pos[:, None]
    hidden = gone[:, None] | (pos > mine)
    if window:
        hidden |= (pos <= mine - window) & (pos >= sinks)
    q = s["query"].float().unflatten(0, (-1, n))
    return _attend(q, k, v, hidden, s["scale"]).flatten(0, 1).to(s["query"].dtype)


def _run_prompt(s):
    case = s["case"]
    window, sinks = case["window"], case["sinks"]
    if own:
        return _kernels().prompt_attention(s["query"], s["key"], s["value"], s["start"], s["scale"], s["max_new"],
                                           s["key_start"] if case["ctx_hi"] else None,
                                           s["max_ctx"] if case["ctx_hi"] else None, window, sinks)
    # Padded to the longest sequence.
    start, key_start = s["start"].long(), s["key_start"].long()
    new, ctx = (start[1:] - start[:-1])[:, None], (key_start[1:] - key_start[:-1])[:, None]
    i, t = torch.arange(s["max_new"], device=DEV), torch.arange(s["max_ctx"], device=DEV)
    q = s["query"][(start[:-1, None] + i).clamp(max=s["query"].shape[0] - 1)].float()
    at = (key_start[:-1, None] + t).clamp(max=s["key"].shape[0] - 1)
    mine = (ctx - new + i)[:, :, None]
    hidden = (t > mine) | (t >= ctx[:, :, None])
    if window:
        hidden |= (t <= mine - window) & (t >= sinks)
    out = _attend(q, s["key"][at].float(), s["value"][at].float(), hidden, s["scale"])
    row = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(start[1:], row, right=True)
    return out[seq, row - start[seq]].to(s["query"].dtype)


# ---- what a pass cannot do without ------------------------------------------------


def work(case):
    ctx, new = _lengths(case)
    H, D, B = case["kv_heads"], case["head_size"], case["batch"]
    if case["kind"] == "store":
        N, bs = int(new.sum()), case["block_size"]
        blocks = int((-(-ctx // bs) - (ctx - new) // bs).sum())
        return {"bytes": 2 * N * H * D * (BYTES[case["src"]] + 1) + 8 * H * (blocks + B) + 4 * (blocks + 2 * B),
                "flops": 4 * N * H * D}
    if case["kind"] == "read":
        N, bs = int(ctx.sum()), case["block_size"]
        blocks = int((-(-ctx // bs)).sum())
        return {"bytes": 2 * N * H * D * (BYTES[case["out"]] + 1) + 8 * H * blocks + 4 * (blocks + B),
                "flops": 2 * N * H * D}
    Hq, window, sinks = case["heads"], case["window"], case["sinks"]
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
    nbytes = 2 * int(new.sum()) * Hq * D * BYTES[case["q"]] + 8 * B
    if case["kind"] == "scaled":
        nbytes += 2 * read * H * D + read // case["block_size"] * (8 * H + 4)
    else:
        nbytes += 2 * read * H * D * BYTES[case["q"]]
    return {"bytes": nbytes, "flops": 4 * pairs * Hq * D}


# ---- the same in 64 bits ----------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "read": _exact_read, "scaled": _exact_attention,
            "prompt": _exact_attention}[case["kind"]](case, s)


def _code_values():
    """The 256 codes (4 exponent bits of bias 7, 3 of the significand) as float64."""
    c = torch.arange(256, dtype=torch.int64, device=DEV)
    e, m = (c >> 3) & 15, (c & 7).double()
    size = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e.double() - 7))
    return torch.where(c >= 128, -size, size)


def _host(s):
    start = s["start"].tolist()
    table, ctx = s["table"].cpu().numpy(), s["ctx"].tolist()
    return [(table[i], ctx[i], start[i], start[i + 1] - start[i]) for i in range(len(ctx))]


def _exact_store(case, s):
    """Block by block: the codes' values before their rounding, in units of the block's scale."""
    values, bs, H, D = _code_values(), case["block_size"], case["kv_heads"], case["head_size"]
    kc, vc, scales = values[s["k"].long()], values[s["v"].long()], s["scales"].double()
    key, value = s["key"].double(), s["value"].double()
    blocks, spans = [], []
    for ids, c, at, n in _host(s):
        for j in range((c - n) // bs, -(-c // bs)):
            lo, hi = max(j * bs, c - n), min((j + 1) * bs, c)
            blocks.append(int(ids[j]))
            spans.append((lo - j * bs, hi - j * bs, at + lo - (c - n)))
    ids = torch.tensor(blocks, device=DEV)
    lo, hi, row = (torch.tensor(x, device=DEV)[:, None] for x in zip(*spans))
    off = torch.arange(bs, device=DEV)
    fresh = (off >= lo) & (off < hi)
    rows = (row + off - lo).clamp(0, key.shape[0] - 1)
    for x, cache, which in ((key, kc, 0), (value, vc, 1)):
        x = torch.where(fresh[:, :, None, None], x[rows], 0.0)  # [blocks, bs, H, D]
        ratio = (x.abs().amax((1, 3)) / 240).clamp(min=2.0 ** -126)
        scale = torch.pow(2.0, torch.ceil(torch.log2(ratio)))
        before = scales[ids, :, which]
        scale = torch.where(lo > 0, torch.maximum(scale, before), scale)
        x = x / scale[:, None, :, None]
        if which == 0:
            x = x.view(-1, bs, H, D // 16, 16).permute(0, 2, 3, 1, 4)
            expand = lambda m: m[:, None, None, :, None]  # noqa: E731
        else:
            x = x.permute(0, 2, 3, 1)
            expand = lambda m: m[:, None, None, :]  # noqa: E731
        was = cache[ids]
        factor = (before / scale).view(before.shape + (1,) * (was.dim() - 2))
        cache[ids] = torch.where(expand(fresh), x, torch.where(expand(off < lo), was * factor, was))
        scales[ids, :, which] = scale
    return kc, vc, scales


def _exact_rows(case, s, ids, lo, hi):
    """Keys and values of tokens [lo, hi) of the sequence with blocks ids: [T, H, D] each."""
    values, bs = _code_values(), case["block_size"]
    pos = torch.arange(lo, hi, device=DEV)
    block = torch.from_numpy(ids.astype(np.int64)).to(DEV)[pos // bs]
    scale = s["scales"].double()[block]
    k = values[s["k"][block, :, :, pos % bs, :].long()].flatten(2) * scale[:, :, :1]
    v = values[s["v"][block, :, :, pos % bs].long()] * scale[:, :, 1:]
    return k, v


def _exact_read(case, s):
    rows = [_exact_rows(case, s, ids, 0, c) for ids, c, _, _ in _host(s)]
    return torch.cat([k for k, _ in rows]), torch.cat([v for _, v in rows])


def _exact_attention(case, s):
    """Sequence by sequence and KV head by KV head."""
    H, D, window, sinks = case["kv_heads"], case["head_size"], case["window"], case["sinks"]
    group = case["heads"] // H
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    if case["kind"] == "scaled":
        seqs = _host(s)
    else:
        start, key_start = s["start"].tolist(), s["key_start"].tolist()
        seqs = [(key_start[i], key_start[i + 1] - key_start[i], start[i], start[i + 1] - start[i])
                for i in range(case["batch"])]
    for where, c, at, n in seqs:
        low = max(0, c - n - window + 1) if window else 0
        if case["kind"] == "scaled":
            pieces = [_exact_rows(case, s, where, 0, min(sinks, low)), _exact_rows(case, s, where, low, c)]
            k, v = (torch.cat(x) for x in zip(*pieces))
            pos = torch.cat([torch.arange(min(sinks, low), device=DEV), torch.arange(low, c, device=DEV)])
        else:
            k, v = s["key"][where:where + c].double(), s["value"][where:where + c].double()
            pos = torch.arange(c, device=DEV)
        step = max(1, (1 << 26) // (group * pos.numel()))
        for h in range(H):
            kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
            for j in range(0, n, step):
                m = min(step, n - j)
                rows = s["query"][at + j:at + j + m, h * group:(h + 1) * group].double()
                mine = torch.arange(c - n + j, c - n + j + m, device=DEV)[:, None]
                hidden = pos > mine
                if window:
                    hidden |= (pos <= mine - window) & (pos >= sinks)
                sc = (rows.reshape(m * group, D) @ kt).view(m, group, -1) * s["scale"]
                p = torch.softmax(sc.masked_fill(hidden[:, None], -math.inf), -1)
                out[at + j:at + j + m, h * group:(h + 1) * group] = (p.view(m * group, -1) @ vh).view(m, group, D)
    return out
