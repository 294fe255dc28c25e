"""Operators of the serving path and the calls they are timed on: appending rotated keys and values to a paged cache held in
8 bits with a scale for each (block, kv head), attention over that cache, and attention with a sliding window and a few first
tokens that stay visible.

A sequence is written "context+new": tokens already cached, and the tokens of this step.  Cache layouts are the package's:
K [blocks, kv_heads, head / x, block, x] with x = 16 bytes of elements, V [blocks, kv_heads, head, block].
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
QMAX = {"block_int8": 127.0, "block_fp8": 448.0}
CODES = {"block_int8": torch.int8, "block_fp8": torch.float8_e4m3fn, "fp8": torch.float8_e4m3fn}


def _ragged(count, low, high, new):
    """`count` sequences with contexts spread over [low, high], `new` tokens each."""
    return " ".join("%d+%d" % (low + (high - low) * ((7 * i + 3) % count) // max(1, count - 1), new) for i in range(count))


def _append(name, lens, **more):
    return {"name": name, "op": "append", "heads": 32, "kv_heads": 8, "head": 128, "dtype": "bf16", "cache": "block_int8", "block": 16, "lens": lens,
            "rot": 128, "neox": True, **more}


def _attend(name, lens, **more):
    return {"name": name, "op": "attend", "heads": 32, "kv_heads": 8, "head": 128, "dtype": "bf16", "cache": "block_int8", "block": 16, "lens": lens,
            "window": 0, "sinks": 0, **more}


def listed():
    return [
        # one token of one conversation: nothing but latency
        _append("append_token", "777+1"),
        # a decode step of a full batch, blocks filled to different heights
        _append("append_batch", _ragged(64, 1, 4001, 1), dtype="fp16", cache="block_fp8"),
        # short prompts on 64-wide heads, interleaved rotation of half the head, larger blocks
        _append("append_partial_rotary", "0+211 37+180 5+117", head=64, rot=32, neox=False, block=32),
        # a scheduler's full step of prompt tokens, one chunk continuing inside a block
        _append("append_prompts", "0+4099 5+2048 100+1500 0+545"),
        # single conversation
        _attend("blocks_decode_one", "1000+1"),
        # decode batch of mixed ages
        _attend("blocks_decode_batch", _ragged(32, 100, 4095, 1)),
        # few very long conversations, 8 query heads to a kv head
        _attend("blocks_decode_long", "131071+1 50001+1", heads=64, cache="block_fp8", block=32),
        # a draft of four tokens checked along with the newest one
        _attend("blocks_verify", _ragged(16, 500, 3500, 5), dtype="fp16"),
        # chunked prompt with its context, a short prompt and a decode row in the same step
        _attend("blocks_chunk", "6144+2048 0+700 3001+1"),
        # decode far beyond the window; what lies between sinks and window is no longer in the cache
        _attend("window_decode", _ragged(32, 200, 16001, 1), cache="auto", window=4096, sinks=4),
        # prompts on 64-wide heads over an 8-bit cache with one scale, window shorter than most of them
        _attend("window_prompts", "0+2047 0+1100 513+300 0+17 900+1", head=64, dtype="fp16", cache="fp8", window=512, sinks=4),
        # one long prompt under a window of half its length
        _attend("window_long_prompt", "0+8192", cache="auto", window=4096, sinks=4),
    ]


def _spread(rng, low, high):
    """Over the logarithm, both ends included."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend"])
    head = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    kind = rng.choice(["decode", "decode", "verify", "prompt"])
    group = rng.choice([1, 3, 4, 4, 8])
    if kind == "prompt":
        group = min(group, 32 // kv_heads)
    case = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "head": head, "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "block": rng.choice([16, 16, 32])}
    if op == "append":
        case["cache"] = rng.choice(["block_int8", "block_fp8"])
        count = _spread(rng, 1, 64)
        if kind != "prompt":
            new = [1] * count
        else:
            count = min(count, 8)
            new = [_spread(rng, 1, 8192 // count) for _ in range(count)]
        ctx = [rng.choice([0, _spread(rng, 1, 4000)]) for _ in range(count)]
        case["rot"] = rng.choice([head, head, head // 2])
        case["neox"] = rng.random() < 0.8
    else:
        case["cache"] = rng.choice(["block_int8", "block_int8", "block_fp8", "auto", "fp8"])
        windowed = case["cache"] in ("auto", "fp8") or rng.random() < 0.3
        case["window"] = _spread(rng, 16, 8192) if windowed else 0
        case["sinks"] = rng.choice([0, 1, 4, 4, 64]) if windowed else 0
        if kind == "decode":
            count = _spread(rng, 1, 64)
            new, ctx = [1] * count, [_spread(rng, 1, 131071 // count) for _ in range(count)]
        elif kind == "verify":
            count, fresh = _spread(rng, 1, 32), rng.randint(2, 8)
            new, ctx = [fresh] * count, [_spread(rng, 1, 65536 // count) for _ in range(count)]
        else:
            count = rng.randint(1, 4)
            new = [_spread(rng, 1, 4096 // count) for _ in range(count)]
            ctx = [rng.choice([0, _spread(rng, 1, 4096 // count)]) for _ in range(count)]
    case["lens"] = " ".join("%d+%d" % p for p in zip(ctx, new))
    return case


def _lens(case):
    return [tuple(int(v) for v in p.split("+")) for p in case["lens"].split()]


def _visible(case, ctx, new):
    """(query, token) pairs that one head of a sequence computes, and tokens that at least one of its queries sees."""
    w, k = case["window"], case["sinks"]
    end = ctx + new
    if not w:
        return new * ctx + new * (new + 1) // 2, end
    pairs = 0
    for p in range(ctx, end):
        low = max(0, p + 1 - w)
        pairs += p + 1 - low + min(k, low)
    low = max(0, ctx + 1 - w)
    return pairs, end - low + min(k, low)


def work(case):
    lens, D, H, K = _lens(case), case["head"], case["heads"], case["kv_heads"]
    rows = sum(new for _, new in lens)
    size = 2 if case["cache"] == "auto" else 1
    if case["op"] == "append":
        blocks = sum((ctx + new - 1) // case["block"] - ctx // case["block"] + 1 for ctx, new in lens)
        angles = rows * (8 + 8 + case["rot"] * 2)
        return {"bytes": rows * D * (4 * H + 4 * K + 2 * K) + angles + blocks * K * 8, "flops": rows * (H + K) * case["rot"] * 3}
    seen = [_visible(case, ctx, new) for ctx, new in lens]
    scales = sum(-(-t // case["block"]) for _, t in seen) * K * 8 if case["cache"] in QMAX else 0
    return {"bytes": rows * H * D * 4 + sum(t for _, t in seen) * K * D * 2 * size + scales, "flops": 4 * D * H * sum(p for p, _ in seen)}


def _fill(codes, scales, x, form):
    """Codes of x [blocks, kv_heads, ...] under a scale for each block and kv head, as a cache that was filled at once holds them."""
    top = x.flatten(2).abs().amax(2) / QMAX[form]
    scales.copy_(top)
    y = x / top[(...,) + (None,) * (x.dim() - 2)]
    codes.view(CODES[form]).copy_(torch.round(y) if form == "block_int8" else y)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    lens, D, H, K, bs, form = _lens(case), case["head"], case["heads"], case["kv_heads"], case["block"], case["cache"]
    dtype = DTYPES[case["dtype"]]
    rows, count = sum(n for _, n in lens), len(lens)
    ctx, new = (torch.tensor(v, dtype=torch.int64) for v in zip(*lens))
    total = ctx + new
    pages = -(-total // bs)
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    # logical pages that some query of the step sees; the others have gone back to the allocator (page 0 stands in their place)
    at = torch.arange(int(pages.max()))
    held = at[None] < pages[:, None]
    if window:
        low = (ctx + 1 - window).clamp(min=0)
        held &= (at[None] * bs < sinks) | ((at[None] + 1) * bs > low[:, None])
    blocks = int(held.sum()) + 3
    order = torch.randperm(blocks - 1, generator=torch.Generator().manual_seed(seed)) + 1
    tables = torch.zeros(held.shape, dtype=torch.int32)
    tables[held] = order[:int(held.sum())].to(torch.int32)
    # keys have a few loud channels, values do not; a fused projection's row holds q | k | v
    loud = torch.exp(torch.randn(K, D, generator=g, device=dev) * 0.5)
    qkv = torch.randn(rows, (H + 2 * K) * D, generator=g, device=dev)
    qkv[:, H * D:(H + K) * D] *= loud.flatten()
    qkv = qkv.to(dtype)
    x = 8 if form == "auto" else 16
    keys = torch.randn(blocks, K, D // x, bs, x, generator=g, device=dev) * loud.view(1, K, D // x, 1, x)
    values = torch.randn(blocks, K, D, bs, generator=g, device=dev) * torch.exp(torch.randn(blocks, K, 1, 1, generator=g, device=dev) * 0.3)
    s = {"case": case, "dtype": dtype, "qkv": qkv, "rows": rows, "scale": D ** -0.5, "max_query": int(new.max()), "max_len": int(total.max()),
         "tables": tables.to(dev), "seq_lens": total.to(torch.int32).to(dev),
         "starts": torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(torch.int32).to(dev)}
    if form == "auto":
        s["kc"], s["vc"] = keys.to(dtype), values.to(dtype)
        s["ks"] = s["vs"] = torch.ones((), device=dev)
    elif form == "fp8":
        s["ks"], s["vs"] = torch.full((), 1 / 32.0, device=dev), torch.full((), 1 / 64.0, device=dev)
        s["kc"] = (keys / s["ks"]).clamp(-448, 448).to(CODES[form]).view(torch.uint8)
        s["vc"] = (values / s["vs"]).clamp(-448, 448).to(CODES[form]).view(torch.uint8)
    else:
        s["kc"], s["vc"] = torch.empty(keys.shape, dtype=torch.uint8, device=dev), torch.empty(values.shape, dtype=torch.uint8, device=dev)
        s["ks"], s["vs"] = torch.empty(blocks, K, device=dev), torch.empty(blocks, K, device=dev)
        _fill(s["kc"], s["ks"], keys, form)
        _fill(s["vc"], s["vs"], values, form)
    if case["op"] == "append":
        pos = torch.cat([torch.arange(c, c + n) for c, n in lens])
        seq = torch.repeat_interleave(torch.arange(count), new)
        s["positions"] = pos.to(dev)
        s["slots"] = (tables[seq, pos // bs].to(torch.int64) * bs + pos % bs).to(dev)
        inv = 500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])
        angle = torch.arange(int(total.max()), dtype=torch.float64)[:, None] * inv
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).to(dtype).to(dev)
    return s


def _ops():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-fork_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from mi355q import ops
    return ops


def _split(s):
    c, D = s["case"], s["case"]["head"]
    H, K = c["heads"] * D, c["kv_heads"] * D
    return s["qkv"][:, :H], s["qkv"][:, H:H + K], s["qkv"][:, H + K:]


def _held(s):
    """The cache as numbers: integers or e4m3 values, to be multiplied by the scales beside them."""
    t = CODES[s["case"]["cache"]]
    return s["kc"].view(t), s["vc"].view(t)


def run(s):
    c = s["case"]
    q, k, v = _split(s)
    if c["op"] == "append":
        if own:
            rotated = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            _ops().rope_and_cache_blocks(s["positions"], q, k, v, c["head"], s["cos_sin"], c["neox"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"],
                                         c["cache"], query_out=rotated)
        else:
            rotated = _append_plain(s, q, k, v)
        keys, values = _held(s)
        return {"query": rotated, "keys": keys, "values": values, "key_scales": s["ks"], "value_scales": s["vs"]}
    q = q.unflatten(1, (c["heads"], c["head"]))
    if own:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _ops().paged_window_attention(out, q, s["kc"], s["vc"], c["kv_heads"], s["scale"], s["tables"], s["seq_lens"], s["starts"], s["max_query"],
                                      s["max_len"], c["cache"], s["ks"], s["vs"], sliding_window=c["window"], sink_tokens=c["sinks"])
        return out
    return _attend_plain(s, q)


# --- the plain forms -----------------------------------------------------------------------------------------------------


def _rotate(x, s):
    """x [rows, heads, head]: the first `rot` elements of a head turned by the row's angles, in 32 bits, rounded once."""
    c = s["case"]
    row = s["cos_sin"][s["positions"]].float()[:, None]
    e = c["rot"] // 2
    cos, sin = row[..., :e], row[..., e:]
    y = x.float()
    a, b = (y[..., :e], y[..., e:2 * e]) if c["neox"] else (y[..., 0:2 * e:2], y[..., 1:2 * e:2])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([a, b], -1) if c["neox"] else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, y[..., 2 * e:]], -1).to(x.dtype)


def _append_one(codes, scales, x, block, offset, at, slot_axis, form):
    """x [rows, kv_heads, head] into codes [blocks, kv_heads, ...] whose axis `slot_axis` runs over a block's tokens."""
    blocks, bs = scales.shape[0], codes.shape[slot_axis]
    x = x.float()
    top = torch.zeros_like(scales).index_reduce_(0, block, x.abs().amax(2) / QMAX[form], "amax")
    first = torch.full((blocks,), bs, device=x.device).index_reduce_(0, block, offset, "amin")
    old = torch.where((first > 0)[:, None], scales, 0.0)
    touched = (first < bs)[:, None]
    new = torch.where(touched, torch.maximum(old, top), scales)
    grown = touched & (new > old)
    shape = [1] * codes.dim()
    shape[slot_axis] = bs
    wide = (blocks, -1) + (1,) * (codes.dim() - 2)
    kept = grown.view(wide) & (torch.arange(bs, device=x.device).view(shape) < first.view((blocks,) + (1,) * (codes.dim() - 1)))
    held = codes.view(CODES[form])
    again = held.float() * torch.where(grown, old / new, 1.0).view(wide)
    held.copy_(torch.where(kept, torch.round(again) if form == "block_int8" else again, held.float()))
    y = x / new[block][..., None]
    y = torch.where(new[block][..., None] > 0, y, 0.0)
    codes[at] = (torch.round(y) if form == "block_int8" else y).to(held.dtype).view(torch.uint8)
    scales.copy_(new)


def _append_plain(s, q, k, v):
    c = s["case"]
    D, bs, K = c["head"], c["block"], c["kv_heads"]
    block, offset = s["slots"] // bs, s["slots"] % bs
    k = _rotate(k.unflatten(1, (K, D)), s)
    v = v.unflatten(1, (K, D))
    h, d = torch.arange(K, device=k.device)[None, :, None], torch.arange(D, device=k.device)[None, None]
    b, o = block[:, None, None], offset[:, None, None]
    _append_one(s["kc"], s["ks"], k, block, offset, (b, h, d // 16, o, d % 16), 3, c["cache"])
    _append_one(s["vc"], s["vs"], v, block, offset, (b, h, d, o), 3, c["cache"])
    return _rotate(q.unflatten(1, (c["heads"], D)), s).flatten(1)


def _attend_plain(s, q):
    c = s["case"]
    D, H, K, bs, form = c["head"], c["heads"], c["kv_heads"], c["block"], c["cache"]
    tables = s["tables"].long()
    S, L = tables.shape[0], tables.shape[1] * bs
    keys, values = s["kc"][tables], s["vc"][tables]                       # [S, pages, K, D / x, bs, x], [S, pages, K, D, bs]
    if form != "auto":
        keys, values = keys.view(CODES[form]), values.view(CODES[form])
    keys, values = keys.float(), values.float()
    if form in QMAX:
        keys, values = keys * s["ks"][tables][..., None, None, None], values * s["vs"][tables][..., None, None]
    elif form == "fp8":
        keys, values = keys * s["ks"], values * s["vs"]
    keys = keys.permute(0, 2, 1, 4, 3, 5).reshape(S, K, L, D)
    values = values.permute(0, 2, 1, 4, 3).reshape(S, K, L, D)
    # rows of the batch laid out as [sequence, row of the longest query]
    starts, n = s["starts"][:-1].long(), s["max_query"]
    lens = s["seq_lens"].long()
    fresh = s["starts"][1:].long() - starts
    row = torch.arange(n, device=q.device)[None]
    index = (starts[:, None] + row).clamp(max=s["rows"] - 1)
    wide = q[index].float().view(S, n, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(S, K, H // K * n, D)
    position = (lens - fresh)[:, None] + row                              # [S, n]
    t = torch.arange(L, device=q.device)[None, None]
    p = position[..., None]
    seen = (t <= p) & (t < lens[:, None, None])
    if c["window"]:
        seen &= (t > p - c["window"]) | (t < c["sinks"])
    logits = (wide @ keys.transpose(2, 3).contiguous() * s["scale"]).view(S, K, H // K, n, L)
    logits = torch.where(seen[:, None, None], logits, -math.inf)
    weight = torch.exp(logits - logits.amax(-1, keepdim=True))
    out = (weight / weight.sum(-1, keepdim=True)).view(S, K, H // K * n, L) @ values
    out = out.view(S, K, H // K, n, D).permute(0, 3, 1, 2, 4).reshape(S, n, H, D)
    return out[row.expand(S, n) < fresh[:, None]].to(q.dtype)


# --- 64 bits ---------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    lens, D, H, K, bs, form = _lens(case), case["head"], case["heads"], case["kv_heads"], case["block"], case["cache"]
    q, k, v = (t.double() for t in _split(s))
    if case["op"] == "append":
        e, dev = case["rot"] // 2, q.device
        first, second = (torch.arange(e), torch.arange(e) + e) if case["neox"] else (2 * torch.arange(e), 2 * torch.arange(e) + 1)
        angles = s["cos_sin"].double()[s["positions"]]
        turn = torch.complex(angles[:, :e], angles[:, e:])[:, None]

        def turned(x):
            x = x.reshape(x.shape[0], -1, D).clone()
            z = torch.complex(x[..., first.to(dev)], x[..., second.to(dev)]) * turn
            x[..., first.to(dev)], x[..., second.to(dev)] = z.real, z.imag
            return x

        def scales(old, x):
            """The largest magnitude of each touched block and head, and what an unfinished block had before."""
            new, at = old.double(), 0
            for i, (ctx, n) in enumerate(lens):
                for page in range(ctx // bs, (ctx + n - 1) // bs + 1):
                    a, b = max(ctx, page * bs), min(ctx + n, (page + 1) * bs)
                    top = x[at + a - ctx:at + b - ctx].abs().amax((0, 2)) / QMAX[form]
                    cell = int(tables[i][page])
                    new[cell] = torch.maximum(new[cell], top) if a > page * bs else top
                at += n
            return new

        tables = s["tables"].tolist()
        key = turned(k).to(s["dtype"]).double()      # the cache takes the rotated key as the model's type holds it
        return {"query": turned(q).flatten(1), "keys": None, "values": None, "key_scales": scales(s["ks"], key), "value_scales": scales(s["vs"], v.view(-1, K, D))}
    out, at = torch.empty(s["rows"], H, D, dtype=torch.float64, device=q.device), 0
    q = q.view(-1, K, H // K, D)
    number = torch.Tensor.double if form == "auto" else lambda codes: codes.contiguous().view(CODES[form]).double()
    for i, (ctx, n) in enumerate(lens):
        end, w, sinks = ctx + n, case["window"], case["sinks"]
        low = max(0, ctx + 1 - w) if w else 0
        token = torch.cat([torch.arange(min(sinks, low)), torch.arange(low, end)]).to(q.device)
        page, place = s["tables"][i].long()[token // bs], token % bs
        position = torch.arange(ctx, end, device=q.device)[:, None]
        hidden = token[None] > position
        if w:
            hidden |= (token[None] + w <= position) & (token[None] >= sinks)
        for h in range(K):
            kk = number(s["kc"][page, h, :, place]).flatten(1)
            vv = number(s["vc"][page, h, :, place])
            if form in QMAX:
                kk, vv = kk * s["ks"][page, h].double()[:, None], vv * s["vs"][page, h].double()[:, None]
            else:
                kk, vv = kk * s["ks"].double(), vv * s["vs"].double()
            for j in range(H // K):
                z = (q[at:at + n, h, j] @ kk.T * s["scale"]).masked_fill(hidden, -math.inf)
                out[at:at + n, h * (H // K) + j] = torch.softmax(z, 1) @ vv
        at += n
    return out
