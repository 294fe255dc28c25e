"""8-bit KV cache with a scale for each (block, kv head), and attention with a sliding window and visible first tokens:
ops.rope_and_cache_blocks, ops.reshape_and_cache_blocks and ops.paged_window_attention against plain restatements.

The append is compared bit for bit: the restatement does the documented fp32 operations one at a time.  Attention is compared
with a 64-bit evaluation of the formula on the very codes the kernel reads; the tolerance is the sum of what the kernel's
roundings can do (see `attention_bound`)."""
import numpy as np
import pytest
import torch

from mi355q import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
QMAX = {"block_int8": 127.0, "block_fp8": 448.0}
CODE = {"block_int8": torch.int8, "block_fp8": torch.float8_e4m3fn, "fp8": torch.float8_e4m3fn}
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------
def cpu(t):
    return t.detach().cpu()


def encode(x, form):
    """fp32 -> the values the codes stand for (before the scale)."""
    return torch.round(x) if form == "block_int8" else x.clamp(-448, 448).to(torch.float8_e4m3fn).float()


def rotate_ref(x, positions, cos_sin, rot, neox, dtype):
    """x [T, heads, D]; fp32 with one rounding per operation, rounded to dtype at the end."""
    if not rot:
        return x.clone()
    y = x.float().clone()
    row = cos_sin.float()[positions.clamp(0, cos_sin.shape[0] - 1)][:, None]
    e = rot // 2
    c, s = row[..., :e], row[..., e:]
    i, j = (slice(0, e), slice(e, rot)) if neox else (slice(0, rot, 2), slice(1, rot, 2))
    a, b = x.float()[..., i], x.float()[..., j]
    y[..., i] = a * c - b * s
    y[..., j] = b * c + a * s
    return y.to(dtype)


def append_ref(codes, scales, x, slots, bs, form):
    """codes: fp32 values [blocks, KVH, bs, D] (changed in place); scales [blocks, KVH]; x [T, KVH, D] in the model's type.
    One run of tokens in one block after the other (at most 64 positions each), as documented."""
    n = codes.shape[0] * bs
    t, T = 0, len(slots)
    while t < T:
        if not 0 <= slots[t] < n:
            t += 1
            continue
        b, end, run = slots[t] // bs, t, []
        while end < min(T, t + 64):
            if 0 <= slots[end] < n:
                if slots[end] // bs != b:
                    break
                run.append(end)
            end += 1
        stands = {slots[i] % bs: i for i in run}       # the last of several for one slot
        first = min(stands)
        take = x[sorted(stands.values())].float()
        top = take.abs().amax((0, 2)) * (torch.tensor(1.0) / torch.tensor(QMAX[form]))
        top = torch.where(torch.isfinite(take).all(2).all(0), top, torch.nan)
        for h in range(x.shape[1]):
            old = scales[b, h].item() if first > 0 else 0.0
            new = top[h].item() if top[h] > old or torch.isnan(top[h]) else old
            if new > old:
                ratio = torch.tensor(old) / torch.tensor(new)
                codes[b, h, :first] = encode(codes[b, h, :first] * ratio, form)
            for o, i in stands.items():
                codes[b, h, o] = encode(x[i, h].float() / torch.tensor(new), form) if new > 0 else 0.0
            scales[b, h] = new
        t = end


class Cache:
    """A paged 8-bit cache with stale contents, and the restatement's copy of it."""

    def __init__(self, blocks, kvh, D, bs, form, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.form, self.bs, self.D = form, bs, D
        stale = torch.randint(-127, 128, (2, blocks, kvh, bs, D), generator=g).float()
        stale = encode(stale, form)
        self.k_ref, self.v_ref = stale[0].clone(), stale[1].clone()
        self.ks_ref, self.vs_ref = (torch.rand(blocks, kvh, generator=g) * 0.02 for _ in range(2))
        self.kc = self.pack_k(self.k_ref).to(DEV)
        self.vc = self.pack_v(self.v_ref).to(DEV)
        self.ks, self.vs = self.ks_ref.to(DEV), self.vs_ref.to(DEV)

    def pack_k(self, x):
        n, h, bs, D = x.shape
        return x.view(n, h, bs, D // 16, 16).transpose(2, 3).contiguous().to(CODE[self.form]).view(torch.uint8)

    def pack_v(self, x):
        return x.transpose(2, 3).contiguous().to(CODE[self.form]).view(torch.uint8)

    def append(self, k, v, slots):
        append_ref(self.k_ref, self.ks_ref, k, slots, self.bs, self.form)
        append_ref(self.v_ref, self.vs_ref, v, slots, self.bs, self.form)

    def check(self):
        """Codes compared as values (e4m3 has two zeros), scales bit for bit."""
        for got, want in ((self.kc, self.pack_k(self.k_ref)), (self.vc, self.pack_v(self.v_ref))):
            a, b = cpu(got).view(CODE[self.form]).float(), want.view(CODE[self.form]).float()
            assert torch.equal(a, b), f"{int((a != b).sum())} of {a.numel()} codes differ"
        for got, want in ((self.ks, self.ks_ref), (self.vs, self.vs_ref)):
            assert torch.equal(torch.nan_to_num(cpu(got), nan=-1.0), torch.nan_to_num(want, nan=-1.0))


def qkv_rows(T, H, KVH, D, dtype, seed, loud=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, (H + 2 * KVH) * D, generator=g)
    x[:, H * D:] *= torch.exp(torch.randn(T, 1, generator=g) * loud)     # tokens of different size: scales grow as they come
    return x.to(dtype)


def angles(rot, rows, dtype):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).to(dtype)


def run_append(c, qkv, H, KVH, D, positions, cos_sin, rot, neox, slots, in_place=False):
    x = qkv.to(DEV)
    q, k, v = x[:, :H * D], x[:, H * D:(H + KVH) * D], x[:, (H + KVH) * D:]
    out = q if in_place else torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    ops.rope_and_cache_blocks(positions.to(DEV), q, k, v, D, cos_sin.to(DEV), neox, c.kc, c.vc, c.ks, c.vs,
                              torch.tensor(slots, device=DEV), c.form, query_out=None if in_place else out)
    torch.cuda.synchronize()
    T = qkv.shape[0]
    q, k, v = (t.unflatten(1, (-1, D)) for t in (qkv[:, :H * D], qkv[:, H * D:(H + KVH) * D], qkv[:, (H + KVH) * D:]))
    want = rotate_ref(q, positions, cos_sin, rot, neox, qkv.dtype).flatten(1)
    assert torch.equal(cpu(out), want)
    assert torch.equal(cpu(x[:, H * D:]).contiguous().view(torch.int16), qkv[:, H * D:].contiguous().view(torch.int16))   # key and value as they were
    c.append(rotate_ref(k, positions, cos_sin, rot, neox, qkv.dtype), v, slots)
    c.check()


@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
@pytest.mark.parametrize("H,KVH,D,bs,rot,neox,dtype,table", [
    (8, 2, 128, 16, 128, True, torch.bfloat16, torch.bfloat16),
    (4, 4, 64, 32, 64, True, torch.float16, torch.float32),
    (6, 2, 64, 16, 32, False, torch.bfloat16, torch.bfloat16),      # half the head, interleaved pairs
    (3, 1, 128, 64, 64, True, torch.float16, torch.float16),
    (5, 1, 128, 48, 36, True, torch.bfloat16, torch.float32),       # a rotation that no 16-element chunk holds
    (16, 1, 64, 16, 6, False, torch.float16, torch.bfloat16),
])
def test_append_prompts_then_tokens(form, H, KVH, D, bs, rot, neox, dtype, table):
    """Three sequences: prompts that end inside a block, a second chunk, then single tokens: every step bit for bit."""
    c = Cache(24, KVH, D, bs, form)
    cs = angles(rot, 4 * bs + 64, table)
    pages = torch.randperm(24, generator=torch.Generator().manual_seed(5)).tolist()
    filled = [0, 0, 0]
    own = [pages[:8], pages[8:16], pages[16:24]]
    for step, new in enumerate([(bs + 5, 1, 2 * bs), (3, 2 * bs - 1, 1), (1, 1, 1), (1, 0, 1), (bs - 2, 1, 1)]):
        pos, slots = [], []
        for s, n in enumerate(new):
            for t in range(filled[s], filled[s] + n):
                pos.append(t)
                slots.append(own[s][t // bs] * bs + t % bs)
            filled[s] += n
        pos += [0, 0]                                                     # graph padding behind the batch
        slots += [-1, -1]
        qkv = qkv_rows(len(pos), H, KVH, D, dtype, seed=step)
        run_append(c, qkv, H, KVH, D, torch.tensor(pos), cs, rot, neox, slots, in_place=step % 2 == 1)


@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
def test_append_many_tokens(form):
    """The many-token variant of the launch (over 512 tokens), ragged, slots skipped inside the batch."""
    H, KVH, D, bs = 4, 2, 128, 16
    c = Cache(80, KVH, D, bs, form)
    cs = angles(D, 1300, torch.bfloat16)
    pages = torch.randperm(80, generator=torch.Generator().manual_seed(1)).tolist()
    pos = list(range(7, 607)) + list(range(0, 431))
    slots = [pages[t // bs] * bs + t % bs for t in range(7, 607)] + [pages[40 + t // bs] * bs + t % bs for t in range(431)]
    for t in list(range(590, 600)) + [100 + 9, 900, 902]:                 # the second sequence's block 18 has gaps
        slots[t] = -1
    qkv = qkv_rows(len(pos), H, KVH, D, torch.bfloat16, 3)
    run_append(c, qkv, H, KVH, D, torch.tensor(pos), cs, D, True, slots)


@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
def test_append_odd_slots(form):
    """Slots outside the cache, repeated slots (the last stays), slots in falling order, zeros, values that are not finite."""
    KVH, D, bs = 2, 64, 16
    c = Cache(6, KVH, D, bs, form)
    cs = angles(D, 64, torch.bfloat16)
    slots = [-5, 6 * bs, 1 << 40, 17, 17, 17, 35, 34, 33, 40, 38, 3, -1, 50, 48, 50, 64]
    qkv = qkv_rows(len(slots), 2, KVH, D, torch.bfloat16, 11)
    qkv[11] = 0.0
    qkv[16, 2 * D + 3] = float("inf")                                     # key of kv head 0
    qkv[16, 2 * D + KVH * D + D + 1] = float("nan")                       # value of kv head 1
    pos = torch.arange(len(slots))
    pos[1], pos[2] = -3, 1 << 40                                          # outside the table: clamped
    run_append(c, qkv, 2, KVH, D, pos, cs, D, True, slots)
    assert torch.isnan(c.ks_ref[4]).tolist() == [True, False] and torch.isnan(c.vs_ref[4]).tolist() == [False, True]
    # a poisoned block stays so until it starts over
    run_append(c, qkv_rows(1, 2, KVH, D, torch.bfloat16, 12), 2, KVH, D, torch.tensor([1]), cs, D, True, [65])
    assert torch.isnan(c.ks_ref[4, 0])
    run_append(c, qkv_rows(1, 2, KVH, D, torch.bfloat16, 13), 2, KVH, D, torch.tensor([0]), cs, D, True, [64])
    assert torch.isfinite(c.ks_ref[4]).all() and torch.isfinite(c.vs_ref[4]).all()


def test_append_behind_long_gaps():
    """Runs that go on behind more than 64, and more than 512, tokens without a slot."""
    KVH, D, bs = 1, 64, 16
    c = Cache(8, KVH, D, bs, "block_int8")
    slots = [-1] * 700 + [19, 20] + [-1] * 90 + [21] + [-1] * 600 + [22, 23, 48] + [-1] * 20 + [49, 70] + [-1] * 70
    qkv = qkv_rows(len(slots), 1, KVH, D, torch.bfloat16, 6)
    run_append(c, qkv, 1, KVH, D, torch.arange(len(slots)), angles(D, len(slots), torch.bfloat16), D, True, slots)


def test_append_one_slot_named_many_times():
    """More neighbours in one block than a stretch of 64."""
    KVH, D, bs = 1, 128, 16
    c = Cache(4, KVH, D, bs, "block_int8")
    slots = [16 + (i * 7) % 16 for i in range(150)]
    qkv = qkv_rows(150, 1, KVH, D, torch.float16, 2)
    run_append(c, qkv, 1, KVH, D, torch.arange(150), angles(D, 150, torch.float16), D, True, slots)


@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
@pytest.mark.parametrize("T", [400, 900])
def test_append_of_a_block_stretched_over_many_positions(form, T):
    """What the header says of a block whose tokens take more than 64 positions: the call does what a call for each stretch does --
    on the way up, back to offset 0, back to an offset between, with slots named again; other blocks beside it."""
    H, KVH, D, bs = 2, 2, 64, 16
    slots = [-1] * T
    for at, slot in [(0, 21), (1, 22), (63, 23), (64, 24), (90, 16), (91, 30), (170, 18), (171, 17), (233, 18), (234, 31), (235, 40), (236, 41),
                     (310, 32), (330, 50), (331, 51), (T - 1, 49)]:
        slots[at] = slot
    one, many = Cache(5, KVH, D, bs, form, seed=3), Cache(5, KVH, D, bs, form, seed=3)
    qkv, pos, cs = qkv_rows(T, H, KVH, D, torch.bfloat16, 15), torch.arange(T), angles(D, T, torch.bfloat16)
    run_append(one, qkv, H, KVH, D, pos, cs, D, True, slots)
    calls, begin, block = [], None, None
    for t, slot in enumerate(slots):
        if slot < 0:
            continue
        if slot // bs != block or t >= begin + 64:
            calls.append([-1] * T)
            begin, block = t, slot // bs
        calls[-1][t] = slot
    assert len(calls) == 8
    for call in calls:
        run_append(many, qkv, H, KVH, D, pos, cs, D, True, call)
    for name in ("kc", "vc", "ks", "vs"):
        assert torch.equal(getattr(one, name), getattr(many, name)), name


def test_append_unaligned_rows_and_strided_scales():
    H, KVH, D, bs = 3, 2, 64, 16
    c = Cache(5, KVH, D, bs, "block_int8")
    qkv = qkv_rows(20, H, KVH, D, torch.bfloat16, 4)
    wide = torch.zeros(20, (H + 2 * KVH) * D + 3, dtype=torch.bfloat16, device=DEV)
    wide[:, 1:-2] = qkv.to(DEV)
    q, k, v = wide[:, 1:1 + H * D], wide[:, 1 + H * D:1 + (H + KVH) * D], wide[:, 1 + (H + KVH) * D:-2]
    ks, vs = torch.zeros(KVH, 5, device=DEV).t(), torch.zeros(KVH, 5, device=DEV).t()
    ks.copy_(c.ks)
    vs.copy_(c.vs)
    c.ks, c.vs = ks, vs
    cs, pos, slots = angles(D, 64, torch.bfloat16), torch.arange(20), list(range(30, 50))
    out = torch.empty(20, H * D, dtype=torch.bfloat16, device=DEV)
    ops.rope_and_cache_blocks(pos.to(DEV), q, k, v, D, cs.to(DEV), True, c.kc, c.vc, c.ks, c.vs, torch.tensor(slots, device=DEV),
                              c.form, query_out=out)
    x = [t.unflatten(1, (-1, D)) for t in (qkv[:, :H * D], qkv[:, H * D:(H + KVH) * D], qkv[:, (H + KVH) * D:])]
    assert torch.equal(cpu(out), rotate_ref(x[0], pos, cs, D, True, torch.bfloat16).flatten(1))
    c.append(rotate_ref(x[1], pos, cs, D, True, torch.bfloat16), x[2], slots)
    c.check()


@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
def test_reshape_and_cache_blocks(form):
    """The append alone, with more key rows than slots (graph padding); and how far the held values may be off: half a step
    for each time a value was rounded (once when written, once each time its block's scale grew)."""
    KVH, D, bs = 3, 128, 32
    c = Cache(4, KVH, D, bs, form)
    written, grew = torch.zeros(bs, KVH, D), torch.zeros(bs, KVH)
    scale = torch.zeros(KVH)
    for t in range(bs):
        x = qkv_rows(2, 0, KVH, D, torch.bfloat16, 40 + t)
        k, v = x[:, :KVH * D].view(2, KVH, D), x[:, KVH * D:].view(2, KVH, D)
        ops.reshape_and_cache_blocks(k.to(DEV), v.to(DEV), c.kc, c.vc, c.ks, c.vs, torch.tensor([64 + t], device=DEV), form)
        c.append(k[:1], v[:1], [64 + t])
        c.check()
        written[t] = v[0].float()
        grew[:t] += (c.vs_ref[2] > scale).float()
        scale = c.vs_ref[2].clone()
    held = c.v_ref[2].transpose(0, 1) * scale[None, :, None]            # [bs, KVH, D]
    off = (held - written).abs()
    if form == "block_int8":   # half a code each time, at a scale no larger than the last
        bound = (grew + 1)[..., None] * 0.5 * scale[None, :, None] * (1 + 2 ** -20)
    else:                      # 2^-4 of the value each time, or half the smallest e4m3 step
        n = (grew + 1)[..., None]
        bound = n * (written.abs() * 2 ** -4 * (1 + 2 ** -4) ** n + 2 ** -10 * scale[None, :, None])
    assert (off <= bound).all()


def test_append_captured_in_a_graph():
    H, KVH, D, bs = 8, 2, 128, 16
    c = Cache(8, KVH, D, bs, "block_int8")
    cs = angles(D, 128, torch.bfloat16)
    x = torch.zeros(2, (H + 2 * KVH) * D, dtype=torch.bfloat16, device=DEV)
    pos, slots = torch.zeros(2, dtype=torch.int64, device=DEV), torch.full((2,), -1, dtype=torch.int64, device=DEV)
    out, table = torch.empty(2, H * D, dtype=torch.bfloat16, device=DEV), cs.to(DEV)

    def step():
        ops.rope_and_cache_blocks(pos, x[:, :H * D], x[:, H * D:(H + KVH) * D], x[:, (H + KVH) * D:], D, table, True, c.kc, c.vc, c.ks, c.vs,
                                  slots, c.form, query_out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for t in range(20):
        rows = qkv_rows(2, H, KVH, D, torch.bfloat16, 60 + t)
        p, s = torch.tensor([t, t]), [16 + t, -1 if t % 3 else 80 + t]
        x.copy_(rows)
        pos.copy_(p)
        slots.copy_(torch.tensor(s))
        g.replay()
        torch.cuda.synchronize()
        q, k, v = (r.unflatten(1, (-1, D)) for r in (rows[:, :H * D], rows[:, H * D:(H + KVH) * D], rows[:, (H + KVH) * D:]))
        assert torch.equal(cpu(out), rotate_ref(q, p, cs, D, True, torch.bfloat16).flatten(1))
        c.append(rotate_ref(k, p, cs, D, True, torch.bfloat16), v, s)
        c.check()


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
class Batch:
    """Sequences "context + new" over a paged cache; everything a call of paged_window_attention takes, and the formula in
    64 bits on the same codes."""

    def __init__(self, lens, H, KVH, D, bs, form, dtype, window=0, sinks=0, seed=0, loud=1.0, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.H, self.KVH, self.D, self.bs, self.form, self.dtype, self.window, self.sinks = lens, H, KVH, D, bs, form, dtype, window, sinks
        total = [c + n for c, n in lens]
        pages = [max(1, -(-t // bs)) for t in total]
        self.blocks = sum(pages) + spare
        order = torch.randperm(self.blocks, generator=g)
        self.tables = torch.full((len(lens), max(pages) + 1), -7, dtype=torch.int32)       # never a page of anybody's
        at = 0
        for s, n in enumerate(pages):
            self.tables[s, :n] = order[at:at + n].to(torch.int32)
            at += n
        self.rows = sum(n for _, n in lens)
        self.qkv = torch.randn(self.rows + 1, H * D, generator=g).to(dtype)                 # one row behind the last sequence
        self.q = self.qkv.view(-1, H, D)
        shape = (self.blocks, KVH, bs, D)
        k = torch.randn(shape, generator=g) * torch.exp(torch.randn(1, KVH, 1, D, generator=g) * 0.5)
        v = torch.randn(shape, generator=g) * torch.exp(torch.randn(self.blocks, KVH, 1, 1, generator=g) * loud)
        x = 8 if form == "auto" else 16
        if form == "auto":
            self.k, self.v = k.to(dtype).double(), v.to(dtype).double()
            kk, vv = k.to(dtype), v.to(dtype)
            self.ks = self.vs = None
        else:
            if form == "fp8":
                self.ks, self.vs = torch.tensor(0.03), torch.tensor(0.02)
                sk, sv = self.ks, self.vs
            else:
                self.ks, self.vs = k.abs().amax((2, 3)) / QMAX[form], v.abs().amax((2, 3)) / QMAX[form]
                sk, sv = self.ks[..., None, None], self.vs[..., None, None]
            kk, vv = ((torch.round(t) if form == "block_int8" else t.clamp(-448, 448)).to(CODE[form]) for t in (k / sk, v / sv))
            self.k, self.v = kk.double() * sk.double(), vv.double() * sv.double()
        byte = kk if form == "auto" else kk.view(torch.uint8)
        self.kc = byte.view(self.blocks, KVH, bs, D // x, x).transpose(2, 3).contiguous().to(DEV)
        byte = vv if form == "auto" else vv.view(torch.uint8)
        self.vc = byte.transpose(2, 3).contiguous().to(DEV)
        self.scale = D ** -0.5
        self.dev = {n: (None if t is None else t.to(DEV)) for n, t in dict(q=self.q, tables=self.tables, ks=self.ks, vs=self.vs).items()}
        self.seq_lens = torch.tensor(total, dtype=torch.int32, device=DEV)
        self.starts = torch.tensor([0] + np.cumsum([n for _, n in lens]).tolist(), dtype=torch.int32, device=DEV)
        self.max_query, self.max_len = max(1, max(n for _, n in lens)), max(1, max(total))

    def run(self, **more):
        out = torch.full(self.q.shape, 3.0, dtype=self.dtype, device=DEV)
        d = self.dev
        a = dict(out=out, query=d["q"], key_cache=self.kc, value_cache=self.vc, num_kv_heads=self.KVH, scale=self.scale, block_tables=d["tables"],
                 seq_lens=self.seq_lens, query_start_loc=self.starts, max_query_len=self.max_query, max_seq_len=self.max_len,
                 kv_cache_dtype=self.form, k_scale=d["ks"], v_scale=d["vs"], sliding_window=self.window, sink_tokens=self.sinks)
        a.update(more)
        ops.paged_window_attention(**a)
        return a["out"]

    def visible(self, s, j):
        c, n = self.lens[s]
        p = c + j
        t = torch.arange(c + n)
        keep = t <= p
        if self.window:
            keep &= (t > p - self.window) | (t < self.sinks)
        return t[keep]

    def reference(self):
        """(out, bound) in 64 bits, [rows, H, D]."""
        out, bound = torch.zeros(self.rows, self.H, self.D, dtype=torch.float64), torch.zeros(self.rows, self.H, self.D, dtype=torch.float64)
        G, row = self.H // self.KVH, 0
        for s, (c, n) in enumerate(self.lens):
            table = self.tables[s].long()
            for j in range(n):
                t = self.visible(s, j)
                if len(t):
                    page, off = table[t // self.bs], t % self.bs
                    inside = (page >= 0) & (page < self.blocks)
                    page, off = page[inside], off[inside]
                    k, v = self.k[page, :, off].transpose(0, 1), self.v[page, :, off].transpose(0, 1)         # [KVH, L, D]
                    q = self.q[row].double().view(self.KVH, G, self.D)
                    z = q @ k.transpose(1, 2) * self.scale
                    w = torch.softmax(z, 2)
                    o = w @ v
                    slip = (q.abs() @ k.abs().transpose(1, 2) * self.scale).amax(2, keepdim=True)
                    out[row] = o.reshape(self.H, self.D)
                    bound[row] = self.attention_bound(o, w @ v.abs(), v.abs().amax(1, keepdim=True), slip, len(t)).reshape(self.H, self.D)
                row += 1
        return out, bound

    def attention_bound(self, o, mass, vmax, slip, n):
        """What the roundings add up to.  mass = sum w |v|:
          probabilities rounded to fp16 (8-bit caches) or the model's type, in the products with V and in their sum: one half step
            of each weight in numerator and denominator, 2 u_p * mass
          logits: products summed in fp32 over the head, at most (D + 8) 2^-24 of sum |q k| each, and the base-2 exponent's own
            error of about 2^-22; both as relative errors of the weights, in numerator and denominator: 2 * (...) * mass
          the sums over n tokens in fp32, and the scale factors: (n / 16 + 32) 2^-24 * mass (products are added 16 and more at a time)
          fp16 probabilities below its normal range: n * 2^-32 of the largest |v| (times 4 for the headroom of the scales)
          the result rounded to the model's type: u_out * (|o| + the above)"""
        u_p = 2 * (UNIT[self.dtype] if self.form == "auto" else 2.0 ** -11)
        weights = 2 * ((self.D + 8) * 2.0 ** -24 * slip * 1.5 + 2.0 ** -21)
        e = (u_p + weights + (n / 16 + 32) * 2.0 ** -24) * mass + n * 2.0 ** -30 * vmax
        return e + UNIT[self.dtype] * (o.abs() + e) + 2.0 ** -25

    def check(self, out=None):
        got = cpu(self.run() if out is None else out).double()
        want, bound = self.reference()
        assert torch.equal(got[self.rows:], torch.full_like(got[self.rows:], 3.0)), "rows behind the last sequence"
        off = (got[:self.rows] - want).abs()
        worst = (off / bound).nan_to_num(0.0).max().item() if self.rows else 0.0
        assert torch.isfinite(got).all() and (off <= bound).all(), f"{worst:.2f} of the bound"


FORMS = ["auto", "fp8", "block_int8", "block_fp8"]
HEADS = [(8, 2, 128, 16, torch.bfloat16), (4, 4, 64, 32, torch.float16), (16, 1, 128, 48, torch.float16), (7, 1, 64, 16, torch.bfloat16),
         (6, 2, 128, 64, torch.bfloat16)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("H,KVH,D,bs,dtype", HEADS)
def test_decode_rows(form, H, KVH, D, bs, dtype):
    lens = [(0, 1), (1, 1), (15, 1), (16, 1), (62, 1), (63, 1), (64, 1), (200, 1), (301, 1), (575, 1)]
    b = Batch(lens, H, KVH, D, bs, form, dtype, seed=1)
    b.check()
    b.check(b.run(query_start_loc=None, query=b.dev["q"], max_query_len=1))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("H,KVH,D,bs,dtype", HEADS)
def test_mixed_rows(form, H, KVH, D, bs, dtype):
    """Prompts, chunks over a context, drafts and decode rows in one batch; a sequence without new rows."""
    b = Batch([(0, 37), (130, 5), (64, 70), (90, 1), (33, 0), (0, 1), (255, 2)], H, KVH, D, bs, form, dtype, seed=2)
    b.check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (63, 0), (64, 4), (65, 70), (100, 17), (4096, 4)])
def test_window_and_sinks(form, window, sinks):
    b = Batch([(0, 150), (299, 1), (200, 9), (0, 1), (40, 60), (333, 1)], 4, 2, 64, 16, form, torch.bfloat16, window=window, sinks=sinks, seed=3)
    b.check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (600, 4)])
def test_long_contexts_are_cut_and_joined(form, window, sinks):
    lens = [(4999, 1), (2047, 3), (64, 1)]
    b = Batch(lens, 4, 1, 128, 16, form, torch.float16, window=window, sinks=sinks, seed=4)
    if not window:
        assert ops.paged_window_attention_workspace_bytes(3, b.rows + 1, 4, 1, 128, 3, 5000, form) > 0
    b.check()
    # a bound on the lengths that is far off changes how the work is cut, not what comes out of it
    b.check(b.run(max_seq_len=64))
    b.check(b.run(max_seq_len=1 << 17))


@pytest.mark.parametrize("form", FORMS)
def test_one_long_context_among_many_short_ones(form):
    """More sequences than the chip has room for at once, one of them cut into stretches: alone, with drafts, and with a prompt."""
    short = [(7 * i % 150, 1) for i in range(39)]
    for more, n in (((9000, 1), 1), ((8300, 5), 5), ((4500, 70), 70)):
        b = Batch(short[:20] + [more] + short[20:] + [(4200, n // 2 + 1)], 8, 2, 64, 16, form, torch.bfloat16, seed=16)
        assert ops.paged_window_attention_workspace_bytes(len(b.lens), b.rows + 1, 8, 2, 64, n, b.max_len, form) > 0
        b.check()
        b.check(b.run(max_seq_len=1 << 17))
        b.check(b.run(max_query_len=n + 20))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("window", [0, 100])
def test_prompts_among_many_sequences(form, window):
    """Prompts find their rows in batches of more sequences than a wave has lanes; sequences without rows among them."""
    for long in (150, 2500):
        lens = [(5 * i % 90, 1) for i in range(140)]
        for at, prompt in ((0, (0, 65)), (3, (long, 33)), (63, (10, 90)), (64, (0, 129)), (66, (20, 0)), (128, (7, 64)), (139, (60, 40))):
            lens[at] = prompt
        b = Batch(lens, 8, 2, 64, 16, form, torch.float16, window=window, sinks=3 if window else 0, seed=20)
        b.check()
        b.seq_lens = torch.cat([b.seq_lens, torch.zeros(60, dtype=torch.int32, device=DEV)])       # a batch padded with empty sequences
        b.starts = torch.cat([b.starts, torch.full((60,), b.rows, dtype=torch.int32, device=DEV)])
        b.dev["tables"] = torch.cat([b.dev["tables"], torch.zeros(60, b.tables.shape[1], dtype=torch.int32, device=DEV)])
        b.check()


@pytest.mark.parametrize("form", ["fp8", "block_int8", "block_fp8"])
def test_values_next_to_nothing(form):
    """V scales that are subnormal in 32 bits: the same rows, smaller by a power of two.  Two results rounded to bf16, half a step
    2^-8 each, of values or (subnormal ones) of 2^-133 steps; where scales are this small, prompt rows round a scale and its
    products with the codes to fp16, 2^-11 each of the largest value."""
    b = Batch([(100, 1), (60, 200), (300, 3), (0, 1)], 4, 2, 64, 16, form, torch.bfloat16, seed=23, loud=0.3)
    want = cpu(b.run())[:b.rows].double() * 2.0 ** -124
    top = b.v.abs().max().item() * 2.0 ** -124
    b.dev["vs"] = b.dev["vs"] * 2.0 ** -62 * 2.0 ** -62
    assert 0 < b.dev["vs"].min().item() < 2.0 ** -127
    got = cpu(b.run())[:b.rows].double()
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -133 + 2.0 ** -10 * top).all()
    if form != "fp8":       # next to blocks of zeros
        b.dev["vs"][::2] = 0.0
        assert torch.isfinite(cpu(b.run())).all()


@pytest.mark.parametrize("bound", [1, 3, 20])
def test_query_longer_than_its_bound(bound):
    """As many rows as the bound says are certain, whatever else the batch holds."""
    b = Batch([(100, 30), (3000, 2), (50, 1)], 8, 2, 64, 16, "block_int8", torch.bfloat16, seed=24)
    want, tolerance = b.reference()
    got = cpu(b.run(max_query_len=bound)).double()
    first = torch.tensor([j < bound for _, n in b.lens for j in range(n)])
    assert ((got[:b.rows] - want).abs() <= tolerance)[first].all()


@pytest.mark.parametrize("form", ["auto", "block_int8"])
@pytest.mark.parametrize("lens,bound", [
    ([(0, 300), (50, 20), (10, 1)], 20),             # one query of several column tiles where the bound says one
    ([(0, 300)], 20), ([(7, 200), (0, 20)], 20), ([(0, 20), (30, 500), (90, 3), (5, 17)], 20),
    ([(4200, 400), (5000, 33), (20, 1)], 33),        # contexts in stretches
    ([(3, 1), (0, 700), (40, 130), (8, 129)], 130),
])
def test_query_of_more_column_tiles_than_its_bound(form, lens, bound):
    """The rows within the bound are certain in every sequence, in a batch whose prompts take more column tiles than announced."""
    b = Batch(lens, 8, 2, 64, 16, form, torch.bfloat16, seed=25)
    want, tolerance = b.reference()
    first = torch.tensor([j < bound for _, n in lens for j in range(n)])
    for window in (0, 100):
        if window:
            b.window, b.sinks = window, 3
            want, tolerance = b.reference()
        got = cpu(b.run(max_query_len=bound)).double()
        assert torch.equal(got[b.rows:], torch.full_like(got[b.rows:], 3.0))
        assert ((got[:b.rows] - want).abs() <= tolerance)[first].all()


@pytest.mark.parametrize("heads", [1, 4, 12, 136])
def test_query_heads_that_do_not_fit_the_cache(heads):
    """Fewer query heads than kv heads, no whole number to each, more than 16 to each: an error, before anything is sized by them."""
    b = Batch([(100, 1), (60, 3)], 16, 8, 64, 16, "block_int8", torch.bfloat16, seed=27)
    q = torch.zeros(b.rows, heads, 64, dtype=torch.bfloat16, device=DEV)
    for window in (0, 50):
        with pytest.raises(RuntimeError, match="query heads"):
            b.run(query=q, out=torch.empty_like(q), sliding_window=window)


def test_workspace_in_pieces_is_refused():
    """Elements that do not lie side by side, or are one element many times over, are no room for the kernels."""
    b = Batch([(2999, 1), (700, 3)], 4, 1, 128, 16, "block_int8", torch.bfloat16, seed=14)
    need = ops.paged_window_attention_workspace_bytes(2, b.rows + 1, 4, 1, 128, b.max_query, b.max_len, b.form)
    for ws in (torch.empty(2 * need, dtype=torch.uint8, device=DEV)[::2], torch.empty(1, dtype=torch.uint8, device=DEV).expand(need)):
        assert ws.numel() == need
        with pytest.raises(RuntimeError, match="contiguous"):
            b.run(workspace=ws)


def test_one_scale_that_is_no_number():
    """Rows that see nothing stay zero whatever the scale is."""
    b = Batch([(0, 3), (20, 2), (0, 300)], 4, 2, 64, 16, "fp8", torch.bfloat16, seed=17)
    b.seq_lens.copy_(torch.tensor([0, 22, 100]))
    for name in ("ks", "vs"):
        held, b.dev[name] = b.dev[name], torch.tensor(float("nan"), device=DEV)
        got = cpu(b.run())
        b.dev[name] = held
        assert torch.equal(got[:3], torch.zeros_like(got[:3])) and torch.isnan(got[3:5]).all()
        assert torch.equal(got[5:205], torch.zeros_like(got[5:205])) and torch.isnan(got[205:305]).all()


@pytest.mark.parametrize("form", FORMS)
def test_query_that_is_no_number(form):
    """A NaN in a query row makes that row of that head NaN, nothing else, and no zero of it."""
    b = Batch([(20, 2), (0, 300), (4500, 1)], 4, 2, 64, 16, form, torch.bfloat16, seed=18)
    clean = cpu(b.run())
    for row, head in ((1, 2), (2, 0), (150, 3), (301, 1), (302, 0)):
        b.dev["q"][row, head, 5] = float("nan")
        clean[row, head] = float("nan")
    got = cpu(b.run())
    assert torch.equal(torch.isnan(got), torch.isnan(clean)) and torch.equal(got.nan_to_num(7.0), clean.nan_to_num(7.0))


def test_scale_zero_and_pages_out_of_range():
    """Every token seen weighs the same; a page outside the cache is nobody's, inside a tile that every row sees whole too."""
    for form in FORMS:
        b = Batch([(300, 1), (290, 40)], 8, 2, 64, 16, form, torch.bfloat16, seed=19)
        b.scale = 0.0
        b.tables[0, 2], b.tables[1, 5] = -1, b.blocks
        b.dev["tables"] = b.tables.to(DEV)
        b.check()


def swap_blocks(b, i, j):
    """Pages i and j of a batch's cache change places, in the tables too."""
    for t in (b.k, b.v, b.kc, b.vc) + ((b.dev["ks"], b.dev["vs"]) if b.form.startswith("block") else ()):
        t[[i, j]] = t[[j, i]]
    at_i, at_j = b.tables == i, b.tables == j
    b.tables[at_i], b.tables[at_j] = j, i
    b.dev["tables"] = b.tables.to(DEV)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 20)])
def test_pages_out_of_range_show_nothing_of_block_0(form, window, sinks):
    """A page outside the cache is nobody's, also where block 0 holds nothing but NaN, in tiles that every row sees whole: decode
    rows, drafts, prompt rows, a context in several stretches."""
    for lens in ([(300, 1), (290, 5), (4500, 1)], [(300, 1), (310, 40), (150, 100)]):
        b = Batch(lens, 8, 2, 64, 16, form, torch.bfloat16, window=window, sinks=sinks, seed=26)
        used = set(b.tables.flatten().tolist())
        swap_blocks(b, 0, next(n for n in range(b.blocks) if n not in used))
        for s, (c, n) in enumerate(lens):
            for i, page in enumerate(range(1 + s, (c + n) // 16, 7)):
                b.tables[s, page] = [-1, b.blocks, 1 << 30, -(1 << 31)][i % 4]
        b.dev["tables"] = b.tables.to(DEV)
        nan = {"auto": 0x7fc0, "fp8": 0x7f, "block_fp8": 0xff, "block_int8": 0x80}[form]
        for t in (b.kc, b.vc):
            t.view(torch.int16 if form == "auto" else torch.uint8)[0] = nan
        if form.startswith("block"):
            b.dev["ks"][0] = b.dev["vs"][0] = float("nan")
        b.check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 4)])
def test_longer_prompts(form, window, sinks):
    """Prompt rows past several tiles and column blocks, with a context whose end is inside a page."""
    Batch([(0, 333), (77, 260), (500, 129)], 8, 2, 128, 16, form, torch.bfloat16, window=window, sinks=sinks, seed=5).check()
    Batch([(0, 300), (13, 200)], 3, 1, 64, 32, form, torch.float16, window=window, sinks=sinks, seed=6).check()


@pytest.mark.parametrize("form", FORMS)
def test_masked_places_hold_anything(form):
    """Pages behind the window given away (numbers outside the cache), stale places after a sequence's end full of NaN, scales of
    pages that nobody sees NaN: none of it shows."""
    b = Batch([(300, 1), (130, 1), (200, 40), (5, 20)], 4, 2, 64, 16, form, torch.float16, window=50, sinks=3, seed=7)
    want = cpu(b.run())
    for s, (c, n) in enumerate(b.lens):
        low = max(0, c + 1 - 50)
        for page in range((c + n + 15) // 16):
            if page * 16 >= 3 and (page + 1) * 16 <= low:
                b.tables[s, page] = [-1, 1 << 30, b.blocks, -(1 << 31)][page % 4]
    b.dev["tables"] = b.tables.to(DEV)
    used = torch.zeros(b.blocks, dtype=torch.bool)
    used[b.tables[(b.tables >= 0) & (b.tables < b.blocks)].long()] = True
    nan = {"auto": 0x7e00, "fp8": 0x7f, "block_fp8": 0x7f, "block_int8": 0x80}[form]
    kc, vc = (t.view(torch.int16 if form == "auto" else torch.uint8) for t in (b.kc, b.vc))
    kc[~used] = nan
    vc[~used] = nan
    for s, (c, n) in enumerate(b.lens):
        end, page = (c + n) % 16, int(b.tables[s, (c + n - 1) // 16])
        if end:
            kc[page, :, :, end:] = nan
            vc[page, :, :, end:] = nan
    if form.startswith("block"):
        b.dev["ks"][~used] = float("nan")
        b.dev["vs"][~used] = float("nan")
    got = cpu(b.run())
    assert torch.equal(got, want)
    b.check(got.to(DEV))


@pytest.mark.parametrize("form", ["auto", "fp8"])
@pytest.mark.parametrize("shape", [(0, 40), (60, 7), (0, 200)])
def test_not_finite_tokens_reach_only_the_rows_that_see_them(form, shape):
    """A key or value that is not finite: rows before it (and behind the window) are as if it were not there."""
    c, n = shape
    b = Batch([shape], 4, 2, 64, 16, form, torch.bfloat16, window=24, sinks=2, seed=8)
    clean = cpu(b.run()).double()
    t, end = c + n // 2, c + n
    page, off = int(b.tables[0, t // 16]), t % 16
    if form == "auto":
        b.vc[page, 0, 5, off] = float("inf")
        b.vc[page, 1, 9, off] = float("nan")
    else:
        b.vc[page, 0, 5, off] = 0x7f
        b.vc[page, 1, 9, off] = 0x7f
    got = cpu(b.run()).double()
    for j in range(n):
        sees = t in b.visible(0, j).tolist()
        for h in range(4):
            d = 5 if h < 2 else 9
            rest = [i for i in range(64) if i != d]
            # other head dims: the same sums in another order at most
            assert torch.allclose(got[j, h, rest], clean[j, h, rest], rtol=2 ** -6, atol=2 ** -7)
            if not sees:
                assert torch.isfinite(got[j, h, d]) and abs(got[j, h, d] - clean[j, h, d]) <= 2 ** -6 * abs(clean[j, h, d]) + 2 ** -7
            elif form == "auto" and h < 2:
                assert got[j, h, d] == float("inf")
            else:
                assert torch.isnan(got[j, h, d])
    # keys: a NaN logit makes its row NaN, and no other
    b = Batch([shape], 4, 2, 64, 16, form, torch.bfloat16, window=24, sinks=2, seed=8)
    b.kc[page, 0, 0, off, 0] = float("nan") if form == "auto" else 0x7f
    got = cpu(b.run()).double()
    for j in range(n):
        sees = t in b.visible(0, j).tolist()
        assert torch.isnan(got[j, :2]).all() if sees else torch.allclose(got[j, :2], clean[j, :2], rtol=2 ** -6, atol=2 ** -7)
        assert torch.equal(got[j, 2:], clean[j, 2:])


@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
def test_poisoned_block_reads_as_nan(form):
    b = Batch([(50, 1), (70, 1), (100, 3)], 4, 2, 128, 16, form, torch.bfloat16, window=32, sinks=0, seed=9)
    clean = cpu(b.run())
    b.dev["ks"][int(b.tables[0, 3]), 0] = float("nan")       # tokens 48 .. 63 of sequence 0
    b.dev["vs"][int(b.tables[1, 1]), 1] = float("nan")       # tokens 16 .. 31 of sequence 1: behind its window
    b.dev["vs"][int(b.tables[2, 4]), 1] = float("nan")       # tokens 64 .. 79 of sequence 2
    got = cpu(b.run())
    assert torch.isnan(got[0, :2]).all() and torch.equal(got[0, 2:], clean[0, 2:])
    assert torch.equal(got[1], clean[1])
    assert torch.equal(got[2:5, :2], clean[2:5, :2]) and torch.isnan(got[2:5, 2:]).all()


def test_rows_that_see_nothing():
    """A sequence of length zero, and rows before the sequence's first token (query longer than the sequence)."""
    for form in FORMS:
        b = Batch([(0, 3), (20, 2), (0, 4)], 4, 2, 64, 16, form, torch.bfloat16, seed=10)
        b.seq_lens.copy_(torch.tensor([0, 22, 2]))
        got = cpu(b.run())
        assert torch.equal(got[:3], torch.zeros_like(got[:3])) and torch.equal(got[5:7], torch.zeros_like(got[5:7]))
        assert got[3:5].abs().sum() > 0 and got[7:9].abs().sum() > 0
        b2 = Batch([(0, 3), (20, 2), (0, 4)], 4, 2, 64, 16, form, torch.bfloat16, seed=10)
        assert torch.equal(cpu(b2.run())[3:5], got[3:5])


@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
@pytest.mark.parametrize("lens", [[(9000, 80)], [(9000, 5)], [(8150, 1), (9100, 9)]])
def test_values_of_another_size_on_long_walks(form, lens):
    """The same where a workgroup walks a long context whole: the larger values come last, or first and are left behind by the window."""
    for window, at in ((0, lambda c, n: c + n // 2), (5000, lambda c, n: c + n // 2 - 5000), (0, lambda c, n: 4000), (5000, lambda c, n: c - 300)):
        b = Batch(lens, 8, 2, 64, 16, form, torch.bfloat16, window=window, sinks=2, seed=31, loud=0.3)
        for s, (c, n) in enumerate(lens):
            page = int(b.tables[s, at(c, n) // 16])
            b.v[page] *= 2.0 ** 40
            b.dev["vs"][page] *= 2.0 ** 40
        b.check(b.run(max_seq_len=64))
        b.check()


def test_logits_of_minus_infinity():
    """A row whose logits are all minus infinity is zeros; next to finite ones such a token weighs nothing."""
    b = Batch([(100, 1), (30, 200), (60, 3)], 4, 2, 64, 16, "auto", torch.float16, seed=30)
    b.dev["q"].abs_().add_(0.5)
    lost = [int(p) for p in b.tables[0, :7]] + [int(b.tables[1, 1]), int(b.tables[2, 2])]
    for page in lost:
        b.kc[page, :, 0, :, 0] = -torch.inf
    b.tables[1, 1] = b.tables[2, 2] = -1                # to the formula, tokens of no weight are tokens that nobody sees
    b.q = cpu(b.dev["q"])
    want, bound = b.reference()
    got = cpu(b.run()).double()
    assert torch.equal(got[0], torch.zeros_like(got[0]))
    assert ((got[1:b.rows] - want[1:]).abs() <= bound[1:]).all()


@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("factor", [2.0 ** 24, 2.0 ** 40, 2.0 ** 90])
def test_values_of_another_size_where_a_row_does_not_see_them(form, window, sinks, factor):
    """Blocks whose V is larger by far, ahead of a row or behind its window: the row is held to the largest value that it sees itself.
    Prompts, chunks, drafts of one and of two column tiles, decode rows beside them; a wave that meets such a block first and walks on."""
    def louder(b, s, page):
        b.v[int(b.tables[s, page])] *= factor
        b.dev["vs"][int(b.tables[s, page])] *= factor

    for D, bs in ((64, 16), (128, 32)):
        for lens in ([(0, 300), (130, 90), (70, 1)], [(200, 12), (300, 4), (62, 5), (190, 1)]):
            b = Batch(lens, 8, 2, D, bs, form, torch.bfloat16, window=window, sinks=sinks, seed=28, loud=0.3)
            for s, (c, n) in enumerate(lens):
                for page in {(c + n - 1) // bs, (c + n // 2) // bs} - {0}:
                    louder(b, s, page)
            b.check()
    if window:
        b = Batch([(5, 1)] * 40 + [(2000, 40)], 2, 2, 64, 16, form, torch.bfloat16, window=1200, sinks=sinks, seed=29, loud=0.3)
        louder(b, 40, 800 // 16)
        b.check()
        b = Batch([(2000, 300)], 2, 2, 64, 16, form, torch.bfloat16, window=1200, sinks=sinks, seed=29, loud=0.3)
        louder(b, 0, 816 // 16)
        b.check()


@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
def test_scales_far_apart(form):
    """Blocks whose V scales differ by factors of up to e^30: the probabilities in between keep their bits."""
    b = Batch([(700, 1), (300, 6)], 4, 2, 128, 16, form, torch.bfloat16, seed=11, loud=6.0)
    b.check()


@pytest.mark.parametrize("form", ["block_int8", "fp8", "auto"])
def test_large_and_small_queries(form):
    """Query rows from 2^-40 to 2^30 (bf16): the power of two that brings them to fp16 comes off again."""
    b = Batch([(100, 1), (60, 3), (200, 1)], 4, 2, 64, 16, form, torch.bfloat16, seed=12)
    b.q *= torch.exp2(torch.tensor([-40.0, 0.0, 3.0, 1.0, 2.0, 0.0]))[:, None, None].to(torch.bfloat16)
    b.q[2, 1] = 0.0
    b.dev["q"] = b.q.to(DEV)
    b.check()
    b.q.mul_(2.0 ** 30)
    b.scale *= 2.0 ** -30
    b.dev["q"] = b.q.to(DEV)
    b.check()


def test_strided_rows_tables_and_cache_heads():
    """Query rows inside a wider projection, output rows inside a wider buffer, a cache whose head pages lie apart."""
    b = Batch([(100, 1), (60, 30), (200, 1)], 4, 2, 64, 16, "block_int8", torch.float16, seed=13)
    wide = torch.zeros(b.rows + 1, 4 * 64 + 128, dtype=torch.float16, device=DEV)
    wide[:, 64:-64] = b.dev["q"].flatten(1)
    out = torch.full((b.rows + 1, 4 * 64 + 32), 3.0, dtype=torch.float16, device=DEV)
    kc = torch.zeros(b.blocks, 4, *b.kc.shape[2:], dtype=torch.uint8, device=DEV)[:, ::2]
    vc = torch.zeros(b.blocks, 4, *b.vc.shape[2:], dtype=torch.uint8, device=DEV)[:, ::2]
    kc.copy_(b.kc)
    vc.copy_(b.vc)
    scales = [torch.empty(2, b.blocks, device=DEV).t().copy_(b.dev[n]) for n in ("ks", "vs")]
    got = b.run(query=wide[:, 64:-64].unflatten(1, (4, 64)), out=out[:, :256].unflatten(1, (4, 64)), key_cache=kc, value_cache=vc,
                k_scale=scales[0], v_scale=scales[1])
    assert torch.equal(out[:, 256:], torch.full_like(out[:, 256:], 3.0))
    b.check(got)


@pytest.mark.parametrize("form", ["auto", "fp8", "block_int8"])
def test_pages_past_four_gib(form):
    """The same pages at the far end of a cache of more than 2^32 bytes: same results, bit for bit."""
    b = Batch([(100, 1), (60, 40), (2500, 3)], 8, 2, 64, 16, form, torch.bfloat16, seed=21)
    want = cpu(b.run())
    page = b.kc[0].numel() * b.kc.element_size()
    blocks = (1 << 32) // page + 1000 + b.blocks
    kc, vc = (torch.empty(blocks, *c.shape[1:], dtype=c.dtype, device=DEV) for c in (b.kc, b.vc))
    kc[-b.blocks:], vc[-b.blocks:] = b.kc, b.vc
    more = dict(key_cache=kc, value_cache=vc, block_tables=torch.where(b.dev["tables"] >= 0, b.dev["tables"] + (blocks - b.blocks), b.dev["tables"]))
    if form == "block_int8":
        scales = [torch.zeros(blocks, 2, device=DEV) for _ in range(2)]
        for far, near in zip(scales, ("ks", "vs")):
            far[-b.blocks:] = b.dev[near]
        more.update(k_scale=scales[0], v_scale=scales[1])
    assert torch.equal(cpu(b.run(**more)), want)
    if form == "block_int8":
        x = qkv_rows(50, 8, 2, 64, torch.bfloat16, seed=22).to(DEV)
        slots = torch.arange(5, 55, device=DEV)
        for k, v, s, at in ((b.kc, b.vc, [b.dev["ks"], b.dev["vs"]], slots), (kc, vc, scales, slots + (blocks - b.blocks) * 16)):
            ops.reshape_and_cache_blocks(x[:, 512:640].unflatten(1, (2, 64)), x[:, 640:].unflatten(1, (2, 64)), k, v, *s, at, form)
        assert torch.equal(kc[-b.blocks:], b.kc) and torch.equal(vc[-b.blocks:], b.vc)
        assert torch.equal(scales[0][-b.blocks:], b.dev["ks"]) and torch.equal(scales[1][-b.blocks:], b.dev["vs"])


def test_streams_graphs_and_a_workspace_of_ones_own():
    b = Batch([(2999, 1), (700, 3)], 4, 1, 128, 16, "block_int8", torch.bfloat16, seed=14)
    want = cpu(b.run())
    need = ops.paged_window_attention_workspace_bytes(2, b.rows + 1, 4, 1, 128, b.max_query, b.max_len, b.form)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    assert torch.equal(cpu(b.run(workspace=ws)), want)
    with pytest.raises(RuntimeError, match="workspace"):
        b.run(workspace=ws[:need - 16])
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i in range(12):
        with torch.cuda.stream(streams[i % 4]):
            outs.append(b.run())
    torch.cuda.synchronize()
    assert all(torch.equal(cpu(o), want) for o in outs)
    # two graphs over the same inputs, replayed at once on two streams
    out = [torch.empty_like(b.dev["q"]) for _ in range(2)]
    graphs = []
    for o in out:
        o.fill_(3.0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.run(out=o)
        graphs.append(g)
    for _ in range(5):
        for o in out:
            o.fill_(3.0)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(cpu(o), want) for o in out)


# ---------------------------------------------------------------------------------------------------------------------
# as they are used: append, then attend, step after step
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_generation_over_the_block_scaled_cache(form, window, sinks):
    """Two conversations: prompt, second chunk, decode steps.  Each step's attention is checked against the formula on what the
    cache then holds; the cache itself against the restated append."""
    H, KVH, D, bs, dtype = 4, 2, 64, 16, torch.bfloat16
    c = Cache(20, KVH, D, bs, form)
    cs = angles(D, 256, dtype)
    own = [[3, 9, 1, 17, 5, 8, 0, 11], [2, 4, 19, 6, 7, 10, 12, 13]]
    filled = [0, 0]
    for step, new in enumerate([(45, 20), (0, 33), (1, 1), (1, 1), (1, 4), (1, 1)]):
        pos = [t for s in range(2) for t in range(filled[s], filled[s] + new[s])]
        slots = [own[s][t // bs] * bs + t % bs for s in range(2) for t in range(filled[s], filled[s] + new[s])]
        qkv = qkv_rows(len(pos), H, KVH, D, dtype, 90 + step, loud=0.3)
        run_append(c, qkv, H, KVH, D, torch.tensor(pos), cs, D, True, slots)
        b = Batch([(filled[s], new[s]) for s in range(2)], H, KVH, D, bs, form, dtype, window=window, sinks=sinks)
        b.q = torch.cat([rotate_ref(qkv[:, :H * D].unflatten(1, (H, D)), torch.tensor(pos), cs, D, True, dtype), b.q[-1:]])
        b.k, b.v = c.k_ref.double() * c.ks_ref.double()[..., None, None], c.v_ref.double() * c.vs_ref.double()[..., None, None]
        b.tables = torch.tensor(own, dtype=torch.int32)
        b.blocks, b.kc, b.vc = 20, c.kc, c.vc
        b.dev = dict(q=b.q.to(DEV), tables=b.tables.to(DEV), ks=c.ks, vs=c.vs)
        filled = [f + n for f, n in zip(filled, new)]
        b.check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (30, 4)])
def test_attention_layer(form, window, sinks):
    """plugin.attention.Attention: the cache update and the attention of a prompt, a chunk with a decode row, and a decode step.  The
    cache is held against a layer of its own making: what it holds is read back and put into the formula."""
    from mi355q.plugin.attention import Attention, CommonAttentionMetadata, Mi355AttentionBackend, Mi355AttentionMetadataBuilder
    if window is None and not form.startswith("block"):
        pytest.skip("the layer without window or block scales is another kernel's")
    H, KVH, D, bs, n, dtype = 8, 2, 128, 16, 24, torch.bfloat16
    with torch.device(DEV):
        layer = Attention(H, D, D ** -0.5, KVH, cache_dtype=form, sliding_window=window, sink_tokens=sinks)
    if form == "fp8":
        layer.k_scale.weight_loader(layer.k_scale, torch.tensor(1 / 32))
        layer.v_scale.weight_loader(layer.v_scale, torch.tensor(1 / 64))
    layer.process_weights_after_loading()
    kv = torch.zeros(Mi355AttentionBackend.get_kv_cache_shape(n, bs, KVH, D), dtype=dtype if form == "auto" else torch.uint8, device=DEV)
    layer.kv_cache = kv
    if form.startswith("block"):
        layer.kv_scales = torch.zeros(Mi355AttentionBackend.get_kv_scales_shape(n, KVH), device=DEV)
    builder = Mi355AttentionMetadataBuilder(bs, DEV)
    tables = torch.randperm(n, generator=torch.Generator().manual_seed(2))[:16].view(2, 8).to(torch.int32)
    filled = [0, 0]
    for step, new in enumerate([(70, 33), (1, 20), (1, 1)]):
        pos = [[filled[s] + j for j in range(new[s])] for s in range(2)]
        slots = [int(tables[s, t // bs]) * bs + t % bs for s in range(2) for t in pos[s]]
        rows = len(slots)
        g = torch.Generator().manual_seed(step)
        q, k, v = (torch.randn(rows, h * D, generator=g).to(dtype) for h in (H, KVH, KVH))
        filled = [f + m for f, m in zip(filled, new)]
        md = builder.build(0, CommonAttentionMetadata(
            query_start_loc=torch.tensor([0, new[0], rows], dtype=torch.int32, device=DEV), seq_lens=torch.tensor(filled, dtype=torch.int32, device=DEV),
            num_actual_tokens=rows, max_query_len=max(new), max_seq_len=max(filled), block_table_tensor=tables.to(DEV),
            slot_mapping=torch.tensor(slots, device=DEV)))
        out = layer(q.to(DEV), k.to(DEV), v.to(DEV), md)
        b = Batch([(filled[s] - new[s], new[s]) for s in range(2)], H, KVH, D, bs, form, dtype, window=window or 0, sinks=sinks)
        b.q, b.tables, b.blocks = torch.cat([q, q[:1]]).view(-1, H, D), tables, n
        x = 8 if form == "auto" else 16
        kc = cpu(kv[0]).view(n, KVH, D // x, bs, x).transpose(2, 3)
        vc = cpu(kv[1]).view(n, KVH, D, bs).transpose(2, 3)
        if form == "auto":
            b.k, b.v = kc.reshape(n, KVH, bs, D).double(), vc.double()
        else:
            b.k = kc.reshape(n, KVH, bs, D).contiguous().view(CODE[form]).double()
            b.v = vc.contiguous().view(CODE[form]).double()
            ks, vs = (layer._k_scale, layer._v_scale) if form == "fp8" else layer.kv_scales
            b.k, b.v = (t * (cpu(s).double() if form == "fp8" else cpu(s).double()[..., None, None]) for t, s in ((b.k, ks), (b.v, vs)))
        tail = torch.full((1, H, D), 3.0, dtype=dtype, device=DEV)
        b.check(torch.cat([out.view(rows, H, D), tail]))
        # the newest tokens are in the cache: what is held is within a step of them
        newest = b.v[[s // bs for s in slots], :, [s % bs for s in slots]]
        top = newest.abs().amax(2, keepdim=True)
        step_of = {"auto": 0.0, "fp8": 2.0 ** -4, "block_int8": 1 / 64, "block_fp8": 2.0 ** -4}[form]
        assert ((newest - v.view(rows, KVH, D).double()).abs() <= step_of * top * 1.5).all()


@pytest.mark.parametrize("form,window,sinks", [("block_int8", 0, 0), ("block_fp8", 24, 4), ("auto", 24, 4), ("fp8", 40, 0)])
def test_model_runner_graph_equals_eager(form, window, sinks):
    """LlamaRunner over the block-scaled caches and with a window: the captured decode step gives the eager step's tokens and cache."""
    from mi355q.model import CONFIGS, LlamaRunner
    prompt = torch.randint(0, 1024, (2, 37), generator=torch.Generator().manual_seed(1))
    seen = []
    for graph in (False, True):
        r = LlamaRunner(CONFIGS["tiny"], quant="gptq", kv_cache_dtype=form, max_batch=2, max_seq_len=96, sliding_window=window, sink_tokens=sinks)
        tokens = [r.prefill(prompt).cpu().tolist()]
        if graph:
            r.capture()
        for _ in range(12):
            r.decode_step()
            tokens.append(r.tokens.cpu().tolist())
        seen.append((tokens, [t.clone() for t in r.kc + r.vc], r.kv_scales.clone() if r.block_scaled else None))
    assert seen[0][0] == seen[1][0]
    # (the page tail past the last token may hold what the warm-up of the capture left, in caches it writes)
    if form.startswith("block"):
        assert all(torch.equal(a, b) for a, b in zip(seen[0][1], seen[1][1])) and torch.equal(seen[0][2], seen[1][2])


def test_model_runner_window_wider_than_the_context_changes_nothing():
    """The same prompt with a window that hides nothing: first tokens equal those of the runner without one (both attention kernels
    round to the same 16 bits; logits of a random model are far apart compared with that)."""
    from mi355q.model import CONFIGS, LlamaRunner
    prompt = torch.randint(0, 2048, (2, 50), generator=torch.Generator().manual_seed(3))
    first = []
    for window in (0, 128):
        r = LlamaRunner(CONFIGS["small"], quant="gptq", max_batch=2, max_seq_len=96, sliding_window=window)
        first.append(r.prefill(prompt).cpu().tolist())
    assert first[0] == first[1]
