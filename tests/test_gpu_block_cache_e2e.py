"""LlamaRunner over the block-scaled caches and with a sliding window, token for token against a model of its own: the oracle's
projections and norms, the append as test_gpu_block_cache.py restates it, attention in 64 bits."""
import numpy as np
import pytest
import torch

import oracle as orc
from test_gpu_block_cache import append_ref

pytestmark = pytest.mark.gpu


class History:
    """What one layer's cache holds of one sequence."""

    def __init__(self, form, KVH, D, bs, max_len, scales):
        self.form, self.bs, self.len, self.one = form, bs, 0, scales
        blocks = -(-max_len // bs)
        self.k, self.v = (torch.zeros(blocks, KVH, bs, D) for _ in range(2))
        self.ks, self.vs = (torch.zeros(blocks, KVH) for _ in range(2))

    def append(self, k, v):
        slots = list(range(self.len, self.len + len(k)))
        self.len += len(k)
        for codes, scales, one, x in ((self.k, self.ks, self.one[0], k), (self.v, self.vs, self.one[1], v)):
            if self.form.startswith("block"):
                append_ref(codes, scales, x, slots, self.bs, self.form)
                continue
            held = x.float() if self.form == "auto" else (x.float() / one).clamp(-448, 448).to(torch.float8_e4m3fn).float()
            for t, row in zip(slots, held):
                codes[t // self.bs, :, t % self.bs] = row

    def tokens(self):
        """(k, v) [kv heads, tokens, head] in 64 bits."""
        out = []
        for codes, scales, one in ((self.k, self.ks, self.one[0]), (self.v, self.vs, self.one[1])):
            scale = scales.double()[..., None, None] if self.form.startswith("block") else 1.0 if self.form == "auto" else float(one)
            out.append((codes.double() * scale).transpose(0, 1).flatten(1, 2)[:, :self.len])
        return out


def generate(runner, prompt, n_new):
    """Tokens [step][sequence] and the logits behind them; a prompt's rows together, as its cache takes them in one call."""
    from oracle_model import _bits, _gemm
    cfg, form, D, H, KVH = runner.cfg, runner.kv_cache_dtype, runner.cfg.head_dim, runner.heads, runner.kv_heads
    window, sinks = runner.sliding_window, runner.sink_tokens
    bf16 = lambda bits: torch.from_numpy(np.ascontiguousarray(bits).view(np.int16)).view(torch.bfloat16)

    def attend(q, past, positions):
        k, v = past.tokens()
        t = torch.arange(past.len)
        p = torch.tensor(positions)[:, None]
        keep = (t <= p) & ((t > p - window) | (t < sinks) if window else t >= 0)
        z = q.double().view(len(positions), KVH, H // KVH, D).permute(1, 2, 0, 3) @ k[:, None].transpose(2, 3) * runner.scale
        w = torch.softmax(z.masked_fill(~keep, -torch.inf), 3)
        return _bits((w @ v[:, None]).permute(2, 0, 1, 3).reshape(len(positions), H * D).to(torch.bfloat16))

    tokens, logits = [[0] * len(prompt) for _ in range(n_new)], [[None] * len(prompt) for _ in range(n_new)]
    for b in range(len(prompt)):
        past = [History(form, KVH, D, runner.block_size, prompt.shape[1] + n_new, (runner.k_scale.cpu(), runner.v_scale.cpu())) for _ in runner.layers]
        new, at = prompt[b].tolist(), 0
        for step in range(n_new):
            positions = list(range(at, at + len(new)))
            h, residual = _bits(runner.embed)[new].copy(), None
            for L, cache in zip(runner.layers, past):
                if residual is None:
                    residual, x = h.copy(), orc.rms_norm(h, _bits(L["ln1"]), cfg.rms_eps)
                else:
                    x, residual = orc.fused_add_rms_norm(h, residual, _bits(L["ln1"]), cfg.rms_eps)
                qkv = _gemm(L["qkv"], x)
                q, k, v = (np.ascontiguousarray(t) for t in (qkv[:, :H * D], qkv[:, H * D:(H + KVH) * D], qkv[:, (H + KVH) * D:]))
                q, k = orc.rotary_embedding(np.array(positions), q, k, _bits(runner.cos_sin), D, True)
                cache.append(*(bf16(t).view(len(new), KVH, D) for t in (k, v)))
                o = _gemm(L["o"], attend(bf16(q), cache, positions))
                o, residual = orc.fused_add_rms_norm(o, residual, _bits(L["ln2"]), cfg.rms_eps)
                h = _gemm(L["down"], orc.silu_and_mul(_gemm(L["gate_up"], o)))
            last, _ = orc.fused_add_rms_norm(h[-1:], residual[-1:], _bits(runner.norm), cfg.rms_eps)
            lg = orc.linear_h16(last, _bits(runner.lm_head))
            tokens[step][b], logits[step][b] = int(orc.argmax_h16(lg)[0]), orc.h16_to_f32(lg[0])
            at += len(new)
            new = [tokens[step][b]]
    return tokens, logits


@pytest.mark.parametrize("model,quant", [("tiny", "gptq"), ("small", "awq")])
@pytest.mark.parametrize("form,window,sinks", [("auto", 24, 4), ("fp8", 24, 0), ("block_int8", 0, 0), ("block_int8", 24, 4), ("block_fp8", 0, 0),
                                               ("block_fp8", 20, 3)])
def test_greedy_tokens_match_a_model_of_its_own(model, quant, form, window, sinks, monkeypatch):
    from mi355q import ops
    from mi355q.model import CONFIGS, LlamaRunner
    from oracle_model import assert_tokens_match
    monkeypatch.setattr(ops, "DEQUANT_MATMUL_MIN_TOKENS", 1 << 30)     # the prompt on the kernels whose arithmetic the oracle restates
    cfg = CONFIGS[model]
    runner = LlamaRunner(cfg, quant=quant, kv_cache_dtype=form, device="cuda:0", max_batch=2, max_seq_len=64, keep_checkpoint=True, seed=5,
                         sliding_window=window, sink_tokens=sinks)
    prompt = torch.randint(0, cfg.vocab, (2, 37), generator=torch.Generator().manual_seed(4))
    got = [runner.prefill(prompt).cpu().tolist()]
    runner.capture()
    for _ in range(5):
        runner.decode_step()
        got.append(runner.tokens.cpu().tolist())
    want, logits = generate(runner, prompt, 6)
    assert_tokens_match(got, want, logits)
    assert got[0] == want[0] and sum(g == w for g, w in zip(got, want)) >= 4


def test_the_window_and_the_codes_matter(monkeypatch):
    """The comparison above can tell: without the window, or over another cache, the logits are others."""
    from mi355q import ops
    from mi355q.model import CONFIGS, LlamaRunner
    monkeypatch.setattr(ops, "DEQUANT_MATMUL_MIN_TOKENS", 1 << 30)
    runner = LlamaRunner(CONFIGS["tiny"], quant="gptq", kv_cache_dtype="block_int8", device="cuda:0", max_batch=1, max_seq_len=64,
                         keep_checkpoint=True, seed=5, sliding_window=24, sink_tokens=4)
    prompt = torch.randint(0, 1024, (1, 37), generator=torch.Generator().manual_seed(4))
    base = generate(runner, prompt, 1)[1][0][0]
    for name, value in (("sliding_window", 12), ("sliding_window", 0), ("kv_cache_dtype", "block_fp8")):
        held = getattr(runner, name)
        setattr(runner, name, value)
        assert np.abs(generate(runner, prompt, 1)[1][0][0] - base).max() > 0
        setattr(runner, name, held)
