"""Refusals and sizing of the block-scaled cache and of windowed attention: host checks only, no kernel is launched."""
import ctypes
import random

import pytest
import torch

from mi355q import _lib, ops
from mi355q.plugin.attention import Attention, Mi355AttentionBackend, Mi355AttentionImpl, Mi355AttentionMetadata

_BUFFER = ctypes.create_string_buffer(4096)
PTR = (ctypes.addressof(_BUFFER) + 63) & ~63   # never read: every call below is refused

APPEND = dict(positions=PTR, query=PTR, query_stride=512, query_out=PTR, query_out_stride=512, key=PTR, key_stride=512, value=PTR,
              value_stride=512, head_size=128, num_heads=4, num_kv_heads=2, cos_sin=PTR, rot_dim=128, max_position=64, cos_dtype=_lib.BF16,
              is_neox=1, key_cache=PTR, value_cache=PTR, num_blocks=8, block_size=16, block_stride=2 * 128 * 16, k_scales=PTR,
              v_scales=PTR, scale_block_stride=2, scale_head_stride=1, slots=PTR, num_tokens=3, dtype=_lib.BF16, code_type=_lib.KV_INT8,
              stream=None)
ATTEND = dict(out=PTR, out_stride=512, query=PTR, q_stride=512, key_cache=PTR, value_cache=PTR, kv_block_stride=2 * 128 * 16,
              kv_head_stride=128 * 16, num_blocks=8, num_rows=3, num_seqs=2, num_heads=4, num_kv_heads=2, head_size=128, scale=0.1,
              tables=PTR, width=4, seq_lens=PTR, starts=PTR, max_query_len=2, block_size=16, max_seq_len=64, window=0, sinks=0,
              dtype=_lib.BF16, kv_type=_lib.KV_INT8, k_scale=PTR, v_scale=PTR, scale_block_stride=2, scale_head_stride=1, workspace=None,
              workspace_bytes=0, stream=None)


def refused(fn, args, message, status=_lib.EINVAL, **over):
    assert set(over) <= set(args)
    assert fn(*{**args, **over}.values()) == status
    assert message in _lib.lib().mi355q_last_error().decode()


@pytest.mark.parametrize("over,message", [
    (dict(dtype=_lib.FP32), "dtype"), (dict(code_type=_lib.KV_16), "codes"), (dict(head_size=96), "head_size"),
    (dict(num_kv_heads=0), "bad sizes"), (dict(num_tokens=-1), "bad sizes"), (dict(key=None), "null"), (dict(k_scales=None), "null"),
    (dict(slots=None), "null"), (dict(query_out=None), "null"), (dict(block_size=24), "block size"), (dict(block_size=80), "block size"),
    (dict(num_blocks=1 << 28), "blocks"), (dict(num_blocks=0), "blocks"), (dict(block_stride=128), "block stride"),
    (dict(block_stride=2 * 128 * 16 + 8), "block stride"), (dict(key_cache=PTR + 8), "aligned"), (dict(rot_dim=130), "rot_dim"),
    (dict(rot_dim=3), "rot_dim"), (dict(positions=None), "positions"), (dict(max_position=0), "positions"), (dict(cos_dtype=7), "cos/sin"),
])
def test_append_refusals(over, message):
    refused(_lib.lib().mi355q_rope_and_cache_blocks, APPEND, message, **over)


def test_more_than_a_launch_holds_is_refused():
    refused(_lib.lib().mi355q_rope_and_cache_blocks, APPEND, "too many", num_tokens=(1 << 31) - 1)
    refused(_lib.lib().mi355q_paged_window_attention, ATTEND, "too many", num_seqs=1 << 24, num_rows=1 << 24, max_query_len=1)


def test_sizes_whose_products_pass_64_bits_are_refused():
    """Workgroups times threads wrap around to a small number, or to none."""
    many = 1 << 30
    refused(_lib.lib().mi355q_rope_and_cache_blocks, APPEND, "too many", num_tokens=1 << 26, num_kv_heads=many, block_stride=many * 128 * 16)
    for heads, longest in ((many, 1), (many, 64), (1 << 25, 1), ((1 << 31) - 1, (1 << 31) - 1)):
        refused(_lib.lib().mi355q_paged_window_attention, ATTEND, "too many", num_seqs=many, num_rows=many, num_heads=heads, num_kv_heads=heads,
                max_query_len=longest)


def test_nothing_to_append_is_no_error():
    assert _lib.lib().mi355q_rope_and_cache_blocks(*{**APPEND, "num_tokens": 0}.values()) == _lib.OK


@pytest.mark.parametrize("over,message", [
    (dict(dtype=_lib.FP32), "dtype"), (dict(kv_type=3), "cache type"), (dict(num_rows=-1), "bad sizes"), (dict(tables=None), "null"),
    (dict(k_scale=None), "k_scale"), (dict(head_size=80), "head_size"), (dict(num_heads=5), "query heads"),
    (dict(num_heads=34), "query heads"), (dict(block_size=8), "block size"), (dict(block_size=272), "block size"),
    (dict(num_blocks=0), "block table"), (dict(width=0), "block table"), (dict(width=1 << 27), "block table"),
    (dict(max_query_len=0), "length"), (dict(max_seq_len=0), "length"), (dict(window=-1), "length"), (dict(sinks=-1), "length"),
    (dict(starts=None, num_seqs=4), "rows"), (dict(kv_head_stride=64), "strides"), (dict(kv_block_stride=2 * 128 * 16 + 8), "strides"),
    (dict(query=PTR + 2), "aligned"), (dict(q_stride=516), "aligned"), (dict(out=PTR + 2), "aligned"), (dict(out_stride=513), "aligned"),
])
def test_attention_refusals(over, message):
    refused(_lib.lib().mi355q_paged_window_attention, ATTEND, message, **over)


def test_workspace_is_asked_for_and_checked():
    L = _lib.lib()
    size = L.mi355q_paged_window_attention_workspace_bytes
    assert size(32, 32, 32, 8, 128, 1, 4096, 0, 0, _lib.KV_INT8) == 0            # a full batch: nothing to join
    need = size(1, 1, 32, 8, 128, 1, 1 << 17, 0, 0, _lib.KV_INT8)
    assert need > 0 and need % (32 * (128 + 2) * 4) == 0
    assert size(1, 1, 32, 8, 128, 1, 1 << 17, 512, 4, _lib.KV_INT8) == 0         # a window bounds the work
    assert size(0, 1, 32, 8, 128, 1, 100, 0, 0, 0) == 0
    long = dict(num_seqs=1, num_rows=1, max_query_len=1, max_seq_len=1 << 17, width=1 << 13)
    refused(L.mi355q_paged_window_attention, ATTEND, "workspace", _lib.ENOSPACE, **long)
    refused(L.mi355q_paged_window_attention, ATTEND, "workspace", _lib.ENOSPACE, **long, workspace=PTR, workspace_bytes=16)
    refused(L.mi355q_paged_window_attention, ATTEND, "16-byte", **long, workspace=PTR + 4, workspace_bytes=1 << 30)


def test_every_batch_has_a_plan_of_bounded_scratch():
    """Any bounds a caller may give, those that contradict each other among them.  Decode rows: at most 32 stretches, or 256
    workgroups of 32 columns; prompts: 256 workgroups of 256 columns, rounded up by less than one stretch of every column."""
    size, rng = _lib.lib().mi355q_paged_window_attention_workspace_bytes, random.Random(1)
    spread = lambda top: int(2 ** rng.uniform(0, top))
    for _ in range(20000):
        seqs, longest, kvh, group, head = spread(10), spread(14), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16]), rng.choice([64, 128])
        rows = rng.choice([seqs, max(seqs, longest), seqs + longest, rng.randint(1, seqs + longest)])
        got = size(seqs, rows, kvh * group, kvh, head, longest, spread(20), rng.choice([0, 0, 1, 100, 4096]), rng.choice([0, 4]), rng.choice([0, 1, 2]))
        assert got % ((head + 2) * 4) == 0 and got <= max(32 * rows * kvh * group, 256 * 256 * 2) * (head + 2) * 4


@pytest.mark.parametrize("heads,kv_heads", [(4, 8), (1, 2), (5, 2), (34, 2), (0, 1), (1, 0), (-4, 2), (4, -2), (-4, -2), (1, 1 << 30)])
def test_heads_that_do_not_fit_are_refused(heads, kv_heads):
    """Also where the size of the scratch is asked for, before the attention has seen them."""
    L = _lib.lib()
    for window in (0, 100):
        for longest in (1, 5, 300):
            assert L.mi355q_paged_window_attention_workspace_bytes(1, 3, heads, kv_heads, 128, longest, 1 << 17, window, 4, _lib.KV_INT8) == 0
            refused(L.mi355q_paged_window_attention, ATTEND, "query heads", num_heads=heads, num_kv_heads=kv_heads, window=window,
                    max_query_len=longest)
    for bad in (dict(window=-1), dict(sinks=-1), dict(window=-(1 << 31))):
        bounds = dict(seqs=1, rows=1, heads=4, kv_heads=2, head=128, longest=1, context=1 << 17, window=0, sinks=0, kv=_lib.KV_INT8)
        assert L.mi355q_paged_window_attention_workspace_bytes(*{**bounds, **bad}.values()) == 0


def test_nothing_to_attend_is_no_error():
    f = _lib.lib().mi355q_paged_window_attention
    assert f(*{**ATTEND, "num_rows": 0}.values()) == _lib.OK and f(*{**ATTEND, "num_seqs": 0}.values()) == _lib.OK


def test_ops_refuse_host_tensors():
    t, i = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    kc, vc, s = torch.zeros(4, 1, 8, 16, 16, dtype=torch.uint8), torch.zeros(4, 1, 128, 16, dtype=torch.uint8), torch.zeros(4, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.rope_and_cache_blocks(i, t, t, t, 128, t, True, kc, vc, s, s, i, "block_int8")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.reshape_and_cache_blocks(t[:, None], t[:, None], kc, vc, s, s, i, "block_fp8")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.paged_window_attention(t[:, None], t[:, None], kc, vc, 1, 0.1, i.int()[:, None], i.int(), None, 1, 1, "block_int8", s, s)


def test_attention_layer_arguments():
    assert Mi355AttentionBackend.supports_sliding_window() and not Mi355AttentionBackend.supports_sink()
    assert Mi355AttentionBackend.get_kv_scales_shape(10, 8) == (2, 10, 8)
    impl = Mi355AttentionImpl(8, 128, 0.1, 2, None, 512, "auto", sink_tokens=4)
    assert impl.windowed and not impl.block_scaled and (impl.sliding_window, impl.sink_tokens) == (512, 4)
    assert not impl.decode_fused_supported() and impl.fused_rope_kvcache_supported()
    for form in ("block_int8", "block_fp8"):
        impl = Mi355AttentionImpl(8, 64, 0.1, 2, kv_cache_dtype=form)
        assert impl.windowed and impl.block_scaled and impl.sliding_window == 0 and not impl.decode_fused_supported()
        with pytest.raises(NotImplementedError):
            impl.forward_decode_fused(None, None, None, None, None, None, None)
    assert not Mi355AttentionImpl(8, 128, 0.1, 2).windowed
    with pytest.raises(NotImplementedError, match="sink logits"):
        Mi355AttentionImpl(8, 128, 0.1, 2, sinks=torch.zeros(8))
    with pytest.raises(NotImplementedError, match="soft-capping"):
        Mi355AttentionImpl(8, 128, 0.1, 2, logits_soft_cap=30.0)
    with pytest.raises(NotImplementedError, match="ALiBi"):
        Mi355AttentionImpl(8, 128, 0.1, 2, [0.1] * 8, 512)
    with pytest.raises(NotImplementedError, match="ALiBi"):
        Mi355AttentionImpl(8, 128, 0.1, 2, [0.1] * 8, None, "block_int8")
    for bad in (dict(sliding_window=0), dict(sliding_window=-3), dict(sink_tokens=-1)):
        with pytest.raises(ValueError):
            Mi355AttentionImpl(8, 128, 0.1, 2, **bad)
    layer = Attention(8, 128, 0.1, 2, cache_dtype="block_fp8", sliding_window=64)
    layer.process_weights_after_loading()
    assert layer.impl.block_scaled and not hasattr(layer, "k_scale") and layer.kv_scales is None


@pytest.mark.parametrize("form", ["block_int8", "block_fp8"])
def test_layer_without_its_scales_says_so(form):
    layer = Attention(4, 64, 0.1, 2, cache_dtype=form)
    layer.kv_cache = torch.zeros(Mi355AttentionBackend.get_kv_cache_shape(3, 16, 2, 64), dtype=torch.uint8)
    q, k = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(2, 128, dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32)
    md = Mi355AttentionMetadata(2, 2, torch.tensor([0, 2], **i32), 2, torch.tensor([2], **i32), torch.zeros(1, 1, **i32), torch.arange(2))
    for call in (lambda: layer(q, k, k, md), lambda: layer.impl.forward(layer, q, k, k, layer.kv_cache, md, torch.empty_like(q)),
                 lambda: layer.impl.do_rope_and_kv_cache_update(layer, q, k, k, torch.arange(2), torch.zeros(4, 64), True, layer.kv_cache, md.slot_mapping)):
        with pytest.raises(RuntimeError, match="kv_scales"):
            call()


def test_registered_operators_have_schemas_and_fakes():
    from mi355q.plugin.torch_ops import register_torch_ops
    register_torch_ops()
    for name, written in (("rope_and_cache_blocks", 5), ("reshape_and_cache_blocks", 4), ("paged_window_attention", 1)):
        schema = getattr(torch.ops.mi355q, name).default._schema
        assert sum(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments) == written
    m = dict(device="meta")
    t = torch.empty(2, 4, 64, dtype=torch.bfloat16, **m)
    torch.ops.mi355q.paged_window_attention(t, t, torch.empty(1, **m), torch.empty(1, **m), 1, 0.1, torch.empty(1, **m), torch.empty(1, **m), None, 1,
                                            1, "auto", None, None, 0, 0)
