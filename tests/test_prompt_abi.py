"""Argument checks of the rotating append and of the attention over packed prompts: made on the
host before any device work (host pools)."""
from __future__ import annotations

import ctypes

import pytest

from lattice_b200 import KcmmError, kcmm

ROPE = dict(rotary_dim=64, inv_freq_ptr=16, positions_ptr=16, sections=[12, 10, 10])
APPEND = dict(head_dim=64, num_q_heads=4, q_ptr=16, q_out_ptr=16, k_ptr=16, v_ptr=16,
              slot_mapping_ptr=16, block_offsets_f16_ptr=16, block_offsets_f16_len=4,
              num_tokens=8)
ATTN = dict(query_ptr=16, key_ptr=16, value_ptr=16, out_ptr=16, q_start_ptr=16, k_start_ptr=16,
            batch=2, num_q_tokens=10, num_k_tokens=10, num_q_heads=8, kv_heads=2, head_dim=64,
            scale=0.125)


def make_pool(factory, **kw):
    return factory(**{**dict(kv_heads=2, head_dim=64, max_batch=2, max_seq_len=64), **kw})


def test_rope_layout():
    assert ctypes.sizeof(kcmm.KcmmRope) == 56
    assert kcmm.KcmmRope.sections.offset == 40
    r = kcmm.make_rope(rotary_dim=32, inv_freq_ptr=1, positions_ptr=2)
    assert (r.axes, r.sections[0], r.mode) == (1, 16, kcmm.RopeMode.NEOX)
    with pytest.raises(ValueError, match="1 to 4"):
        kcmm.make_rope(rotary_dim=32, inv_freq_ptr=1, positions_ptr=2, sections=[4, 4, 4, 2, 2])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rope,kw,msg", [
    ({}, dict(q_ptr=0), "null pointer"), ({}, dict(q_out_ptr=0), "null pointer"),
    ({}, dict(k_ptr=0), "null pointer"), ({}, dict(slot_mapping_ptr=0), "null pointer"),
    (dict(inv_freq_ptr=0), {}, "null pointer"), (dict(positions_ptr=0), {}, "null pointer"),
    (dict(inv_freq_ptr=18), {}, "4-byte"), (dict(positions_ptr=17), {}, "4-byte"),
    ({}, dict(num_tokens=0), "must be positive"), ({}, dict(block_offsets_f16_len=0), "positive"),
    ({}, dict(head_dim=63), "even"), ({}, dict(head_dim=258), "even"),
    ({}, dict(head_dim=128), "the pool's"), ({}, dict(num_q_heads=65536), "65535"),
    (dict(rotary_dim=0, sections=[0]), {}, "rotary_dim"),
    (dict(rotary_dim=66, sections=[33]), {}, "rotary_dim"),
    (dict(rotary_dim=31, sections=[15]), {}, "rotary_dim"),
    (dict(sections=[12, 10, 9]), {}, "add up"), (dict(sections=[33, 0]), {}, "add up"),
    (dict(sections=[2 ** 32 - 1, 33]), {}, "add up"),
    (dict(sections=[2, 15, 15], layout="interleaved"), {}, "more pairs"),
    (dict(positions_row_stride=7), {}, "row stride"),
    (dict(positions_row_stride=-8), {}, "row stride"),
    ({}, dict(q_stride_head=32), "strides"), ({}, dict(q_out_stride_head=63), "strides"),
    ({}, dict(k_row_stride=127), "strides"), ({}, dict(v_row_stride=-128), "strides"),
    ({}, dict(k_out_ptr=16, k_out_row_stride=64), "strides"),
    ({}, dict(q_stride_token=-1), "strides"),
    ({}, dict(q_ptr=17), "aligned"), ({}, dict(k_out_ptr=17), "aligned"),
    ({}, dict(cache_format=2), "cache_format"), ({}, dict(cache_format=1), "needs 18"),
    ({}, dict(layer=2), "out of bounds"), ({}, {}, "no device memory"),
    (dict(sections=None), dict(num_q_heads=0, q_ptr=0, q_out_ptr=0), "no device memory")])
def test_rope_append_checks(host_pool_factory, rope, kw, msg, dtype):
    pool = make_pool(host_pool_factory)
    args = {**APPEND, "dtype": dtype, **kw}
    layer = args.pop("layer", 0)
    with pytest.raises(KcmmError, match=msg):
        pool.rope_append(layer, rope=kcmm.make_rope(**{**ROPE, **rope}), **args)


@pytest.mark.parametrize("field,value,msg", [("mode", 0, "rope mode"), ("mode", 3, "rope mode"),
                                             ("axes", 0, "axes"), ("axes", 5, "axes"),
                                             ("layout", 2, "layout")])
def test_rope_fields(host_pool_factory, field, value, msg):
    pool = make_pool(host_pool_factory)
    rope = kcmm.make_rope(**ROPE)
    setattr(rope, field, value)
    with pytest.raises(KcmmError, match=msg):
        pool.rope_append(0, rope=rope, **APPEND)


def test_rope_append_into_a_four_bit_pool(host_pool_factory):
    pool = make_pool(host_pool_factory, head_dim=kcmm.kv4_row_elems(64))
    rope = kcmm.make_rope(**ROPE)
    with pytest.raises(KcmmError, match="the pool's"):
        pool.rope_append(0, rope=rope, **APPEND)
    with pytest.raises(KcmmError, match="no device memory"):
        pool.rope_append(0, rope=rope, cache_format=kcmm.CacheFormat.KV4, **APPEND)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kw,msg", [
    *((dict([(p, 0)]), "null pointer") for p in ("query_ptr", "key_ptr", "value_ptr", "out_ptr",
                                                 "q_start_ptr", "k_start_ptr")),
    *((dict([(p, 0)]), "must be positive") for p in ("batch", "num_q_tokens", "num_k_tokens",
                                                     "num_q_heads", "kv_heads")),
    (dict(batch=65536), "limit"), (dict(num_q_heads=65536), "limit"),
    (dict(num_q_tokens=2 ** 31), "limit"), (dict(num_k_tokens=2 ** 31), "limit"),
    (dict(num_q_tokens=2 ** 31 - 1, num_q_heads=256), "limit"),
    (dict(kv_heads=3), "multiple of kv_heads"), (dict(kv_heads=16), "multiple of kv_heads"),
    (dict(head_dim=0), "unsupported"), (dict(head_dim=60), "unsupported"),
    (dict(head_dim=264), "unsupported"), (dict(causal=2), "causal"),
    (dict(q_stride_head=56), "head strides"), (dict(v_stride_head=8), "head strides"),
    (dict(k_stride_token=132), "multiples of 8"), (dict(out_stride_token=-512), "multiples of 8"),
    (dict(q_stride_head=68), "multiples of 8"), (dict(v_stride_token=2 ** 39), "multiples of 8"),
    (dict(query_ptr=8), "16-byte"), (dict(value_ptr=18), "16-byte"), (dict(out_ptr=24), "16-byte"),
    (dict(q_start_ptr=18), "4-byte"), (dict(k_start_ptr=17), "4-byte"),
    *((dict(scale=x), "scale must be positive")
      for x in (0.0, -0.125, float("nan"), float("inf"), 3e38)),
    (dict(num_k_tokens=2 ** 31 - 1), "limit"),
    ({}, "no device memory")])
def test_prompt_attn_checks(host_pool_factory, kw, msg, dtype):
    pool = make_pool(host_pool_factory)
    with pytest.raises(KcmmError, match=msg):
        pool.prompt_attn(**{**ATTN, "dtype": dtype, **kw})


def test_null_pool(kcmm_lib):
    rope = kcmm.make_rope(**ROPE)
    fn = kcmm_lib.lib.kcmm_rope_append_bf16_on_stream
    assert fn(None, 0, 0, 64, ctypes.byref(rope), 16, 0, 0, 16, 0, 0, 4, 16, 0, 16, 0, 0, 0, 16, 16,
              0, 4, 8, 0, 0) == -1
    fn = kcmm_lib.lib.kcmm_prompt_attn_f16_on_stream
    assert fn(None, 16, 0, 0, 16, 0, 0, 16, 0, 0, 16, 0, 0, 16, 16, 2, 10, 10, 8, 2, 64, 0.125, 1,
              0) == -1
