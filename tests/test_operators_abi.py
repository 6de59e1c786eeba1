"""Argument checks of the 4-bit cache, the accumulated weights, the eviction and the beam
entry points: made on the host before any device work (host pools)."""
from __future__ import annotations

import pytest

from lattice_b200 import KcmmError, kcmm


def test_kv4_row_elems(kcmm_lib):
    for d in (32, 64, 96, 128, 256):
        assert kcmm.kv4_row_elems(d) == kcmm_lib.lib.kcmm_kv4_row_elems(d) == 9 * d // 32
    for d in (0, 16, 100, 288):
        assert kcmm_lib.lib.kcmm_kv4_row_elems(d) == 0
        with pytest.raises(ValueError, match="multiples of 32"):
            kcmm.kv4_row_elems(d)


def kv4_pool(factory, **kw):
    kw = {**dict(kv_heads=2, head_dim=kcmm.kv4_row_elems(64), max_batch=2, max_seq_len=64), **kw}
    return factory(**kw)


ROWS = dict(slot_mapping_ptr=16, block_offsets_f16_ptr=16, block_offsets_f16_len=4, num_tokens=4,
            head_dim=64)


@pytest.mark.parametrize("kw,msg", [
    (dict(slot_mapping_ptr=0), "null pointer"), (dict(num_tokens=0), "must be positive"),
    (dict(block_offsets_f16_len=0), "must be positive"), (dict(head_dim=100), "multiples of 32"),
    (dict(head_dim=128), "needs 36"), (dict(k_row_stride=100), "row strides"),
    (dict(v_row_stride=-128), "row strides"), (dict(k=17), "aligned"),
    (dict(layer=2), "out of bounds"), ({}, "no device memory")])
def test_kv4_rows_checks(host_pool_factory, kw, msg):
    pool = kv4_pool(host_pool_factory)
    args = {**ROWS, **kw}
    k, layer = args.pop("k", 16), args.pop("layer", 0)
    with pytest.raises(KcmmError, match=msg):
        pool.kv4_append(layer, k_src_ptr=k, v_src_ptr=16, **args)
    with pytest.raises(KcmmError, match=msg):
        pool.kv4_read(layer, k_dst_ptr=k, v_dst_ptr=16, **args)


def test_kv4_refuses_short_pages(host_pool_factory):
    pool = kv4_pool(host_pool_factory, block_size=8)
    with pytest.raises(KcmmError, match="multiples of 16"):
        pool.kv4_append(0, k_src_ptr=16, v_src_ptr=16, **ROWS)


DECODE = dict(query_ptr=16, out_ptr=16, block_tables_ptr=16, seq_lens_ptr=16,
              block_offsets_f16_ptr=16, batch=2, num_q_heads=8, kv_heads=2, head_dim=64,
              block_size=16, max_blocks_per_seq=4, scale=0.125)
WEIGHTS = dict(weights_in_ptr=16, weights_out_ptr=16, weights_row_stride=64)


@pytest.mark.parametrize("kw,msg", [
    (dict(query_ptr=0), "null pointer"), (dict(batch=0), "must be positive"),
    (dict(batch=65536), "65535"), (dict(num_q_heads=1), "at least kv_heads"),
    (dict(q_stride_head=32), "strides"), (dict(block_tables_row_stride=3), "strides"),
    (dict(weights_in_ptr=0), "go together"), (dict(weights_row_stride=0), "go together"),
    (dict(weights_out_ptr=18), "4-byte aligned"), (dict(num_q_heads=1024), "at most 256"),
    (dict(layer=9), "out of bounds"), ({}, "no device memory")])
def test_decode_weights_checks(host_pool_factory, kw, msg):
    """The same refusals over both caches."""
    args = {**DECODE, **WEIGHTS, **kw}
    layer = args.pop("layer", 0)
    with pytest.raises(KcmmError, match=msg):
        kv4_pool(host_pool_factory).kv4_paged_attn_decode(layer, **args)
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=2, max_seq_len=64)
    with pytest.raises(KcmmError, match=msg):
        pool.paged_attn_decode_weights(layer, **args)


def test_decode_weights_pool_shape_checks(host_pool_factory):
    pool = kv4_pool(host_pool_factory)
    for kw, msg in ((dict(kv_heads=4), "the pool's"), (dict(block_size=32), "the pool's"),
                    (dict(head_dim=128), "needs 36"), (dict(weights_in_ptr=16), "go together")):
        with pytest.raises(KcmmError, match=msg):
            pool.kv4_paged_attn_decode(0, **{**DECODE, **kw})
    with pytest.raises(KcmmError, match="no device memory"):
        pool.kv4_paged_attn_decode(0, **DECODE)  # weights are optional over the 4-bit cache
    plain = host_pool_factory(kv_heads=2, head_dim=64, max_batch=2, max_seq_len=64)
    with pytest.raises(KcmmError, match="go together"):
        plain.paged_attn_decode_weights(0, **DECODE)
    with pytest.raises(KcmmError, match="multiple of 16"):
        plain.paged_attn_decode_weights(0, **{**DECODE, **WEIGHTS, "block_size": 8})
