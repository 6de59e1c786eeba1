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


EVICT = dict(head_dim=64, block_tables_ptr=16, seq_lens_ptr=16, block_offsets_f16_ptr=16, batch=2,
             max_blocks_per_seq=4, budget=32, sinks=2, recent=8, weights_in_ptr=16,
             weights_out_ptr=16, weights_row_stride=64, positions_in_ptr=16, positions_out_ptr=16,
             next_positions_ptr=16, kept_lens_ptr=16, new_lens_ptr=16)


@pytest.mark.parametrize("kw,msg", [
    (dict(kept_lens_ptr=0), "null pointer"), (dict(positions_in_ptr=18), "4-byte aligned"),
    (dict(budget=0), "must be positive"), (dict(weights_row_stride=0), "must be positive"),
    (dict(batch=65536), "limit"), (dict(block_tables_row_stride=3), "row stride"),
    (dict(sinks=30), "must not exceed budget"), (dict(cache_format=2), "unknown cache_format"),
    (dict(head_dim=32), "the pool's"), (dict(cache_format=1), "needs 18"),
    (dict(layer=2), "out of bounds"), ({}, "no device memory")])
def test_evict_checks(host_pool_factory, kw, msg):
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=2, max_seq_len=64)
    args = {**EVICT, **kw}
    layer = args.pop("layer", 0)
    with pytest.raises(KcmmError, match=msg):
        pool.evict_tokens(layer, **args)


SELECT = dict(logits_ptr=16, dtype="bf16", scores_in_ptr=16, batch=2, beams=4, vocab=1000,
              n_select=8, scores_out_ptr=16, parents_out_ptr=16, tokens_out_ptr=16)


@pytest.mark.parametrize("kw,msg", [
    (dict(logits_ptr=0), "null pointer"), (dict(vocab=0), "must be positive"),
    (dict(n_select=65), "n_select <= 64"), (dict(beams=1, vocab=5), "beams \\* vocab"),
    (dict(batch=20000), "65535"), (dict(vocab=1 << 30), "2\\^31"), (dict(row_stride=999), "stride"),
    (dict(logits_ptr=17), "aligned"), (dict(finished_ptr=16, eos_token=1000), "eos_token"),
    ({}, "no device memory")])
def test_beam_select_checks(host_pool_factory, kw, msg):
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=2, max_seq_len=64)
    with pytest.raises(KcmmError, match=msg):
        pool.beam_select(**{**SELECT, **kw})


def test_beam_select_unknown_dtype(kcmm_lib, host_pool_factory):
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=2, max_seq_len=64)
    assert kcmm_lib.lib.kcmm_beam_select_on_stream(pool.handle, 16, 3, 0, 16, 0, 0, 1, 1, 8, 1, 16,
                                                   16, 16, 0) == -1
    assert "unknown dtype" in pool.last_error()


GATHER = dict(src_ptr=1024, dst_ptr=65536, row_bytes=64, parents_ptr=16, batch=2, beams=4,
              n_select=4)


@pytest.mark.parametrize("kw,msg", [
    (dict(parents_ptr=0), "null pointer"), (dict(row_bytes=0), "must be positive"),
    (dict(row_bytes=66), "multiples of 4"), (dict(dst_ptr=1024 + 256), "overlap"),
    (dict(batch=65535), "65535"), (dict(tokens_ptr=16, token_index=16), "past the row"),
    ({}, "no device memory")])
def test_beam_gather_checks(host_pool_factory, kw, msg):
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=2, max_seq_len=64)
    with pytest.raises(KcmmError, match=msg):
        pool.beam_gather(**{**GATHER, **kw})


def test_truncate_sequence(host_pool_factory):
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=4, max_seq_len=64)
    blocks = pool.alloc_blocks(4)
    seq = pool.register_sequence(blocks)
    pool.update_seq_len(seq, 60)
    fork = pool.fork_sequence(seq)
    pool.truncate_sequence(seq, 33)
    assert pool.block_table(seq) == blocks[:3] and pool.seq_len(seq) == 33
    assert pool.blocks_in_use() == 4 and pool.refcount(blocks[3]) == 1  # the fork's
    pool.truncate_sequence(fork, 32)
    assert pool.block_table(fork) == blocks[:2] and pool.blocks_in_use() == 3
    pool.truncate_sequence(seq, 33)
    pool.truncate_sequence(seq, 0)
    assert pool.block_table(seq) == [] and pool.blocks_in_use() == 2
    with pytest.raises(KcmmError, match="exceeds"):
        pool.truncate_sequence(fork, 33)
    with pytest.raises(KcmmError, match="out of bounds"):
        pool.truncate_sequence(9, 0)


def test_reorder_sequences(host_pool_factory):
    """Whole blocks move by reference counts alone; nothing changes on an error."""
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=4, max_seq_len=64)
    tables = [pool.alloc_blocks(2) for _ in range(3)]
    seqs = [pool.register_sequence(t) for t in tables]
    for s, n in zip(seqs, (32, 32, 16)):
        pool.update_seq_len(s, n)

    def state():
        return ([pool.block_table(s) for s in seqs], [pool.seq_len(s) for s in seqs],
                pool.blocks_in_use(), [pool.refcount(b) for t in tables for b in t])

    before = state()
    for bad, msg in (((seqs, [0, 1, 3]), "out of bounds"), (([0, 1, 7], [0, 1, 2]), "out of bounds"),
                     (([0, 1, 0], [0, 1, 2]), "twice"),
                     ((seqs, [2, 2, 2]), "no device memory")):  # a spare block of 2 is shared
        with pytest.raises(KcmmError, match=msg):
            pool.reorder_sequences(*bad)
        assert state() == before
    pool.reorder_sequences(seqs, [0, 1, 2])
    assert state() == before
    pool.reorder_sequences(seqs, [1, 0, 2])  # a swap frees nothing
    assert state() == ([tables[1], tables[0], tables[2]], [32, 32, 16], 6, [1] * 6)
    pool.reorder_sequences(seqs, [1, 1, 2])  # table 1 is dropped, table 0 has two owners
    assert state() == ([tables[0], tables[0], tables[2]], [32, 32, 16], 4, [2, 2, 0, 0, 1, 1])


def test_reorder_sequences_wants_a_parent_for_each(host_pool_factory):
    """The library reads as many parents as there are sequences."""
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=4, max_seq_len=64)
    seqs = [pool.register_sequence(pool.alloc_blocks(1)) for _ in range(3)]
    for parents in ([0, 1], [], [0, 1, 2, 0]):
        with pytest.raises(ValueError, match="3 sequences"):
            pool.reorder_sequences(seqs, parents)


def test_beam_gather_sizes_past_64_bits(host_pool_factory):
    """The source's 2^64 bytes hold the destination."""
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=2, max_seq_len=64)
    with pytest.raises(KcmmError, match="overlap"):
        pool.beam_gather(**{**GATHER, "batch": 1, "beams": 1 << 30, "row_bytes": 1 << 34,
                            "n_select": 1, "dst_ptr": 65536})
