"""Decode over the 16-bit cache with accumulated attention weights, against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from kv_cases import Cache, check_decode, torch_cuda

pytestmark = pytest.mark.gpu

LENS = [0, 1, 15, 16, 17, 33, 160, 777]


@pytest.mark.parametrize("dtype,hq,hkv,d,bs", [
    ("bf16", 32, 8, 128, 16), ("f16", 16, 4, 64, 16), ("bf16", 8, 1, 128, 32),
    ("f16", 6, 6, 32, 16), ("bf16", 12, 4, 96, 16), ("bf16", 16, 1, 256, 16),
    ("f16", 14, 2, 160, 48), ("bf16", 40, 2, 128, 16), ("f16", 9, 1, 112, 16),
    ("bf16", 7, 3, 192, 16), ("f16", 8, 8, 80, 64)])
def test_decode_weights(dtype, hq, hkv, d, bs):
    torch = torch_cuda()
    c = Cache(LENS, hkv, d, bs, dtype=dtype, seed=hq + d)
    try:
        rows = c.fill_rows(k_amp=1.3)
        q = torch.from_numpy(c.rng.standard_normal((len(LENS), hq, d))).cuda().to(c.tdt)
        out = torch.full_like(q, float("nan"))
        w_in = torch.rand(len(LENS), hkv, max(LENS) + 3, device="cuda")
        w_out = torch.full_like(w_in, -5.0)
        c.decode(q, d ** -0.5, out, w_in=w_in, w_out=w_out)
        check_decode(c, rows, q, out, d ** -0.5, w_in=w_in, w_out=w_out,
                     untouched=np.full((len(LENS), hq, d), np.nan))
        for b, n in enumerate(LENS):
            assert bool((w_out[b, :, n:] == -5.0).all())
        assert c.pool.kernel_status() == 0
    finally:
        c.close()


def test_output_equals_the_plain_decode():
    """The weights do not change the output: the merge is the only difference."""
    torch = torch_cuda()
    c = Cache([300, 1, 47], 2, 128, seed=3)
    try:
        c.fill_rows()
        q = torch.from_numpy(c.rng.standard_normal((3, 8, 128))).cuda().to(c.tdt)
        w = torch.zeros(3, 2, 304, device="cuda")
        out = c.decode(q, 0.09, torch.zeros_like(q), w_in=w, w_out=w)
        plain = torch.zeros_like(q)
        c.pool.paged_attn_decode(
            0, query_ptr=q.data_ptr(), out_ptr=plain.data_ptr(),
            block_tables_ptr=c.d_tables.data_ptr(), seq_lens_ptr=c.d_lens.data_ptr(),
            block_offsets_f16_ptr=c.d_offsets.data_ptr(), batch=3, num_q_heads=8, kv_heads=2,
            head_dim=128, block_size=16, max_blocks_per_seq=c.max_bps, scale=0.09,
            stream_ptr=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        diff = (out.float() - plain.float()).abs()
        assert bool((diff <= 2.0 ** -7 * plain.float().abs() + 1e-6).all())  # a unit of bf16
        # every query head's weights sum to 1
        assert np.allclose(w.sum(-1).cpu().numpy(), 4.0, atol=1e-4)
    finally:
        c.close()


def test_long_rows_short_weights_and_a_stream():
    """A context of many splits, a weights row shorter than it, in place, on another stream."""
    torch = torch_cuda()
    c = Cache([9001, 2048], 1, 64, dtype="f16", seed=5)
    try:
        rows = c.fill_rows()
        q = torch.from_numpy(c.rng.standard_normal((2, 8, 64))).cuda().to(c.tdt)
        w = torch.rand(2, 1, 5000, device="cuda")
        before = w.clone()
        out = torch.zeros_like(q)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            c.decode(q, 0.125, out, w_in=w, w_out=w)
        check_decode(c, rows, q, out, 0.125, w_in=before, w_out=w)
    finally:
        c.close()


@pytest.mark.parametrize("kv4", [False, True])
def test_pages_that_cannot_be_read_weigh_nothing(kv4):
    """Table entries of -1 are reported, and their tokens weigh nothing: all of a sequence's,
    those of a whole split, single pages."""
    from kv_cases import attention

    torch = torch_cuda()
    lens, d = [50, 6000, 50], 64
    c = Cache(lens, 1, d, kv4=kv4, seed=9)
    try:
        rows = c.fill_rows()
        c.d_tables[0] = -1
        gone = np.zeros(6000, bool)
        for first, last in ((1600, 4800), (160, 176), (5984, 6000)):
            c.d_tables[1, first // 16: last // 16] = -1
            gone[first:last] = True
        q = torch.from_numpy(c.rng.standard_normal((3, 4, d))).cuda().to(c.tdt)
        w_in = torch.rand(3, 1, 6000, device="cuda")
        w_out = torch.full_like(w_in, -5.0)
        out = c.decode(q, 0.125, torch.full_like(q, 7.0), w_in=w_in, w_out=w_out)
        assert c.pool.kernel_status() == 2
        assert torch.equal(w_out[0, 0, :50], w_in[0, 0, :50]) and bool((out[0] == 0).all())
        for b, keep in ((1, ~gone), (2, np.ones(50, bool))):
            k, v = (x[keep] for x in rows[b])
            ref, mass, w = attention(q[b].double().cpu().numpy(), k, v, 0.125)
            err = np.abs(out[b].double().cpu().numpy() - ref)
            assert (err <= 1.25 * 2.0 ** -11 * mass + 2.0 ** -8 * np.abs(ref) + 1e-7).all()
            step = np.zeros(lens[b])
            step[keep] = w[0]
            before, after = (x[b, 0, : lens[b]].double().cpu().numpy() for x in (w_in, w_out))
            want = before + step
            assert (np.abs(after - want) <= 2.0 ** -14 * step + 2.0 ** -23 * want + 1e-9).all()
            assert np.array_equal(after[~keep], before[~keep])
    finally:
        c.close()


def test_nan_scores_give_nan_weights():
    torch = torch_cuda()
    for kv4 in (False, True):
        c = Cache([40, 40], 1, 64, kv4=kv4, seed=9)
        try:
            c.fill_rows()
            q = torch.from_numpy(c.rng.standard_normal((2, 4, 64))).cuda().to(c.tdt)
            q[0] = float("nan")
            w = torch.zeros(2, 1, 40, device="cuda")
            out = c.decode(q, 0.125, torch.zeros_like(q), w_in=w, w_out=w)
            assert bool(torch.isnan(w[0]).all()) and bool(torch.isnan(out[0]).all())
            assert bool(torch.isfinite(w[1]).all()) and bool(torch.isfinite(out[1]).all())
        finally:
            c.close()
