"""Calls that several host threads make on one stream: launches of a call hand results to each
other through the stream's scratch, which no other call's launches may use in between."""
from __future__ import annotations

import threading

import numpy as np
import pytest

from kv_cases import Cache, torch_cuda

pytestmark = pytest.mark.gpu


def test_calls_of_several_threads_on_one_stream():
    torch = torch_cuda()
    stream = torch.cuda.Stream()
    made = []

    def evict():
        c = Cache([3000, 2500], 4, 64, seed=1)
        made.append(c)
        c.fill_rows()
        z = lambda dt: torch.zeros(2, 4, 3000, device="cuda", dtype=dt)  # noqa: E731
        w, w_out = torch.rand(2, 4, 3000, device="cuda"), z(torch.float32)
        p, p_out = z(torch.int32), z(torch.int32)
        kept, new = torch.zeros_like(c.d_lens), torch.zeros_like(c.d_lens)

        def call():  # the kept rows beyond the budget move to the same slots every time
            c.pool.evict_tokens(
                0, head_dim=64, block_tables_ptr=c.d_tables.data_ptr(),
                seq_lens_ptr=c.d_lens.data_ptr(), block_offsets_f16_ptr=c.d_offsets.data_ptr(),
                batch=2, max_blocks_per_seq=c.max_bps, budget=1000, sinks=4, recent=100,
                weights_in_ptr=w.data_ptr(), weights_out_ptr=w_out.data_ptr(),
                weights_row_stride=3000, positions_in_ptr=p.data_ptr(),
                positions_out_ptr=p_out.data_ptr(), next_positions_ptr=c.d_lens.data_ptr(),
                kept_lens_ptr=kept.data_ptr(), new_lens_ptr=new.data_ptr(),
                stream_ptr=stream.cuda_stream)

        return call, [w_out, p_out, new, c.region("k"), c.region("v")], c

    def decode(kv4):
        c = Cache([700, 1900], 2, 128, kv4=kv4, seed=2)
        made.append(c)
        c.fill_rows()
        q = torch.from_numpy(c.rng.standard_normal((2, 8, 128))).cuda().to(c.tdt)
        out = torch.zeros_like(q)
        w = torch.rand(2, 2, 1900, device="cuda")
        w_out = torch.zeros_like(w)
        args = dict(query_ptr=q.data_ptr(), out_ptr=out.data_ptr(),
                    block_tables_ptr=c.d_tables.data_ptr(), seq_lens_ptr=c.d_lens.data_ptr(),
                    block_offsets_f16_ptr=c.d_offsets.data_ptr(), batch=2, num_q_heads=8,
                    kv_heads=2, head_dim=128, block_size=16, max_blocks_per_seq=c.max_bps,
                    scale=0.1, dtype="bf16", stream_ptr=stream.cuda_stream)
        weights = dict(weights_in_ptr=w.data_ptr(), weights_out_ptr=w_out.data_ptr(),
                       weights_row_stride=1900)

        def call():
            if kv4:
                c.pool.kv4_paged_attn_decode(0, **args, **weights)
            else:
                c.pool.paged_attn_decode(0, **args)  # split, then merged

        return call, [out, w_out], (c, q, w)

    jobs = [evict(), decode(True), decode(False)]
    try:
        torch.cuda.synchronize()
        for call, _, _ in jobs:
            call()
        stream.synchronize()
        want = [[x.clone() for x in outs] for _, outs, _ in jobs]
        torch.cuda.synchronize()
        errors = []

        def work(call):
            try:
                for _ in range(400):
                    call()
            except Exception as err:  # noqa: BLE001
                errors.append(str(err))

        for _ in range(3):
            threads = [threading.Thread(target=work, args=(call,)) for call, _, _ in jobs]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            stream.synchronize()
            assert not errors
            for (_, outs, _), refs in zip(jobs, want):
                for got, ref in zip(outs, refs):
                    assert torch.equal(got, ref)
        assert all(c.pool.kernel_status() == 0 for c in made)
        assert np.array_equal(jobs[0][1][2].cpu().numpy(), [1000, 1000])
    finally:
        for c in made:
            c.close()


@pytest.mark.parametrize("many", [300, 4000])
def test_shared_prefix_decodes_of_two_threads(many):
    """Batches of different sizes, each thread on a stream of its own."""
    from test_shared_prefix_gpu import _build

    torch = torch_cuda()
    jobs, errors = [], []
    try:
        for batch in (4, many):
            wl = _build([2] * (batch // 2), [1] * (batch // 2), [20] * batch, hq=4, hkv=1)
            starts = torch.arange(0, batch + 1, 2, dtype=torch.int32, device="cuda")
            prefix = torch.full((batch // 2,), 16, dtype=torch.int32, device="cuda")
            out, stream = torch.zeros_like(wl.q), torch.cuda.Stream()

            def call(wl=wl, starts=starts, prefix=prefix, out=out, stream=stream):
                rc = wl.pool.lib.kcmm_paged_attn_decode_shared_prefix_bf16_on_stream(
                    wl.pool.handle, 0, wl.q.data_ptr(), out.data_ptr(), wl.d_tables.data_ptr(),
                    wl.d_seq_lens.data_ptr(), wl.d_offsets.data_ptr(), wl.batch, 4, 1, 128, 16,
                    wl.max_blocks_per_seq, wl.scale, starts.data_ptr(), prefix.data_ptr(),
                    wl.batch // 2, 2, stream.cuda_stream)
                if rc != 0:
                    raise RuntimeError(wl.pool.last_error())

            jobs.append((wl, call, out, stream))
        torch.cuda.synchronize()
        want = []
        for _, call, out, stream in jobs:
            call()
            stream.synchronize()
            want.append(out.clone())
        torch.cuda.synchronize()

        def work(call):
            try:
                for _ in range(2000):
                    call()
            except RuntimeError as err:
                errors.append(str(err))

        threads = [threading.Thread(target=work, args=(j[1],)) for j in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not errors
        for (wl, _, out, _), ref in zip(jobs, want):
            assert torch.equal(out, ref) and wl.pool.kernel_status() == 0
    finally:
        for wl, *_ in jobs:
            wl.close()
