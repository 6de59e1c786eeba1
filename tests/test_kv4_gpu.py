"""The 4-bit KV cache on the GPU through the C ABI: append, read-back and decode against the
definitions in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from kv_cases import Cache, check_decode, quantised, torch_cuda

pytestmark = pytest.mark.gpu


def equal_rows(got, want, dtype):
    """Bit equality: the read rounds the exact value once."""
    torch = torch_cuda()
    w = torch.from_numpy(want).cuda().to(torch.bfloat16 if dtype == "bf16" else torch.float16)
    return torch.equal(torch.nan_to_num(got, nan=123.0), torch.nan_to_num(w, nan=123.0))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hkv,d,bs", [(1, 32, 16), (8, 128, 16), (4, 64, 32), (3, 96, 16),
                                      (2, 256, 48), (5, 160, 16), (1, 224, 64), (2, 192, 16)])
def test_append_and_read_back(dtype, hkv, d, bs):
    c = Cache([3 * bs + 5, 1, bs], hkv, d, bs, kv4=True, dtype=dtype, seed=d + hkv)
    try:
        rows = c.fill_rows(k_amp=2.5, v_amp=0.1)
        for b, (k, v) in enumerate(rows):
            gk, gv = c.read(c.slots(b, np.arange(c.lens[b])))
            assert equal_rows(gk, k, dtype) and equal_rows(gv, v, dtype)
        assert int(c.status.item()) == 0
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_append_ties_zeros_and_extremes(dtype):
    """Values half way between codes, all-zero groups, the type's largest and smallest."""
    torch = torch_cuda()
    c = Cache([16], 1, 128, kv4=True, dtype=dtype)
    try:
        x = np.zeros((16, 1, 128))
        x[0, 0, :32] = np.arange(32) / 2 - 7       # scale 8.5/7: near ties
        x[0, 0, 32:64] = np.arange(32) % 15 - 7    # scale 1: the codes themselves
        x[1, 0, :32] = (np.arange(32) % 15 - 7) / 2  # scale 1/2
        x[1, 0, 32:64] = np.where(np.arange(32) == 0, 7, np.arange(32) % 7 - 3 + 0.5)  # ties
        x[2, 0, :] = float(torch.finfo(c.tdt).max) * (1 - 2 * (np.arange(128) % 2))
        x[3, 0, :] = float(torch.finfo(c.tdt).tiny) * (np.arange(128) % 5 - 2)
        x[4, 0, 5] = 1.0
        x[5, 0, :] = np.random.default_rng(1).standard_normal(128)
        x[6, 0, 40] = 2.0 ** -24 if dtype == "f16" else 2.0 ** -133  # the smallest subnormal
        t = torch.from_numpy(x).cuda().to(c.tdt)
        c.write(t, t.flip(0).contiguous(), c.slots(0, np.arange(16)))
        want = quantised(t.double().cpu().numpy())
        gk, gv = c.read(c.slots(0, np.arange(16)))
        assert equal_rows(gk, want, dtype) and equal_rows(gv, want[::-1].copy(), dtype)
    finally:
        c.close()


def test_append_non_finite_groups_read_as_nan():
    torch = torch_cuda()
    c = Cache([16], 2, 64, kv4=True)
    try:
        x = torch.randn(16, 2, 64, device="cuda").to(c.tdt)
        x[3, 0, 5], x[4, 1, 40], x[5, 0, 33] = float("nan"), float("inf"), float("-inf")
        c.write(x, x, c.slots(0, np.arange(16)))
        want = quantised(x.double().cpu().numpy())
        for got in c.read(c.slots(0, np.arange(16))):
            assert equal_rows(got, want, "bf16")
        assert np.isnan(want).sum() == 3 * 32
    finally:
        c.close()


def test_append_strides_skips_and_bad_slots():
    """Rows inside a fused QKV projection (odd offsets too), slots < 0 skipped, a block past
    the table or marked free reported in the status word and left alone."""
    torch = torch_cuda()
    for shift in (0, 1):
        c = Cache([40], 2, 64, kv4=True, seed=3)
        try:
            wide = torch.randn(40, 2 * 128 + 77, device="cuda").to(c.tdt)
            k, v = wide[:, shift:shift + 128], wide[:, 128 + shift:256 + shift]
            slots = c.slots(0, np.arange(40))
            slots[7] = -1
            c.write(k, v, slots, k_row_stride=wide.stride(0), v_row_stride=wide.stride(0))
            keep = np.arange(40) != 7
            kk, vv = (x.reshape(40, 2, 64)[torch.from_numpy(keep).cuda()].double().cpu().numpy()
                      for x in (k, v))
            out = torch.zeros(39, 500, device="cuda", dtype=c.tdt)
            c.read(slots[keep], k_dst_ptr=out.data_ptr() + 2 * shift, k_row_stride=500,
                   v_dst_ptr=out.data_ptr() + 2 * (200 + shift), v_row_stride=500)
            gk = out[:, shift:shift + 128].reshape(39, 2, 64)
            gv = out[:, 200 + shift:328 + shift].reshape(39, 2, 64)
            assert equal_rows(gk, quantised(kk), "bf16") and equal_rows(gv, quantised(vv), "bf16")
            assert int(out[:, 328 + shift:].abs().max()) == 0 and int(c.status.item()) == 0
            before = [c.region(x).clone() for x in "kv"]
            c.write(k[:1], v[:1], [len(c.offsets) * 16 + 3])
            assert int(c.status.item()) == 1
            c.status.zero_()
            valid = torch.zeros(len(c.offsets), dtype=torch.uint8, device="cuda")
            c.write(k[:1], v[:1], slots[:1], valid_blocks_ptr=valid.data_ptr())
            assert int(c.status.item()) == 2
            for x, old in zip("kv", before):
                assert torch.equal(c.region(x), old)
        finally:
            c.close()


def test_append_touches_only_its_slots():
    torch = torch_cuda()
    c = Cache([48], 3, 96, kv4=True, seed=5)
    try:
        c.fill_rows()
        want = [x.clone() for x in c.read(c.slots(0, np.arange(48)))]
        x = torch.randn(3, 3, 96, device="cuda").to(c.tdt)
        at = np.array([17, 2, 40])
        c.write(x, x, c.slots(0, at))
        new = torch.from_numpy(quantised(x.double().cpu().numpy())).cuda().to(c.tdt)
        for got, old in zip(c.read(c.slots(0, np.arange(48))), want):
            old[torch.from_numpy(at).cuda()] = new
            assert torch.equal(got, old)
    finally:
        c.close()


LENS = [0, 1, 15, 16, 17, 33, 160, 777]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("dtype,hq,hkv,d,bs", [
    ("bf16", 32, 8, 128, 16), ("f16", 16, 4, 64, 16), ("bf16", 8, 1, 128, 32),
    ("f16", 6, 6, 32, 16), ("bf16", 12, 4, 96, 16), ("bf16", 16, 1, 256, 16),
    ("f16", 14, 2, 160, 48), ("bf16", 40, 2, 128, 16), ("f16", 9, 1, 224, 16),
    ("bf16", 7, 3, 192, 16), ("f16", 8, 8, 256, 64)])
def test_decode(dtype, hq, hkv, d, bs, weights):
    """Lengths 0, 1, around a page and a split, uneven head groups, every head dim's kernel;
    slots past a context hold NaN scales."""
    torch = torch_cuda()
    c = Cache(LENS, hkv, d, bs, kv4=True, dtype=dtype, seed=hq + d)
    try:
        rows = c.fill_rows(k_amp=1.3)
        q = torch.from_numpy(c.rng.standard_normal((len(LENS), hq, d))).cuda().to(c.tdt)
        out = torch.full_like(q, float("nan"))
        kw = {}
        if weights:
            w_in = torch.rand(len(LENS), hkv, max(LENS) + 3, device="cuda")
            w_out = torch.full_like(w_in, -5.0)
            kw = dict(w_in=w_in, w_out=w_out)
        c.decode(q, d ** -0.5, out, **kw)
        check_decode(c, rows, q, out, d ** -0.5,
                     untouched=np.full((len(LENS), hq, d), np.nan), **kw)
        if weights:
            for b, n in enumerate(LENS):  # entries past the length are not written
                assert bool((w_out[b, :, n:] == -5.0).all())
        assert c.pool.kernel_status() == 0
    finally:
        c.close()


@pytest.mark.parametrize("amp", [1e-6, 1.0, 300.0])
def test_decode_scales_far_from_one(amp):
    """P carries V's scales in f16: tiny and large V, and a V whose loudest tokens come last
    (the normaliser has to rise) or have almost no weight."""
    torch = torch_cuda()
    n, hkv, d = 300, 2, 64
    c = Cache([n, n], hkv, d, kv4=True, dtype="bf16", seed=9)
    try:
        rows = []
        for b in range(2):
            k = c.rng.standard_normal((n, hkv, d))
            v = c.rng.standard_normal((n, hkv, d)) * amp
            v *= np.geomspace(1e-4, 1e4, n)[::1 if b == 0 else -1, None, None]
            tk, tv = (torch.from_numpy(x).cuda().to(c.tdt) for x in (k, v))
            c.write(tk, tv, c.slots(b, np.arange(n)))
            rows.append(tuple(quantised(x.double().cpu().numpy()) for x in (tk, tv)))
        q = torch.from_numpy(c.rng.standard_normal((2, 8, d)) * 6).cuda().to(c.tdt)
        out = c.decode(q, d ** -0.5, torch.zeros_like(q))
        check_decode(c, rows, q, out, d ** -0.5)
    finally:
        c.close()


@pytest.mark.parametrize("factor", [1e-20, 1e-3, 1e4, 1e18])
def test_decode_queries_of_any_magnitude(factor):
    """q goes through f16 scaled by its own power of two; one head is all zero."""
    torch = torch_cuda()
    c = Cache([100], 1, 128, kv4=True, seed=4)
    try:
        rows = c.fill_rows()
        q = torch.from_numpy(c.rng.standard_normal((1, 5, 128)) * factor).cuda().to(c.tdt)
        q[0, 3] = 0
        out = c.decode(q, 128 ** -0.5 / factor, torch.zeros_like(q))
        check_decode(c, rows, q, out, 128 ** -0.5 / factor)
    finally:
        c.close()


def test_decode_strides_and_streams():
    """q and out as views of wider buffers, a wider block table, on a stream of the caller's."""
    torch = torch_cuda()
    for shift in (0, 3):
        c = Cache([70, 5, 200], 2, 64, kv4=True, dtype="f16", seed=6)
        try:
            rows = c.fill_rows()
            wide = torch.from_numpy(c.rng.standard_normal((3, 9, 80))).cuda().to(c.tdt)
            q = wide[:, :8, shift:shift + 64]
            obuf = torch.zeros(3, 10, 72, device="cuda", dtype=c.tdt)
            tables = torch.zeros(3, c.max_bps + 5, dtype=torch.int32, device="cuda")
            tables[:, :c.max_bps] = c.d_tables
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                c.decode(q, 0.125, obuf[:, 1:9, 3:67], q_stride_token=q.stride(0),
                         q_stride_head=q.stride(1), out_stride_token=obuf.stride(0),
                         out_stride_head=obuf.stride(1), block_tables_ptr=tables.data_ptr(),
                         block_tables_row_stride=tables.stride(0))
            check_decode(c, rows, q, obuf[:, 1:9, 3:67], 0.125)
            assert float(obuf[:, 0].abs().max()) == 0 and float(obuf[:, :, :3].abs().max()) == 0
        finally:
            c.close()


def test_decode_weights_rows_shorter_than_the_context_and_in_place():
    torch = torch_cuda()
    c = Cache([100, 20], 2, 64, kv4=True, seed=8)
    try:
        rows = c.fill_rows()
        q = torch.from_numpy(c.rng.standard_normal((2, 4, 64))).cuda().to(c.tdt)
        w = torch.rand(2, 2, 64, device="cuda")
        before = w.clone()
        out = c.decode(q, 0.125, torch.zeros_like(q), w_in=w, w_out=w)
        check_decode(c, rows, q, out, 0.125, w_in=before, w_out=w)
    finally:
        c.close()


def test_decode_long_context_many_splits():
    torch = torch_cuda()
    c = Cache([20011, 4097], 1, 128, kv4=True, seed=12)
    try:
        rows = c.fill_rows(k_amp=1.5)
        q = torch.from_numpy(c.rng.standard_normal((2, 8, 128))).cuda().to(c.tdt)
        w_in = torch.rand(2, 1, 20011, device="cuda")
        w_out = torch.zeros_like(w_in)
        out = c.decode(q, 128 ** -0.5, torch.zeros_like(q), w_in=w_in, w_out=w_out)
        check_decode(c, rows, q, out, 128 ** -0.5, w_in=w_in, w_out=w_out)
    finally:
        c.close()


def test_decode_nan_rows_stay_in_their_sequence():
    """A NaN in one sequence's live K or V reaches that sequence's heads alone."""
    torch = torch_cuda()
    c = Cache([50, 50, 50], 1, 64, kv4=True, seed=13)
    try:
        rows = c.fill_rows()
        x = torch.randn(1, 1, 64, device="cuda").to(c.tdt)
        bad = x.clone()
        bad[0, 0, 3] = float("nan")
        c.write(bad, x, c.slots(0, [10]))
        c.write(x, bad, c.slots(2, [49]))
        q = torch.from_numpy(c.rng.standard_normal((3, 4, 64))).cuda().to(c.tdt)
        out = c.decode(q, 0.125, torch.zeros_like(q))
        assert bool(torch.isnan(out[0]).all())
        assert bool(torch.isnan(out[2, :, :32]).all()) and not bool(torch.isnan(out[2, :, 32:]).any())
        got = out[1:2].double().cpu().numpy()
        from kv_cases import attention
        ref, mass, _ = attention(q[1].double().cpu().numpy(), *rows[1], 0.125)
        assert (np.abs(got[0] - ref) <= 1.25 * 2.0 ** -11 * mass + 2.0 ** -8 * np.abs(ref)).all()
    finally:
        c.close()


def test_bad_block_is_reported():
    torch = torch_cuda()
    c = Cache([40], 1, 64, kv4=True, seed=14)
    try:
        c.fill_rows()
        c.d_tables[0, 1] = -1
        q = torch.randn(1, 4, 64, device="cuda").to(c.tdt)
        c.decode(q, 0.125, torch.zeros_like(q))
        assert c.pool.kernel_status() == 2
        assert c.pool.kernel_status() == 0
    finally:
        c.close()


def append_and_read_long_chunk(dtype, hkv, d, bs, first, n):
    torch = torch_cuda()
    c = Cache([n + first], hkv, d, bs, kv4=True, dtype=dtype, seed=d)
    try:
        x = c.rng.standard_normal((2, n, hkv, d))
        x *= np.geomspace(1e-7 if dtype == "f16" else 1e-37, 1e4, n)[None, :, None, None]
        x[0, 100] = np.round(x[0, 100] / x[0, 100].max() * 14) / 2  # ties
        x[1, 200, 0, 5], x[0, 300, 0, 7] = np.nan, np.inf
        tk, tv = (torch.from_numpy(y).cuda().to(c.tdt) for y in x)
        slots = c.slots(0, first + np.arange(n))
        skipped = np.array([3, 40, 777])
        at = slots.copy()
        at[skipped] = -1
        c.write(tk, tv, at)
        got = c.read(slots)
        keep = np.setdiff1d(np.arange(n), skipped)
        kt = torch.from_numpy(keep).cuda()
        for g, y in zip(got, (tk, tv)):
            assert equal_rows(g[kt], quantised(y.double().cpu().numpy())[keep], dtype)
            assert bool(torch.isnan(g[torch.from_numpy(skipped).cuda()]).all())  # NaN bits as made
        assert int(c.status.item()) == 0
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hkv,d,bs,first", [(2, 128, 16, 0), (3, 64, 32, 16), (1, 96, 48, 32),
                                            (2, 256, 16, 5), (1, 32, 16, 0), (5, 160, 64, 1)])
def test_append_and_read_long_chunks(dtype, hkv, d, bs, first):
    """Chunks of many rows: whole units, ends that are not, chunks that start inside a unit,
    skipped rows among them; magnitudes from the smallest to the largest."""
    append_and_read_long_chunk(dtype, hkv, d, bs, first, 1200)


@pytest.mark.parametrize("hkv,d,bs,first,n", [(8, 128, 16, 5, 1900), (12, 64, 32, 16, 1303),
                                              (3, 96, 48, 32, 4100), (1, 32, 16, 0, 12001),
                                              (16, 256, 16, 0, 2 * 777)])
def test_append_and_read_chunks_of_whole_units(hkv, d, bs, first, n):
    """The same where the rows are enough for tiles of a whole unit."""
    for dtype in ("bf16", "f16"):
        append_and_read_long_chunk(dtype, hkv, d, bs, first, n)


@pytest.mark.parametrize("hq,hkv,d", [(320, 320, 32), (700, 700, 32), (128, 2, 64), (96, 96, 256)])
def test_decode_many_heads(hq, hkv, d):
    """More kv heads, and tiles of a kv head's query heads, than CTAs that run at once."""
    torch = torch_cuda()
    c = Cache(LENS, hkv, d, kv4=True, seed=hq + d)
    try:
        rows = c.fill_rows(k_amp=1.3)
        q = torch.from_numpy(c.rng.standard_normal((len(LENS), hq, d))).cuda().to(c.tdt)
        out = torch.full_like(q, float("nan"))
        c.decode(q, d ** -0.5, out)
        check_decode(c, rows, q, out, d ** -0.5, untouched=np.full((len(LENS), hq, d), np.nan))
        assert c.pool.kernel_status() == 0
    finally:
        c.close()


@pytest.mark.parametrize("dtype,hq,hkv,d,n,most", [("bf16", 32, 8, 128, 900, 40),
                                                   ("f16", 8, 1, 64, 3000, 90),
                                                   ("bf16", 6, 2, 256, 500, 70)])
def test_decode_many_sequences_a_cta(dtype, hq, hkv, d, n, most):
    """CTAs that take several short sequences one after another reuse their copy buffers
    between them: every output right, and the same bits each time."""
    torch = torch_cuda()
    lens = np.random.default_rng(n).integers(0, most, n)
    c = Cache(lens, hkv, d, kv4=True, dtype=dtype, seed=n)
    try:
        total = len(c.offsets) * c.bs
        x = [torch.from_numpy(c.rng.standard_normal((total, hkv, d)).astype(np.float32)).cuda().to(
            c.tdt) for _ in "kv"]
        c.write(*x, np.arange(total))
        hk, hv = (quantised(y.double().cpu().numpy()) for y in x)
        rows = [(hk[s], hv[s]) for s in (c.slots(b, np.arange(m)) for b, m in enumerate(lens))]
        q = torch.from_numpy(c.rng.standard_normal((n, hq, d))).cuda().to(c.tdt)
        first = c.decode(q, d ** -0.5, torch.zeros_like(q))
        check_decode(c, rows, q, first, d ** -0.5, untouched=np.zeros((n, hq, d)))
        for _ in range(20):
            assert torch.equal(c.decode(q, d ** -0.5, torch.zeros_like(q)), first)
        assert c.pool.kernel_status() == 0
    finally:
        c.close()


@pytest.mark.parametrize("dtype,apart", [("bf16", 12), ("bf16", 20), ("bf16", 24), ("bf16", 90),
                                         ("f16", 12), ("f16", 20), ("f16", 24)])
def test_decode_groups_far_apart(dtype, apart):
    """A quiet group of V beside one 2^apart louder: output dims do not depend on each other,
    so each is held to its own sum of p |v|."""
    torch = torch_cuda()
    n, hkv, d = 300, 2, 128
    c = Cache([n, 40, 1], hkv, d, kv4=True, dtype=dtype, seed=apart)
    try:
        rows = []
        for b, m in enumerate(c.lens):
            k = c.rng.standard_normal((m, hkv, d))
            v = np.clip(c.rng.standard_normal((m, hkv, d)), -3, 3)
            v[..., :32] *= 2.0 ** (apart if dtype == "bf16" else 12)
            v[..., 96:] *= 2.0 ** (0 if dtype == "bf16" else 12 - apart)
            tk, tv = (torch.from_numpy(x).cuda().to(c.tdt) for x in (k, v))
            c.write(tk, tv, c.slots(b, np.arange(m)))
            rows.append(tuple(quantised(x.double().cpu().numpy()) for x in (tk, tv)))
        q = torch.from_numpy(c.rng.standard_normal((3, 8, d))).cuda().to(c.tdt)
        out = c.decode(q, d ** -0.5, torch.zeros_like(q))
        check_decode(c, rows, q, out, d ** -0.5)
    finally:
        c.close()


@pytest.mark.parametrize("at", [0, 150, 299])
@pytest.mark.parametrize("low,loud", [(20, 12), (40, 24), (60, 50), (30, 30)])
def test_decode_loud_token_of_little_weight(at, low, loud):
    """One token of probability near 2^-low whose V is 2^loud times the others': it counts for
    its share, and the others for theirs."""
    torch = torch_cuda()
    n, d = 300, 64
    c = Cache([n], 1, d, kv4=True, seed=at + low)
    try:
        k, v = c.rng.standard_normal((2, n, 1, d))
        direction = np.where(np.arange(d) % 2, 1.0, -1.0)
        k[at] = -direction * (low * np.log(2) / d)
        v[at] *= 2.0 ** loud
        tk, tv = (torch.from_numpy(x).cuda().to(c.tdt) for x in (k, v))
        c.write(tk, tv, c.slots(0, np.arange(n)))
        rows = [tuple(quantised(x.double().cpu().numpy()) for x in (tk, tv))]
        q = direction + 0.05 * c.rng.standard_normal((1, 6, d))
        q = torch.from_numpy(q).cuda().to(c.tdt)
        out = c.decode(q, 1.0, torch.zeros_like(q))
        check_decode(c, rows, q, out, 1.0)
    finally:
        c.close()


@pytest.mark.parametrize("dtype,apart", [("bf16", 12), ("bf16", 24), ("bf16", 40), ("f16", 12),
                                         ("f16", 20)])
def test_decode_queries_and_keys_far_apart(dtype, apart):
    """Dims where the query is small and the keys are large count like the others."""
    torch = torch_cuda()
    n, hkv, d = 300, 2, 128
    c = Cache([n, 33], hkv, d, kv4=True, dtype=dtype, seed=apart)
    try:
        low = np.where(np.arange(d) < 64, 2.0 ** -apart, 1.0) * (2.0 ** 8 if dtype == "f16" else 1)
        rows = []
        for b, m in enumerate(c.lens):
            k = c.rng.standard_normal((m, hkv, d)) / low
            v = c.rng.standard_normal((m, hkv, d))
            tk, tv = (torch.from_numpy(x).cuda().to(c.tdt) for x in (k, v))
            c.write(tk, tv, c.slots(b, np.arange(m)))
            rows.append(tuple(quantised(x.double().cpu().numpy()) for x in (tk, tv)))
        q = torch.from_numpy(c.rng.standard_normal((2, 8, d)) * low).cuda().to(c.tdt)
        out = c.decode(q, d ** -0.5, torch.zeros_like(q))
        check_decode(c, rows, q, out, d ** -0.5)
    finally:
        c.close()


@pytest.mark.parametrize("n", [1, 2, 300, 5000])
def test_decode_values_near_the_largest(n):
    """bf16 values near the type's largest: their weighted mean is finite, their sum is not."""
    torch = torch_cuda()
    d = 64
    c = Cache([n], 1, d, kv4=True, seed=n)
    try:
        k, v = c.rng.standard_normal((2, n, 1, d))
        v[..., :32] = 2e38 * (1 + 0.2 * c.rng.random((n, 1, 32)))
        v[..., 16:32] *= -1
        tk, tv = (torch.from_numpy(x).cuda().to(c.tdt) for x in (k, v))
        c.write(tk, tv, c.slots(0, np.arange(n)))
        rows = [tuple(quantised(x.double().cpu().numpy()) for x in (tk, tv))]
        q = torch.from_numpy(0.3 * c.rng.standard_normal((1, 4, d))).cuda().to(c.tdt)
        out = c.decode(q, d ** -0.5, torch.zeros_like(q))
        assert bool(torch.isfinite(out).all())
        check_decode(c, rows, q, out, d ** -0.5)
    finally:
        c.close()
