"""Attention over packed prompts on the GPU against the definition in 64 bits.

The bound on an output: half a unit of its type, half a unit for each weight's rounding to that
type (of sum p |v|), and 2^-12 of sum p |v| for 32-bit scores and sums (scores of some tens, off
by 2^-18 of that)."""
from __future__ import annotations

import numpy as np
import pytest

from kv_cases import torch_cuda

pytestmark = pytest.mark.gpu

HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def pool():
    torch_cuda()
    from lattice_b200 import kcmm, workloads

    p = workloads.library().create_pool(kcmm.make_config(
        num_layers=1, kv_heads=1, head_dim=64, max_batch=1, max_seq_len=64))
    yield p
    p.destroy()


def dt(torch, dtype):
    return torch.bfloat16 if dtype == "bf16" else torch.float16


def reference(q, k, v, scale, causal):
    """One sequence in float64: out and sum p |v|; zeros where a query sees no key."""
    import torch

    nq, hq, d = q.shape
    nk, hkv = k.shape[:2]
    if nk == 0 or nq == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    kvh = torch.arange(hq, device=q.device) // (hq // hkv)
    s = torch.einsum("ihd,jhd->hij", q, k[:, kvh]) * scale
    if causal:
        j, i = torch.arange(nk, device=q.device), torch.arange(nq, device=q.device)
        s = s.masked_fill(j[None, None, :] > i[None, :, None] + (nk - nq), -torch.inf)
    p = torch.softmax(s, -1)
    p = torch.where(torch.isneginf(s).all(-1, keepdim=True), torch.zeros_like(p), p)
    vv = v[:, kvh]
    return torch.einsum("hij,jhd->ihd", p, vv), torch.einsum("hij,jhd->ihd", p, vv.abs())


def starts(lens, first=0):
    return first + np.concatenate(([0], np.cumsum(lens)))


def call(pool, q, k, v, out, qs, ks, causal, dtype, scale, **kw):
    torch = torch_cuda()
    dq, dk = (torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in (qs, ks))
    args = dict(query_ptr=q.data_ptr(), q_stride_token=q.stride(0), q_stride_head=q.stride(1),
                key_ptr=k.data_ptr(), k_stride_token=k.stride(0), k_stride_head=k.stride(1),
                value_ptr=v.data_ptr(), v_stride_token=v.stride(0), v_stride_head=v.stride(1),
                out_ptr=out.data_ptr(), out_stride_token=out.stride(0),
                out_stride_head=out.stride(1), q_start_ptr=dq.data_ptr(),
                k_start_ptr=dk.data_ptr(), batch=len(qs) - 1, num_q_tokens=q.shape[0],
                num_k_tokens=k.shape[0], num_q_heads=q.shape[1], kv_heads=k.shape[1],
                head_dim=q.shape[2], scale=scale, causal=causal, dtype=dtype,
                stream_ptr=torch.cuda.current_stream().cuda_stream)
    args.update(kw)
    pool.prompt_attn(**args)
    torch.cuda.synchronize()
    return out


def check(q, k, v, out, qs, ks, causal, dtype, scale):
    worst = 0.0
    for b in range(len(qs) - 1):
        qb, got = q[qs[b]:qs[b + 1]].double(), out[qs[b]:qs[b + 1]].double()
        ref, mass = reference(qb, k[ks[b]:ks[b + 1]].double(), v[ks[b]:ks[b + 1]].double(), scale,
                              causal)
        bound = HALF[dtype] * (ref.abs() + mass) + 2.0 ** -12 * mass + 1e-7
        over = ((got - ref).abs() - bound)
        assert not torch_cuda().isnan(over).any(), (b, "NaN")
        if over.numel():
            worst = max(worst, float(over.max()))
            assert worst <= 0, (b, int(qs[b + 1] - qs[b]), int(ks[b + 1] - ks[b]), worst)


def inputs(nq, nk, hq, hkv, d, dtype, seed, q_amp=1.5):
    torch = torch_cuda()
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (torch.randn(n, h, d, device="cuda", generator=g) for n, h in
               ((nq, hq), (nk, hkv), (nk, hkv)))
    return [x.to(dt(torch, dtype)) for x in (q * q_amp, k, v)]


LENS = [1, 2, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 0, 300, 511]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,d,hq,hkv", [
    ("bf16", 128, 8, 2), ("f16", 128, 4, 4), ("bf16", 64, 16, 1), ("f16", 64, 6, 2),
    ("bf16", 80, 7, 1), ("f16", 72, 4, 2), ("bf16", 8, 2, 1), ("f16", 40, 3, 3),
    ("bf16", 192, 8, 2), ("f16", 136, 2, 1), ("bf16", 256, 4, 1), ("f16", 256, 3, 3)])
def test_ragged(pool, dtype, d, hq, hkv, causal):
    torch = torch_cuda()
    n = sum(LENS)
    q, k, v = inputs(n, n, hq, hkv, d, dtype, 1)
    qs = starts(LENS)
    out = call(pool, q, k, v, torch.full_like(q, 9.0), qs, qs, causal, dtype, d ** -0.5)
    check(q, k, v, out, qs, qs, causal, dtype, d ** -0.5)
    assert pool.kernel_status() == 0


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("group", [3, 5, 9, 12, 20, 28, 65, 96, 128, 130, 200])
def test_groups_that_do_not_divide_a_tile(pool, group, d):
    """Tiles of whole tokens with idle rows, groups whose tokens lie across tiles, and groups of
    more than a tile."""
    torch = torch_cuda()
    lens, past = [1, 43, 90, 0, 131], [0, 70, 3, 5, 200]
    total = [n + p for n, p in zip(lens, past)]
    q, k, v = inputs(sum(lens), sum(total), group, 1, d, "bf16", 18)
    qs, ks = starts(lens), starts(total)
    out = call(pool, q, k, v, torch.full_like(q, 9.0), qs, ks, True, "bf16", d ** -0.5)
    check(q, k, v, out, qs, ks, True, "bf16", d ** -0.5)
    assert pool.kernel_status() == 0


@pytest.mark.parametrize("dtype,d,hq,hkv", [("bf16", 128, 8, 2), ("f16", 64, 4, 4),
                                            ("bf16", 256, 5, 1), ("f16", 192, 4, 2)])
def test_pasts_and_rows_without_keys(pool, dtype, d, hq, hkv):
    """Chunks behind a past, single tokens, and sequences with fewer keys than queries, whose
    first queries see none."""
    torch = torch_cuda()
    nq = [1, 5, 130, 1, 64, 200, 3, 90, 1]
    nk = [700, 69, 131, 1, 1000, 77, 0, 1, 64]
    q, k, v = inputs(sum(nq), sum(nk), hq, hkv, d, dtype, 2)
    qs, ks = starts(nq), starts(nk)
    out = call(pool, q, k, v, torch.full_like(q, 9.0), qs, ks, True, dtype, d ** -0.5)
    check(q, k, v, out, qs, ks, True, dtype, d ** -0.5)
    b = nq.index(200)
    assert (out[qs[b]:qs[b] + 123] == 0).all() and (out[qs[6]:qs[7]] == 0).all()
    assert pool.kernel_status() == 0


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,d,hq,hkv", [("bf16", 128, 8, 2), ("f16", 64, 4, 4),
                                            ("bf16", 256, 5, 1), ("f16", 136, 4, 2)])
def test_few_queries_over_many_keys(pool, dtype, d, hq, hkv, causal):
    """So few items that their keys are cut into parts, whose sums are merged."""
    torch = torch_cuda()
    nq = [1, 7, 64, 0, 200, 1, 130]
    nk = [5000, 3001, 2100, 900, 4096, 1023, 8191]
    qs, ks = starts(nq), starts(nk)
    for seed, q_amp in ((15, 1.5), (16, 8.0)):  # flat rows, and peaked ones
        q, k, v = inputs(sum(nq), sum(nk), hq, hkv, d, dtype, seed, q_amp)
        out = call(pool, q, k, v, torch.full_like(q, 9.0), qs, ks, causal, dtype, d ** -0.5)
        check(q, k, v, out, qs, ks, causal, dtype, d ** -0.5)
        again = call(pool, q, k, v, torch.full_like(q, 9.0), qs, ks, causal, dtype, d ** -0.5)
        assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    assert pool.kernel_status() == 0


def test_parts_that_see_nothing(pool):
    """One sequence whose first queries see no key and the last many: of its tile's parts some
    give some rows nothing."""
    torch = torch_cuda()
    nq, nk = [1500, 40], [1400, 2000]
    qs, ks = starts(nq), starts(nk)
    q, k, v = inputs(sum(nq), sum(nk), 1, 1, 128, "bf16", 17)
    out = call(pool, q, k, v, torch.full_like(q, 9.0), qs, ks, True, "bf16", 0.09)
    check(q, k, v, out, qs, ks, True, "bf16", 0.09)
    assert (out[:100] == 0).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("bf16", 256)])
def test_strided_views_and_rows_outside(pool, dtype, d):
    """Views of a fused projection, heads outermost for k, out inside a larger tensor; rows in
    front of the first sequence and behind the last one are left as they were, and what they hold
    reaches nothing."""
    torch = torch_cuda()
    hq, hkv, lens = 8, 2, [70, 1, 190]
    n = sum(lens) + 16
    q0, k0, v0 = inputs(n, n, hq, hkv, d, dtype, 3)
    qkv = torch.cat((q0, k0, v0), 1)
    qs = starts(lens, 7)
    out_of = (np.arange(n) < qs[0]) | (np.arange(n) >= qs[-1])
    qkv[torch.from_numpy(out_of).cuda()] = float("nan")
    q, v = qkv[:, :hq], qkv[:, hq + hkv:]
    k = qkv[:, hq:hq + hkv].permute(1, 0, 2).contiguous().permute(1, 0, 2)
    big = torch.full((n, hq + 3, d + 8), 9.0, dtype=q.dtype, device="cuda")
    out = big[:, 1:1 + hq, :d]
    call(pool, q, k, v, out, qs, qs, True, dtype, d ** -0.5)
    check(q, k, v, out, qs, qs, True, dtype, d ** -0.5)
    rest = big.clone()
    rest[qs[0]:qs[-1], 1:1 + hq, :d] = 9.0
    assert (rest == 9.0).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("bf16", 192)])
def test_a_sequence_of_nan_leaves_its_neighbours(pool, dtype, d):
    torch = torch_cuda()
    lens = [65, 100, 30]
    q, k, v = inputs(sum(lens), sum(lens), 4, 2, d, dtype, 4)
    qs = starts(lens)
    for x in (k, v):
        x[qs[1]:qs[2]] = float("nan")
    out = call(pool, q, k, v, torch.zeros_like(q), qs, qs, True, dtype, d ** -0.5)
    assert torch.isnan(out[qs[1]:qs[2]]).all()
    k[qs[1]:qs[2]] = v[qs[1]:qs[2]] = 0
    out[qs[1]:qs[2]] = 0
    check(q, k, v, out, qs, qs, True, dtype, d ** -0.5)


@pytest.mark.parametrize("dtype,d,hq,hkv", [("bf16", 128, 8, 2), ("f16", 64, 4, 4),
                                            ("bf16", 256, 2, 1), ("f16", 80, 7, 1)])
@pytest.mark.parametrize("past", [0, 150, 2600])
def test_infinities_and_nan_reach_only_the_rows_that_see_them(pool, dtype, d, hq, hkv, past):
    """V with infinities and NaN, K with NaN, at tokens in the middle: no row in front of them
    changes by a bit; a row that sees an infinity of V has it in that column, one that sees both
    signs or a NaN has NaN there, one that sees a NaN of K is NaN."""
    torch = torch_cuda()
    nq = [300, 61, 520]
    nk = [n + past for n in nq]
    qs, ks = starts(nq), starts(nk)
    q, k, v = inputs(sum(nq), sum(nk), hq, hkv, d, dtype, 12)
    clean = call(pool, q, k, v, torch.zeros_like(q), qs, ks, True, dtype, d ** -0.5)
    bad = v.clone()
    marks = []  # sequence, key, kv head, column, value
    r = np.random.default_rng(13)
    for b in range(3):
        for _ in range(12):
            marks.append((b, int(r.integers(0, nk[b])), int(r.integers(hkv)), int(r.integers(d)),
                          [np.inf, -np.inf, np.nan][r.integers(3)]))
    marks += [(2, nk[2] - 1, 0, 3, np.nan), (2, nk[2] - 2, 0, 3, np.inf), (0, 0, 0, 1, np.inf)]
    want, odd = clean.clone(), torch.zeros(clean.shape, dtype=torch.bool, device="cuda")
    group = hq // hkv
    for b, j, h, c, x in marks:
        bad[ks[b] + j, h, c] = x
    for b, j, h, c, _ in set(marks):
        x = float(bad[ks[b] + j, h, c])
        first = max(0, j - (nk[b] - nq[b]))
        rows = want[qs[b] + first:qs[b + 1], h * group:(h + 1) * group, c]
        before = torch.isfinite(rows)
        rows.copy_(torch.where(before, torch.full_like(rows, x), rows + x))
        odd[qs[b] + first:qs[b + 1], h * group:(h + 1) * group, c] = True
    got = call(pool, q, k, bad, torch.zeros_like(q), qs, ks, True, dtype, d ** -0.5)
    assert torch.equal(got[~odd].view(torch.int16), clean[~odd].view(torch.int16))
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf])
    # K: the whole row
    for b, j in ((0, 200 + past), (1, 60 + past), (2, 300 + past)):
        k[ks[b] + j] = float("nan")
    got = call(pool, q, k, v, torch.zeros_like(q), qs, ks, True, dtype, d ** -0.5)
    for b, j in ((0, 200), (1, 60), (2, 300)):
        assert torch.equal(got[qs[b]:qs[b] + j].view(torch.int16),
                           clean[qs[b]:qs[b] + j].view(torch.int16))
        assert torch.isnan(got[qs[b] + j:qs[b + 1]]).all()
    assert pool.kernel_status() == 0


def test_infinite_rows_of_a_bidirectional_batch_stay_in_their_sequence(pool):
    torch = torch_cuda()
    lens = [100, 40, 77]
    q, k, v = inputs(sum(lens), sum(lens), 4, 4, 64, "bf16", 14)
    qs = starts(lens)
    v[qs[1] + 3, :, 5] = float("inf")
    out = call(pool, q, k, v, torch.zeros_like(q), qs, qs, False, "bf16", 0.125)
    assert torch.isinf(out[qs[1]:qs[2], :, 5]).all()
    v[qs[1] + 3, :, 5] = 0
    out[qs[1]:qs[2], :, 5] = 0
    keep = torch.ones(64, dtype=torch.bool)
    keep[5] = False
    for b in (0, 2):
        assert torch.isfinite(out[qs[b]:qs[b + 1]]).all()
    assert torch.isfinite(out[qs[1]:qs[2]][:, :, keep]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_peaked_rising_and_falling_scores(pool, dtype):
    """Rows whose maximum keeps rising (O is rescaled every step), falls, or sits on one key."""
    torch = torch_cuda()
    n, d = 700, 128
    q, k, v = inputs(n, n, 2, 1, d, dtype, 5)
    u = torch.ones(d, device="cuda", dtype=q.dtype) / d ** 0.5
    t = torch.arange(n, device="cuda", dtype=torch.float32)[:, None, None] / n
    qs = np.array([0, n])
    for ramp in (60 * t, 60 * (1 - t), 60 * (t * n % 97 == 5)):
        kk = (0.1 * k.float() + ramp * u.float()).to(k.dtype)
        qq = (0.1 * q.float() + 8 * u.float()).to(q.dtype)
        out = call(pool, qq, kk, v, torch.zeros_like(q), qs, qs, True, dtype, 0.3)
        check(qq, kk, v, out, qs, qs, True, dtype, 0.3)


def test_many_sequences(pool):
    """More sequences than a warp has lanes, empty ones among them, and more items than SMs."""
    torch = torch_cuda()
    r = np.random.default_rng(6)
    lens = r.integers(0, 40, 500)
    q, k, v = inputs(int(lens.sum()), int(lens.sum()), 4, 2, 64, "bf16", 6)
    qs = starts(lens)
    out = call(pool, q, k, v, torch.full_like(q, 9.0), qs, qs, True, "bf16", 0.125)
    check(q, k, v, out, qs, qs, True, "bf16", 0.125)
    assert pool.kernel_status() == 0


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("bad", [[0, 50, 40, 90], [0, 50, 90, 5000], [-3, 50, 90, 90]])
def test_malformed_starts_are_reported(pool, which, bad):
    """A descending, passing or negative start: nothing is read or written out of range."""
    torch = torch_cuda()
    good = np.array([0, 30, 60, 90])
    q, k, v = inputs(90, 90, 4, 2, 64, "bf16", 7)
    big = torch.full((90 + 64, 4, 64), 9.0, dtype=q.dtype, device="cuda")
    out = big[32:32 + 90]
    bad = np.array(bad)
    call(pool, q, k, v, out, *((bad, good) if which == "q" else (good, bad)), True, "bf16", 0.125)
    assert pool.kernel_status() == 4
    assert (big[:32] == 9.0).all() and (big[32 + 90:] == 9.0).all()


def test_malformed_starts_among_many(pool):
    """Sequences in front of the 32 that hold a malformed one are answered; those behind it, which
    overlap it here, are not."""
    torch = torch_cuda()
    lens = np.full(32, 5)
    q, k, v = inputs(260, 260, 4, 2, 64, "bf16", 8)
    good = starts(lens)
    bad = np.concatenate([good, np.tile([260, 160], 24)])
    out = call(pool, q, k, v, torch.full_like(q, 9.0), bad, bad, True, "bf16", 0.125)
    assert pool.kernel_status() == 4
    check(q[:160], k[:160], v[:160], out[:160], good, good, True, "bf16", 0.125)
    assert (out[160:] == 9.0).all()


def test_other_stream_and_graph(pool):
    """On a side stream, and captured into a graph that is replayed on new inputs."""
    torch = torch_cuda()
    lens = [200, 3, 1511]  # in parts
    qs = starts(lens)
    q, k, v = inputs(sum(lens), sum(lens), 8, 2, 128, "bf16", 8)
    out = torch.zeros_like(q)
    d_starts = torch.from_numpy(qs.astype(np.int32)).cuda()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call(pool, q, k, v, out, qs, qs, True, "bf16", 0.1)
    check(q, k, v, out, qs, qs, True, "bf16", 0.1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.prompt_attn(
            query_ptr=q.data_ptr(), key_ptr=k.data_ptr(), value_ptr=v.data_ptr(),
            out_ptr=out.data_ptr(), q_start_ptr=d_starts.data_ptr(),
            k_start_ptr=d_starts.data_ptr(), batch=3, num_q_tokens=q.shape[0],
            num_k_tokens=k.shape[0], num_q_heads=8, kv_heads=2, head_dim=128, scale=0.1,
            stream_ptr=torch.cuda.current_stream().cuda_stream)
    for seed in (9, 10):
        for x, y in zip((q, k, v), inputs(sum(lens), sum(lens), 8, 2, 128, "bf16", seed)):
            x.copy_(y)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        check(q, k, v, out, qs, qs, True, "bf16", 0.1)


def test_two_graphs_at_once(pool):
    """Two captured calls with keys in parts, replayed side by side: neither has the other's sums."""
    torch = torch_cuda()
    lens = [64, 5]
    qs, ks = starts(lens), starts([3000, 2500])
    sets, graphs, streams = [], [], []
    d_q, d_k = (torch.from_numpy(x.astype(np.int32)).cuda() for x in (qs, ks))
    for seed in (12, 13):
        q, k, v = inputs(69, 5500, 8, 1, 128, "bf16", seed)
        out = torch.zeros_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            pool.prompt_attn(
                query_ptr=q.data_ptr(), key_ptr=k.data_ptr(), value_ptr=v.data_ptr(),
                out_ptr=out.data_ptr(), q_start_ptr=d_q.data_ptr(), k_start_ptr=d_k.data_ptr(),
                batch=2, num_q_tokens=69, num_k_tokens=5500, num_q_heads=8, kv_heads=1,
                head_dim=128, scale=0.1, stream_ptr=torch.cuda.current_stream().cuda_stream)
        sets.append((q, k, v, out))
        graphs.append(g)
        streams.append(torch.cuda.Stream())
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for q, k, v, out in sets:
        check(q, k, v, out, qs, ks, True, "bf16", 0.1)
    assert pool.kernel_status() == 0


def test_same_bits_twice(pool):
    torch = torch_cuda()
    lens = [900, 40, 1300]
    qs = starts(lens)
    q, k, v = inputs(sum(lens), sum(lens), 8, 2, 128, "f16", 11)
    a = call(pool, q, k, v, torch.zeros_like(q), qs, qs, True, "f16", 0.1)
    b = call(pool, q, k, v, torch.zeros_like(q), qs, qs, True, "f16", 0.1)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))
