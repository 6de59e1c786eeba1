"""Beam selection and the beams' states, against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from kv_cases import Cache, torch_cuda

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pool():
    torch_cuda()
    from lattice_b200 import kcmm, workloads

    p = workloads.library().create_pool(kcmm.make_config(
        num_layers=2, kv_heads=1, head_dim=64, max_batch=8, max_seq_len=256))
    yield p
    p.destroy()


def reference(x, scores, n, finished=None, eos=0):
    """Scores and flat indices of the n best of one request, x [beams, vocab] in float64."""
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
    m = x.max(-1, keepdims=True)
    safe = np.where(np.isfinite(m), m, 0)
    lse = safe + np.log(np.maximum(np.exp(x - safe).sum(-1, keepdims=True), 1e-300))
    s = np.where(np.isneginf(x), -np.inf, x - lse + scores[:, None])
    for k in np.flatnonzero(finished if finished is not None else []):
        s[k] = -np.inf
        s[k, eos] = scores[k]
    s = np.where(np.isnan(s), -np.inf, s).reshape(-1)
    top = np.lexsort((np.arange(s.size), -s))[:n]
    return s[top], top


def select(pool, logits, scores, n, finished=None, eos=0, dtype="f32", **kw):
    torch = torch_cuda()
    B, K, V = logits.shape
    s = torch.full((B, n), 123.0, device="cuda")
    p, t = (torch.full((B, n), -1, dtype=torch.int32, device="cuda") for _ in "pt")
    args = dict(logits_ptr=logits.data_ptr(), dtype=dtype, scores_in_ptr=scores.data_ptr(),
                batch=B, beams=K, vocab=V, n_select=n, scores_out_ptr=s.data_ptr(),
                parents_out_ptr=p.data_ptr(), tokens_out_ptr=t.data_ptr(),
                stream_ptr=torch.cuda.current_stream().cuda_stream)
    if finished is not None:
        args.update(finished_ptr=finished.data_ptr(), eos_token=eos)
    args.update(kw)
    pool.beam_select(**args)
    torch.cuda.synchronize()
    return s.cpu().numpy(), p.cpu().numpy(), t.cpu().numpy()


def check(pool, logits, scores, n, finished=None, eos=0, dtype="f32", **kw):
    """Scores within 2^-20 of the magnitudes that enter them (a 32-bit log of a sum of
    2^17 terms and two subtractions); the choices equal, for inputs whose scores differ by
    more than that or are exactly equal."""
    s, p, t = select(pool, logits, scores, n, finished, eos, dtype, **kw)
    B, K, V = logits.shape
    for b in range(B):
        x = logits[b].double().cpu().numpy()
        sc = scores[b].double().cpu().numpy()
        want, top = reference(x, sc, n, None if finished is None else finished[b].cpu().numpy(), eos)
        assert np.array_equal(p[b], top // V) and np.array_equal(t[b], top % V), (b, s[b], want)
        fin = np.isfinite(want)
        assert np.array_equal(fin, np.isfinite(s[b]))
        bound = 2.0 ** -20 * (np.abs(want[fin]) + np.abs(x[np.isfinite(x)]).max(initial=0) + 20)
        assert (np.abs(s[b][fin] - want[fin]) <= bound).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 4, 31, 8), (2, 3, 1000, 6), (5, 4, 4096, 4),
                                     (1, 2, 8193, 64), (3, 1, 32001, 40), (2, 8, 50257, 16),
                                     (1, 4, 128256, 8), (2, 64, 700, 64)])
def test_select(pool, dtype, B, K, V, n):
    torch = torch_cuda()
    g = torch.Generator(device="cuda").manual_seed(B * 1000 + V + n)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    # distinct logits within a row, in all three types, would need more values than bf16 has:
    # equal logits of one row tie and go to the lower token
    logits = (2 * torch.randn(B, K, V, device="cuda", generator=g)).to(dt)
    scores = -5 * torch.rand(B, K, device="cuda", generator=g)
    check(pool, logits, scores, min(n, K * V), dtype=dtype)


@pytest.mark.parametrize("V,off,pad", [(1000, 1, 0), (5003, 3, 2), (8192, 7, 1), (9000, 0, 5)])
def test_unaligned_rows_and_strides(pool, V, off, pad):
    torch = torch_cuda()
    for dt, name in ((torch.bfloat16, "bf16"), (torch.float32, "f32")):
        g = torch.Generator(device="cuda").manual_seed(V)
        buf = torch.full((6 * (V + pad) + off,), float("inf"), device="cuda", dtype=dt)
        rows = buf[off:].as_strided((2, 3, V), (3 * (V + pad), V + pad, 1))
        rows.copy_(torch.randn(2, 3, V, device="cuda", generator=g) * 2)
        scores = -torch.rand(2, 3, device="cuda", generator=g)
        check(pool, rows, scores, 12, dtype=name, row_stride=V + pad)


def test_ties_go_to_the_lowest_index(pool):
    torch = torch_cuda()
    for V in (5, 300, 20000):
        logits = torch.zeros(2, 3, V, device="cuda")
        logits[1, :, V // 2:] = 1.0
        check(pool, logits, torch.full((2, 3), -2.0, device="cuda"), min(64, 3 * V))


@pytest.mark.parametrize("n", [1, 4, 8, 9])
def test_ties_of_few_selected(pool, n):
    """More equal logits than are ranked one against all, in part of a row, a row, all rows."""
    torch = torch_cuda()
    for V in (300, 20000, 70001):
        for dt, name in ((torch.bfloat16, "bf16"), (torch.float32, "f32")):
            logits = torch.zeros(3, 2, V, device="cuda", dtype=dt)
            logits[1, :, V // 2:] = 1.0
            logits[2, 0, ::2] = -float("inf")
            logits[2, 1, 5:] = -float("inf")
            check(pool, logits, torch.full((3, 2), -2.0, device="cuda"), n, dtype=name)


def test_beams_whose_candidates_crowd_one_warp(pool):
    """One warp of the ranking holds more candidates above the others' best than are ranked one
    against all."""
    torch = torch_cuda()
    g = torch.Generator(device="cuda").manual_seed(8)
    logits = torch.randn(1, 256, 50, device="cuda", generator=g)
    scores = -100 - torch.rand(1, 256, device="cuda", generator=g)
    scores[0, torch.arange(256, device="cuda") % 32 < 4] += 99
    check(pool, logits, scores, 8)


def test_masked_rows_and_specials(pool):
    """-inf over parts, whole rows and whole requests; NaN and +inf logits; beams of score
    -inf (the first step, where only beam 0 counts)."""
    torch = torch_cuda()
    inf = float("inf")
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(6, 4, 9001, device="cuda", generator=g) * 3
    scores = -torch.rand(6, 4, device="cuda", generator=g)
    x[0, :, 10:] = -inf
    x[1, 2] = -inf
    x[2] = -inf
    x[3, 0, ::3] = float("nan")
    x[3, 1] = float("nan")
    scores[4, 1:] = -inf
    scores[5, 2] = float("nan")
    check(pool, x, scores, 50)
    y = torch.randn(1, 2, 100, device="cuda", generator=g)
    y[0, 1, 77] = inf
    s, p, t = select(pool, y, torch.zeros(1, 2, device="cuda"), 1)
    assert (p[0, 0], t[0, 0]) == (1, 77) and s[0, 0] == 0


def test_finished_beams(pool):
    torch = torch_cuda()
    g = torch.Generator(device="cuda").manual_seed(4)
    for eos in (0, 2, 499):
        x = torch.randn(4, 3, 500, device="cuda", generator=g)
        x[0, 0] = float("nan")  # a finished beam's logits are not read
        scores = -3 * torch.rand(4, 3, device="cuda", generator=g)
        fin = torch.tensor([[1, 0, 0], [0, 1, 1], [1, 1, 1], [0, 0, 0]], dtype=torch.uint8,
                           device="cuda")
        check(pool, x, scores, 7, finished=fin, eos=eos)
        check(pool, x, scores, 1, finished=fin, eos=eos)


def test_gather(pool):
    torch = torch_cuda()
    g = torch.Generator(device="cuda").manual_seed(5)
    for B, K, n, cols in ((1, 1, 1, 1), (3, 4, 4, 37), (2, 2, 5, 64), (2, 8, 8, 70001)):
        src = torch.randint(0, 1 << 30, (B, K, cols), dtype=torch.int32, device="cuda", generator=g)
        par = torch.randint(0, K, (B, n), dtype=torch.int32, device="cuda", generator=g)
        tok = torch.randint(0, 99, (B, n), dtype=torch.int32, device="cuda", generator=g)
        want = torch.stack([src[b][par[b].long()] for b in range(B)])
        for at in (None, 0, cols // 2, cols - 1):
            dst = torch.full((B, n, cols), -1, dtype=torch.int32, device="cuda")
            kw = {} if at is None else dict(tokens_ptr=tok.data_ptr(), token_index=at)
            pool.beam_gather(src_ptr=src.data_ptr(), dst_ptr=dst.data_ptr(), row_bytes=4 * cols,
                             parents_ptr=par.data_ptr(), batch=B, beams=K, n_select=n,
                             stream_ptr=torch.cuda.current_stream().cuda_stream, **kw)
            ref = want.clone()
            if at is not None:
                ref[:, :, at] = tok
            assert torch.equal(dst, ref)
    par.fill_(8)
    dst.fill_(-1)
    pool.beam_gather(src_ptr=src.data_ptr(), dst_ptr=dst.data_ptr(), row_bytes=4 * cols,
                     parents_ptr=par.data_ptr(), batch=B, beams=K, n_select=n,
                     stream_ptr=torch.cuda.current_stream().cuda_stream)
    assert pool.kernel_status() == 4 and bool((dst == -1).all())


def test_reorder_copies_shared_tails():
    """Beams 0, 0, 2: both children of beam 0 keep its whole blocks and write their own
    partly filled one."""
    torch = torch_cuda()
    c = Cache([40, 40, 40], 1, 64, seed=1, extra_blocks=4)
    try:
        c.fill_rows()
        seqs = []
        for b in range(3):
            seqs.append(c.pool.register_sequence([int(x) for x in c.tables[b]]))
            c.pool.update_seq_len(seqs[b], 40)
        rows = [[x.clone() for x in c.read(c.slots(b, np.arange(40)))] for b in range(3)]
        used = c.pool.blocks_in_use()
        c.pool.reorder_sequences(seqs, [0, 0, 2],
                                 stream_ptr=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        new = [c.pool.block_table(s) for s in seqs]
        assert new[0][:2] == new[1][:2] and new[0][2] != new[1][2]
        assert new[2] == [int(x) for x in c.tables[2]]
        assert [c.pool.refcount(x) for x in new[0]] == [2, 2, 1]
        assert c.pool.blocks_in_use() == used - 3 + 1
        c.offsets = np.array(c.pool.all_block_offsets_f16(), np.uint64).astype(np.int64)
        for b, parent in enumerate([0, 0, 2]):
            c.tables[b] = new[b]
            for got, want in zip(c.read(c.slots(b, np.arange(40))), rows[parent]):
                assert torch.equal(got, want)
    finally:
        c.close()


TYPES = ["f32", "bf16", "f16"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 900, 20000, 70001])
@pytest.mark.parametrize("n", [1, 4, 8, 9, 40])
def test_ties_of_beams_without_a_score(pool, dtype, V, n):
    """Beams of score -inf or NaN over distinct logits: all their tokens tie, and the lowest come
    first, after every candidate that has a score."""
    torch = torch_cuda()
    g = torch.Generator(device="cuda").manual_seed(V + n)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    logits = (2 * torch.randn(4, 3, V, device="cuda", generator=g)).to(dt)
    scores = torch.full((4, 3), -float("inf"), device="cuda")
    scores[1] = float("nan")
    scores[2, 1] = -3.0  # one beam with 2 finite logits
    logits[2, 1] = -float("inf")
    logits[2, 1, [V // 3, V - 1]] = torch.tensor([1.0, 2.0], device="cuda", dtype=dt)
    scores[3, 1] = -1.0  # a finished beam between two without a score
    done = torch.zeros(4, 3, dtype=torch.uint8, device="cuda")
    done[3, 1] = 1
    check(pool, logits, scores, n, finished=done, eos=V // 2, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 20000, 70001])
@pytest.mark.parametrize("n", [1, 4, 8, 33])
def test_ties_by_rounding_of_the_score(pool, dtype, V, n):
    """At scores of 1e9 all log-probabilities round away (a unit is 64): every token of the best
    beams ties.  Units of 2^-10, at 1e4, join some neighbours and not others."""
    torch = torch_cuda()
    g = torch.Generator(device="cuda").manual_seed(V * 7 + n)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    for big in (1e9, 1e4):
        if big == 1e9:
            logits = (2 * torch.randn(3, 2, V, device="cuda", generator=g)).to(dt)
            logits[0, 1, V // 2] = float("nan")
            logits[1, 0, : V // 2] = -float("inf")
        else:  # levels 1/4 apart, and in 32 bits 4 values within 2^-14 of each: one score
            steps = torch.randint(0, 40, (3, 2, V), device="cuda", generator=g)
            logits = (0.25 * steps.float() - 12).to(dt)
            if dtype == "f32":
                logits += torch.randint(0, 4, (3, 2, V), device="cuda", generator=g) * 2.0 ** -16
        scores = torch.full((3, 2), -big, device="cuda")
        scores[2, 0] = -2 * big
        s, p, t = select(pool, logits, scores, n, dtype=dtype)
        for b in range(3):
            x = logits[b].double().cpu().numpy()
            x = np.where(np.isnan(x), -np.inf, x)
            m = x.max(-1, keepdims=True)
            sc = scores[b].double().cpu().numpy()[:, None]
            exact = x - (m + np.log(np.exp(x - m).sum(-1, keepdims=True))) + sc
            unit = np.spacing(np.float32(big)) * (1.0 if b < 2 else 2.0)
            fin = np.isfinite(exact)
            if big == 1e4:  # a score this near a rounding boundary says nothing
                off = np.abs(exact[fin] / unit - np.floor(exact[fin] / unit) - 0.5)
                if off.min() < 0.02:
                    continue
            score = exact.astype(np.float32).reshape(-1)
            top = np.lexsort((np.arange(score.size), -score))[:n]
            assert np.array_equal(s[b], score[top])
            assert np.array_equal(p[b], top // V) and np.array_equal(t[b], top % V)


def test_the_largest_vocabulary(pool):
    """2^31 - 1 logits: the last few have equal scores in 32 bits and distinct logits."""
    torch = torch_cuda()
    V, n = (1 << 31) - 1, 3
    logits = torch.full((1, 1, V), -float("inf"), device="cuda", dtype=torch.float16)
    at = torch.tensor([V - 1000, V - 900, V - 30, V - 20, V - 1], device="cuda")
    logits[0, 0, at] = torch.tensor([0.0, 1.0, 2.0, 3.0, 4.0], device="cuda", dtype=torch.float16)
    for big, want in ((-1e9, at[:n]), (-3.0, at.flip(0)[:n])):
        scores = torch.full((1, 1), big, device="cuda")
        s, p, t = select(pool, logits, scores, n, dtype="f16")
        assert np.array_equal(t[0], want.cpu().numpy()) and (p == 0).all()
