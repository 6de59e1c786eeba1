"""Eviction by accumulated attention weight, against the definition on the host."""
from __future__ import annotations

import numpy as np
import pytest

from kv_cases import Cache, attention, torch_cuda

pytestmark = pytest.mark.gpu


def plan(w, pos, n, nxt, budget, sinks, recent):
    """Source slot of every kept slot of one row ([min(n, budget)])."""
    m = min(n, budget)
    if n <= budget:
        return np.arange(n)
    held = (pos < sinks) | (pos >= nxt - recent)
    key = np.where(np.isnan(w[:n]), -np.inf, w[:n]).astype(np.float64)
    best = np.lexsort((np.arange(n), -key, ~held))[:m]
    kept = np.zeros(n, bool)
    kept[best] = True
    src = np.arange(m)
    src[~kept[:m]] = m + np.flatnonzero(kept[m:])
    return src


class Evict:
    def __init__(self, c, stride, kept=None, gap=0, seed=0):
        torch = torch_cuda()
        self.c, self.stride = c, stride
        B, H = len(c.lens), c.hkv
        rng = self.rng = np.random.default_rng(seed)
        self.w = (rng.random((B, H, stride)) ** 4).astype(np.float32)
        self.kept = np.zeros(B, np.int32) if kept is None else np.asarray(kept, np.int32)
        self.nxt = (np.asarray(c.lens) + gap).astype(np.int32)
        self.pos = np.zeros((B, H, stride), np.int32)
        for b in range(B):
            for h in range(H):
                k = int(self.kept[b])
                self.pos[b, h, :k] = rng.permutation(k + gap)[:k]
        self.torch = torch

    def row_positions(self, b, h):
        n = int(self.c.lens[b])
        p = np.arange(n) + int(self.nxt[b]) - n
        k = min(int(self.kept[b]), n)
        p[:k] = self.pos[b, h, :k]
        return p

    def run(self, budget, sinks, recent, in_place=False, **kw):
        torch, c = self.torch, self.c
        t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
        self.d = dict(w=t(self.w), p=t(self.pos), kept=t(self.kept), nxt=t(self.nxt))
        self.w_out = self.d["w"] if in_place else torch.full_like(self.d["w"], -7.0)
        self.p_out = self.d["p"] if in_place else torch.full_like(self.d["p"], -7)
        self.new = torch.full_like(c.d_lens, -1)
        args = dict(head_dim=c.d, block_tables_ptr=c.d_tables.data_ptr(),
                    seq_lens_ptr=c.d_lens.data_ptr(),
                    block_offsets_f16_ptr=c.d_offsets.data_ptr(), batch=len(c.lens),
                    max_blocks_per_seq=c.max_bps, budget=budget, sinks=sinks, recent=recent,
                    weights_in_ptr=self.d["w"].data_ptr(), weights_out_ptr=self.w_out.data_ptr(),
                    weights_row_stride=self.stride, positions_in_ptr=self.d["p"].data_ptr(),
                    positions_out_ptr=self.p_out.data_ptr(),
                    next_positions_ptr=self.d["nxt"].data_ptr(),
                    kept_lens_ptr=self.d["kept"].data_ptr(), new_lens_ptr=self.new.data_ptr(),
                    cache_format=1 if c.kv4 else 0,
                    stream_ptr=torch.cuda.current_stream().cuda_stream)
        args.update(kw)
        c.pool.evict_tokens(0, **args)
        torch.cuda.synchronize()

    def check(self, budget, sinks, recent, before, in_place=False):
        torch, c = self.torch, self.c
        w_out, p_out = self.w_out.cpu().numpy(), self.p_out.cpu().numpy()
        assert self.new.tolist() == [min(int(n), budget) for n in c.lens]
        for b, n in enumerate(int(x) for x in c.lens):
            m = min(n, budget)
            after = c.read(c.slots(b, np.arange(n))) if n else []
            for h in range(c.hkv):
                pos = self.row_positions(b, h)
                src = plan(self.w[b, h], pos, n, int(self.nxt[b]), budget, sinks, recent)
                assert np.array_equal(p_out[b, h, :m], pos[src])
                assert np.array_equal(w_out[b, h, :m], self.w[b, h, src], equal_nan=True)
                assert (w_out[b, h, m:n] == 0).all()
                if not in_place:
                    assert (w_out[b, h, n:] == -7).all() and (p_out[b, h, m:] == -7).all()
                s = torch.from_numpy(src).cuda()
                for got, old in zip(after, before[b] if n else []):
                    assert torch.equal(got[:m, h], old[s, h])
                    assert torch.equal(got[m:, h], old[m:, h])  # rows past the budget stay
        assert c.pool.kernel_status() == 0

    def snapshot(self):
        c = self.c
        return [[x.clone() for x in c.read(c.slots(b, np.arange(n)))] if n else []
                for b, n in enumerate(c.lens)]


LENS = [0, 1, 40, 41, 100, 333, 64]


@pytest.mark.parametrize("kv4,dtype,hkv,d,bs", [
    (False, "bf16", 2, 128, 16), (False, "f16", 3, 64, 8), (False, "bf16", 1, 40, 16),
    (True, "bf16", 2, 128, 16), (True, "f16", 3, 96, 32), (True, "bf16", 1, 256, 16)])
@pytest.mark.parametrize("budget,sinks,recent", [(40, 4, 8), (40, 0, 0), (40, 10, 30), (1, 0, 1),
                                                 (300, 1, 64)])
def test_evict(kv4, dtype, hkv, d, bs, budget, sinks, recent):
    c = Cache(LENS, hkv, d, bs, kv4=kv4, dtype=dtype, seed=budget)
    try:
        c.fill_rows()
        e = Evict(c, 340, seed=budget + hkv)
        before = e.snapshot()
        e.run(budget, sinks, recent)
        e.check(budget, sinks, recent, before)
    finally:
        c.close()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kv4", [False, True])
def test_evict_again(kv4, in_place):
    """A cache that was cut before: stored positions out of order, and more of them than the
    new budget in one sequence."""
    c = Cache([90, 100, 57], 2, 64, kv4=kv4, seed=2)
    try:
        c.fill_rows()
        e = Evict(c, 128, kept=[60, 90, 57], gap=200, seed=4)
        before = e.snapshot()
        e.run(60, 3, 16, in_place=in_place)
        e.check(60, 3, 16, before, in_place=in_place)
    finally:
        c.close()


@pytest.mark.parametrize("n,budget", [(5000, 4999), (20000, 3000), (40003, 30000)])
def test_evict_long_rows(n, budget):
    """Rows that a cluster of CTAs shares, odd slices, weights with many ties."""
    c = Cache([n, 17], 1, 64, seed=n)
    try:
        c.fill_rows()
        e = Evict(c, n, seed=1)
        e.w = np.round(e.w * 50).astype(np.float32)
        before = e.snapshot()
        e.run(budget, 4, 128)
        e.check(budget, 4, 128, before)
    finally:
        c.close()


@pytest.mark.parametrize("n,hkv,budget", [(16999, 4, 16384), (33000, 1, 1024), (9001, 3, 4500),
                                          (8500, 40, 8000)])
def test_evict_long_rows_of_distinct_weights(n, hkv, budget):
    """The last few candidates for the threshold differ: they are ranked one against all."""
    c = Cache([n, n - 700], hkv, 64, seed=n)
    try:
        c.fill_rows()
        e = Evict(c, n, seed=3)
        before = e.snapshot()
        e.run(budget, 1, 200)
        e.check(budget, 1, 200, before)
    finally:
        c.close()


@pytest.mark.parametrize("kind", ["equal", "zeros", "special", "nan"])
def test_evict_ties_and_special_weights(kind):
    """All weights equal, signed zeros, infinities, negatives and NaN."""
    c = Cache([200, 200], 2, 64, seed=3)
    try:
        c.fill_rows()
        e = Evict(c, 200, seed=5)
        if kind == "equal":
            e.w[:] = 0.25
        elif kind == "zeros":
            e.w[:] = np.where(e.rng.random(e.w.shape) < 0.5, 0.0, -0.0)
        elif kind == "special":
            e.w[:] = e.rng.choice([np.inf, -np.inf, -1.0, 3e38, 1e-45, 0.0], e.w.shape)
        else:
            e.w[e.rng.random(e.w.shape) < 0.7] = np.nan
        before = e.snapshot()
        e.run(64, 4, 16)
        e.check(64, 4, 16, before)
    finally:
        c.close()


def test_evict_only_moves_what_has_to_move():
    """Slots below the budget that stay are not rewritten, and a bad table entry is reported."""
    c = Cache([64], 1, 64, seed=6)
    try:
        c.fill_rows()
        e = Evict(c, 64, seed=7)
        e.w[0, 0, :48] = 10  # the first 48 stay: nothing moves, whatever the tail's table says
        c.d_tables[0, 3] = -1
        before = e.snapshot()
        e.run(48, 0, 0)
        e.check(48, 0, 0, before)
        e.run(32, 0, 32)  # now the tail has to move
        assert c.pool.kernel_status() == 2
    finally:
        c.close()


def test_evict_more_tokens_than_the_arrays_hold():
    c = Cache([64, 20], 1, 64, seed=6)
    try:
        c.fill_rows()
        e = Evict(c, 32, seed=7)
        e.run(16, 0, 4)
        assert c.pool.kernel_status() == 4 and e.new.tolist() == [64, 16]
        assert bool((e.w_out[0] == -7).all())
    finally:
        c.close()


def test_evict_then_decode_and_truncate():
    """The path as used: decode with weights, evict, truncate, decode over what is left."""
    torch = torch_cuda()
    lens, hkv, d, budget = [150, 90], 2, 64, 64
    for kv4 in (False, True):
        c = Cache(lens, hkv, d, kv4=kv4, seed=11)
        try:
            rows = c.fill_rows()
            seqs = []
            for b, n in enumerate(lens):
                seqs.append(c.pool.register_sequence([int(x) for x in c.tables[b] if x >= 0]))
                c.pool.update_seq_len(seqs[b], n)
            q = torch.from_numpy(c.rng.standard_normal((2, 8, d))).cuda().to(c.tdt)
            w = torch.zeros(2, hkv, 160, device="cuda")
            c.decode(q, 0.3, torch.zeros_like(q), w_in=w, w_out=w)
            e = Evict(c, 160)
            e.w = w.cpu().numpy()
            e.run(budget, 2, 16)
            c.d_lens.copy_(e.new)
            c.lens = e.new.tolist()
            used = c.pool.blocks_in_use()
            for s in seqs:
                c.pool.truncate_sequence(s, budget)
                assert c.pool.seq_len(s) == budget and len(c.pool.block_table(s)) == 4
            assert c.pool.blocks_in_use() == used - (10 - 4) - (6 - 4)
            out = c.decode(q, 0.3, torch.zeros_like(q), w_in=e.w_out, w_out=e.w_out)
            for b in range(2):
                k, v = (np.stack([x[plan(e.w[b, h], np.arange(lens[b]), lens[b], lens[b], budget,
                                         2, 16), h] for h in range(hkv)], 1) for x in rows[b])
                ref, mass, _ = attention(q[b].double().cpu().numpy(), k, v, 0.3)
                err = np.abs(out[b].double().cpu().numpy() - ref)
                assert (err <= 1.25 * 2.0 ** -11 * mass + 2.0 ** -8 * np.abs(ref) + 1e-7).all()
        finally:
            c.close()


def test_evict_rows_past_the_keys_that_shared_memory_holds():
    """50,001 tokens a row, more rows than clusters fit: the keys are computed anew."""
    c = Cache([50001], 75, 8, seed=15)
    try:
        c.fill_rows()
        e = Evict(c, 50001, seed=16)
        before = e.snapshot()
        e.run(2000, 4, 100)
        e.check(2000, 4, 100, before)
    finally:
        c.close()


@pytest.mark.parametrize("lens,hkv,budget,kept", [
    ([90, 100, 57, 20], 16, 60, [60, 90, 57, 0]), ([17003, 16500], 4, 16384, [16384, 100]),
    ([9000] * 3, 60, 4000, [4000, 0, 9000])])
@pytest.mark.parametrize("shared", ["kept", "seq_lens", "nxt"])
def test_evict_new_lens_in_place(lens, hkv, budget, kept, shared):
    """new_lens in the array of the last eviction's, or of the lengths: every head and every CTA
    of a row sees the old values."""
    c = Cache(lens, hkv, 64, seed=21)
    try:
        c.fill_rows()
        e = Evict(c, max(lens), kept=kept, gap=300, seed=22)
        before = e.snapshot()
        torch = torch_cuda()
        array = {"kept": torch.from_numpy(e.kept).cuda(), "nxt": torch.from_numpy(e.nxt).cuda(),
                 "seq_lens": c.d_lens.clone()}[shared]
        name = {"kept": "kept_lens_ptr", "nxt": "next_positions_ptr",
                "seq_lens": "seq_lens_ptr"}[shared]
        e.run(budget, 3, 16, new_lens_ptr=array.data_ptr(), **{name: array.data_ptr()})
        assert bool((e.new == -1).all())
        e.new = array
        e.check(budget, 3, 16, before)
    finally:
        c.close()


def test_evict_from_two_threads():
    """Calls of different widths at the same time, each thread on a stream of its own."""
    import threading

    torch = torch_cuda()
    errors = []
    caches = [Cache([n], 80, 8, seed=n) for n in (4800, 45001)]
    try:
        evicts = []
        for c in caches:
            c.fill_rows()
            e = Evict(c, int(c.lens[0]), seed=1)
            e.run(600, 4, 100)
            want = [x.clone() for x in (e.w_out, e.p_out, e.new)]
            evicts.append((c, e, want))

        def work(c, e, want):
            stream = torch.cuda.Stream()
            try:
                for _ in range(1500):
                    c.pool.evict_tokens(
                        0, head_dim=8, block_tables_ptr=c.d_tables.data_ptr(),
                        seq_lens_ptr=c.d_lens.data_ptr(),
                        block_offsets_f16_ptr=c.d_offsets.data_ptr(), batch=1,
                        max_blocks_per_seq=c.max_bps, budget=600, sinks=4, recent=100,
                        weights_in_ptr=e.d["w"].data_ptr(), weights_out_ptr=e.w_out.data_ptr(),
                        weights_row_stride=e.stride, positions_in_ptr=e.d["p"].data_ptr(),
                        positions_out_ptr=e.p_out.data_ptr(),
                        next_positions_ptr=e.d["nxt"].data_ptr(),
                        kept_lens_ptr=e.d["kept"].data_ptr(), new_lens_ptr=e.new.data_ptr(),
                        stream_ptr=stream.cuda_stream)
                stream.synchronize()
            except Exception as err:  # noqa: BLE001
                errors.append(str(err))

        threads = [threading.Thread(target=work, args=x) for x in evicts]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors
        for c, e, want in evicts:
            for got, x in zip((e.w_out, e.p_out, e.new), want):
                assert torch.equal(got, x)
            assert c.pool.kernel_status() == 0
    finally:
        for c in caches:
            c.close()


@pytest.mark.parametrize("budget", [4096, (1 << 31) - 1])
def test_evict_budget_past_the_table(budget):
    """No row can be cut: every sequence keeps its slots, and no lists are made for the budget."""
    c = Cache([40, 700, 0, 64], 40, 64, seed=31)
    try:
        c.fill_rows()
        e = Evict(c, 700, kept=[40, 12, 0, 0], gap=20, seed=32)
        before = e.snapshot()
        e.run(budget, 3, 16)
        e.check(budget, 3, 16, before)
    finally:
        c.close()
