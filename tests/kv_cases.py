"""Shared by the GPU tests of the 4-bit cache, the accumulated attention weights and the
eviction: a paged cache whose pages start as NaN bits, and the operators in 64 bits."""
from __future__ import annotations

import numpy as np


def torch_cuda():
    import pytest
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def bf16(x):
    """float64 -> bf16 -> float64, ties to even (no input here lies near a tie of float32)."""
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16).double().numpy()


def quantised(x):
    """The values a 4-bit cache holds for rows x [..., D], from the definition in 64 bits."""
    g = np.asarray(x, np.float64).reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    bad = ~np.isfinite(g).all(-1, keepdims=True)
    g = np.where(bad, 0.0, g)
    s = bf16(np.abs(g).max(-1, keepdims=True) / 7)
    c = np.where(s > 0, np.clip(np.rint(g / np.where(s > 0, s, 1)), -7, 7), 0)
    return np.where(bad, np.nan, c * s).reshape(x.shape)


def attention(q, k, v, scale):
    """One sequence: q [hq, D], k / v [n, hkv, D] -> out [hq, D], sum_t p |v| [hq, D] and the
    softmax weights summed over each kv head's query heads [hkv, n]."""
    hq, hkv, n = q.shape[0], k.shape[1], k.shape[0]
    kvh = np.arange(hq) * hkv // hq
    s = np.einsum("hd,nhd->hn", q, k[:, kvh]) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    w = np.zeros((hkv, n))
    np.add.at(w, kvh, p)
    return (np.einsum("hn,nhd->hd", p, v[:, kvh]),
            np.einsum("hn,nhd->hd", p, np.abs(v[:, kvh])), w)


class Cache:
    """A one-layer pool with a random block table per sequence; every byte of its pages is
    set before the rows are written, so that what a kernel reads past a context is NaN."""

    def __init__(self, lens, hkv, d, bs=16, kv4=False, dtype="bf16", seed=0, extra_blocks=2,
                 max_bps=None, fill=0xFF):
        torch = torch_cuda()
        from lattice_b200 import kcmm, workloads

        self.lens, self.hkv, self.d, self.bs, self.kv4, self.dtype = lens, hkv, d, bs, kv4, dtype
        self.tdt = torch.bfloat16 if dtype == "bf16" else torch.float16
        self.rng = np.random.default_rng(seed)
        self.row = kcmm.kv4_row_elems(d) if kv4 else d
        self.max_bps = max_bps or max(1, max(-(-int(n) // bs) for n in lens))
        need = [max(1, -(-int(n) // bs)) for n in lens]
        total = sum(need) + extra_blocks
        self.pool = workloads.library().create_pool(kcmm.make_config(
            num_layers=1, kv_heads=hkv, head_dim=self.row, max_batch=1, max_seq_len=total * bs,
            block_size=bs))
        ids = np.array(self.pool.alloc_blocks(total), np.int64)
        self.rng.shuffle(ids)
        self.tables = np.full((len(lens), self.max_bps), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = ids[at:at + n]
            at += n
        self.offsets = np.array(self.pool.all_block_offsets_f16(), np.uint64).astype(np.int64)
        self.d_offsets = torch.from_numpy(self.offsets).cuda()
        self.d_tables = torch.from_numpy(self.tables).cuda()
        self.d_lens = torch.from_numpy(np.asarray(lens, np.int32)).cuda()
        self.region_elems = int(self.offsets.max()) + self.row * hkv * bs
        for kind in "kv":
            self.region(kind).fill_(-1 if fill == 0xFF else fill)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def region(self, kind):
        """The pages as 16-bit words."""
        torch = torch_cuda()
        base = self.pool.va_k(0) if kind == "k" else self.pool.va_v(0)

        class _View:
            __cuda_array_interface__ = {"shape": (self.region_elems,), "typestr": "<i2",
                                        "data": (base, False), "version": 3}

        return torch.as_tensor(_View(), device="cuda")

    def slots(self, b, tokens):
        t = np.asarray(tokens, np.int64)
        return self.tables[b, t // self.bs].astype(np.int64) * self.bs + t % self.bs

    def fill_rows(self, k_amp=1.0, v_amp=1.0):
        """Random rows for every sequence, written through the library; returns, per
        sequence, the values the cache holds in float64 ([n, hkv, D] K and V)."""
        torch = torch_cuda()
        out = []
        for b, n in enumerate(int(x) for x in self.lens):
            k = self.rng.standard_normal((n, self.hkv, self.d)) * k_amp
            v = self.rng.standard_normal((n, self.hkv, self.d)) * v_amp
            tk, tv = (torch.from_numpy(x).cuda().to(self.tdt) for x in (k, v))
            if n:
                self.write(tk, tv, self.slots(b, np.arange(n)))
            hk, hv = (x.double().cpu().numpy() for x in (tk, tv))
            out.append((quantised(hk), quantised(hv)) if self.kv4 else (hk, hv))
        return out

    def write(self, tk, tv, slots, **kw):
        torch = torch_cuda()
        ds = torch.from_numpy(np.asarray(slots, np.int64)).cuda()
        args = dict(slot_mapping_ptr=ds.data_ptr(), block_offsets_f16_ptr=self.d_offsets.data_ptr(),
                    block_offsets_f16_len=len(self.offsets), k_src_ptr=tk.data_ptr(),
                    v_src_ptr=tv.data_ptr(), status_ptr=self.status.data_ptr(),
                    stream_ptr=torch.cuda.current_stream().cuda_stream)
        args.update(kw)
        if self.kv4:
            self.pool.kv4_append(0, num_tokens=len(slots), head_dim=self.d, dtype=self.dtype,
                                 **args)
        else:
            self.pool.append_kv_device_slots_on_stream(0, batch=len(slots), valid_blocks_ptr=0,
                                                       **args)
        torch.cuda.synchronize()

    def read(self, slots, **kw):
        """The rows of the slots in the cache's 16-bit type."""
        torch = torch_cuda()
        n = len(slots)
        ds = torch.from_numpy(np.asarray(slots, np.int64)).cuda()
        if not self.kv4:
            e = torch.from_numpy(self.offsets).cuda()[ds // self.bs] + (ds % self.bs) * (
                self.hkv * self.d)
            idx = e[:, None] + torch.arange(self.hkv * self.d, device="cuda")[None, :]
            return [self.region(x)[idx].view(self.tdt).view(n, self.hkv, self.d) for x in "kv"]
        k, v = (torch.zeros(n, self.hkv, self.d, dtype=self.tdt, device="cuda") for _ in "kv")
        args = dict(slot_mapping_ptr=ds.data_ptr(), block_offsets_f16_ptr=self.d_offsets.data_ptr(),
                    block_offsets_f16_len=len(self.offsets), num_tokens=n, head_dim=self.d,
                    k_dst_ptr=k.data_ptr(), v_dst_ptr=v.data_ptr(), dtype=self.dtype,
                    status_ptr=self.status.data_ptr(),
                    stream_ptr=torch.cuda.current_stream().cuda_stream)
        args.update(kw)
        self.pool.kv4_read(0, **args)
        torch.cuda.synchronize()
        return [k, v]

    def decode(self, q, scale, out, w_in=None, w_out=None, **kw):
        torch = torch_cuda()
        args = dict(query_ptr=q.data_ptr(), out_ptr=out.data_ptr(),
                    block_tables_ptr=self.d_tables.data_ptr(), seq_lens_ptr=self.d_lens.data_ptr(),
                    block_offsets_f16_ptr=self.d_offsets.data_ptr(), batch=len(self.lens),
                    num_q_heads=q.shape[1], kv_heads=self.hkv, head_dim=self.d,
                    block_size=self.bs, max_blocks_per_seq=self.max_bps, scale=scale,
                    dtype=self.dtype, stream_ptr=torch.cuda.current_stream().cuda_stream)
        if w_out is not None:
            args.update(weights_in_ptr=w_in.data_ptr(), weights_out_ptr=w_out.data_ptr(),
                        weights_row_stride=w_out.shape[2])
        args.update(kw)
        call = self.pool.kv4_paged_attn_decode if self.kv4 else self.pool.paged_attn_decode_weights
        call(0, **args)
        torch.cuda.synchronize()
        return out

    def close(self):
        self.pool.destroy()


def check_decode(cache, rows, q, out, scale, w_in=None, w_out=None, untouched=None):
    """out and the weights against 64 bits.

    The bound on an output is 2^-11 sum(p |v|) for P's rounding to f16 (P to 2^-17 or better
    in the 16-bit cache), a quarter of that for 32-bit scores and sums, and half a unit of the
    output's type; on a weight, 2^-14 of the step's weights (scores off by 2^-17 of at most
    some tens) and a unit of the 32-bit sum."""
    half = 2.0 ** (-8 if cache.dtype == "bf16" else -11)
    got, qd = out.double().cpu().numpy(), q.double().cpu().numpy()
    for b, n in enumerate(int(x) for x in cache.lens):
        if n == 0:
            if untouched is not None:
                assert np.array_equal(got[b], untouched[b], equal_nan=True)
            continue
        ref, mass, w = attention(qd[b], *rows[b], scale)
        bound = 1.25 * 2.0 ** -11 * mass + half * np.abs(ref) + 1e-7
        err = np.abs(got[b] - ref)
        assert (err <= bound).all(), (b, n, float((err - bound).max()), float(err.max()))
        if w_out is not None:
            m = min(n, w_out.shape[2])
            before = w_in[b].double().cpu().numpy()
            after = w_out[b].double().cpu().numpy()
            want = before[:, :m] + w[:, :m]
            err = np.abs(after[:, :m] - want)
            assert (err <= 2.0 ** -14 * w[:, :m] + 2.0 ** -23 * np.abs(want) + 1e-9).all(), (b, n)
