"""Rotation and append on the GPU, bit for bit against the definition: angles in 64 bits, their
cosines and sines rounded to 32, products and sums rounded to 32, results to 16.

A cosine of 64 bits that lies within its own error (2^-52) of where rounding to 32 bits turns
may round otherwise here than there; one in 2^27 does, and moves a result by at most one unit of
the 16-bit type.  No case below has so many angles."""
from __future__ import annotations

import numpy as np
import pytest

from kv_cases import Cache, quantised, torch_cuda

pytestmark = pytest.mark.gpu


def pair_axes(rot, sections, layout):
    n = len(sections)
    if n == 1:
        return np.zeros(rot // 2, np.int64)
    if layout == "sections":
        return np.repeat(np.arange(n), sections)
    i = np.arange(rot // 2)
    return np.where(i < n * np.array(sections)[i % n], i % n, 0)


def rotate(x, pos, inv_freq, rot, sections, mode, layout):
    """x a 16-bit tensor [t, h, d] on the CPU, pos int [axes, t] -> the rotated rows."""
    import torch

    axes = pair_axes(rot, sections, layout)
    angle = torch.from_numpy(pos[axes].T.astype(np.float64)) * inv_freq.double()
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    y = x.float()
    i = torch.arange(rot // 2)
    at, by = (i, i + rot // 2) if mode == "neox" else (2 * i, 2 * i + 1)
    a, b = y[..., at], y[..., by]
    out = y.clone()
    out[..., at] = a * c - b * s
    out[..., by] = b * c + a * s
    out = out.to(x.dtype)
    out[..., rot:] = x[..., rot:]
    return out


class Case:
    def __init__(self, tokens, hq, hkv, d, rot, *, mode="neox", layout="sections", sections=None,
                 dtype="bf16", kv4=False, seed=0, bs=16, pos=None, blocks=None):
        torch = torch_cuda()
        self.__dict__.update(tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, mode=mode,
                             layout=layout, dtype=dtype, kv4=kv4)
        self.sections = sections or [rot // 2]
        r = np.random.default_rng(seed)
        self.cache = Cache([blocks * bs if blocks else tokens + 3], hkv, d, bs=bs, kv4=kv4,
                           dtype=dtype, seed=seed)
        n_slots = self.cache.tables.shape[1] * bs
        where = r.permutation(n_slots)[:tokens] if tokens < 40 else np.arange(tokens)
        self.slots = self.cache.slots(0, where)
        self.pos = pos if pos is not None else r.integers(
            0, 1 << 17, (len(self.sections), tokens)).astype(np.int32)
        self.inv_freq = torch.from_numpy(
            (1e4 ** (-2.0 * np.arange(rot // 2) / rot)).astype(np.float32))
        tdt = torch.bfloat16 if dtype == "bf16" else torch.float16
        g = torch.Generator().manual_seed(seed)
        self.qkv = (3 * torch.randn(tokens, hq + 2 * hkv, d, generator=g)).to(tdt)
        self.want_q = rotate(self.qkv[:, :hq], self.pos, self.inv_freq, rot, self.sections, mode,
                             layout)
        self.want_k = rotate(self.qkv[:, hq:hq + hkv], self.pos, self.inv_freq, rot,
                             self.sections, mode, layout)
        self.v = self.qkv[:, hq + hkv:]
        self.dev = self.qkv.cuda()
        self.d_pos, self.d_freq = torch.from_numpy(self.pos).cuda(), self.inv_freq.cuda()
        self.d_slots = torch.from_numpy(self.slots).cuda()

    def rope(self, **kw):
        from lattice_b200 import kcmm

        return kcmm.make_rope(**{**dict(
            mode=self.mode, rotary_dim=self.rot, inv_freq_ptr=self.d_freq.data_ptr(),
            positions_ptr=self.d_pos.data_ptr(), sections=self.sections, layout=self.layout), **kw})

    def views(self, x):
        return x[:, :self.hq], x[:, self.hq:self.hq + self.hkv], x[:, self.hq + self.hkv:]

    def run(self, q, k, v, q_out, k_out=None, **kw):
        torch = torch_cuda()
        args = dict(rope=self.rope(), head_dim=self.d, num_q_heads=self.hq, q_ptr=q.data_ptr(),
                    q_stride_token=q.stride(0), q_stride_head=q.stride(1),
                    q_out_ptr=q_out.data_ptr(), q_out_stride_token=q_out.stride(0),
                    q_out_stride_head=q_out.stride(1), k_ptr=k.data_ptr(),
                    k_row_stride=k.stride(0), v_ptr=v.data_ptr(), v_row_stride=v.stride(0),
                    slot_mapping_ptr=self.d_slots.data_ptr(),
                    block_offsets_f16_ptr=self.cache.d_offsets.data_ptr(),
                    block_offsets_f16_len=len(self.cache.offsets), num_tokens=self.tokens,
                    cache_format=int(self.kv4), status_ptr=self.cache.status.data_ptr(),
                    dtype=self.dtype, stream_ptr=torch.cuda.current_stream().cuda_stream)
        if k_out is not None:
            args.update(k_out_ptr=k_out.data_ptr(), k_out_row_stride=k_out.stride(0))
        args.update(kw)
        self.cache.pool.rope_append(0, **args)
        torch.cuda.synchronize()

    def check_cache(self, written=None):
        """The written slots hold k' and v (or the values 4 bits give them)."""
        torch = torch_cuda()
        w = np.arange(self.tokens) if written is None else np.flatnonzero(written)
        got = self.cache.read(self.slots[w])
        for x, want in zip(got, (self.want_k[w], self.v[w])):
            if self.kv4:
                want = torch.from_numpy(quantised(want.double().numpy()) + 0.0).to(x.dtype)  # no -0
            assert same(x.cpu(), want)


def same(a, b):
    import torch

    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


SHAPES = [
    # tokens, hq, hkv, d, rot, mode, layout, sections, dtype
    (1, 8, 2, 128, 128, "neox", "sections", None, "bf16"),
    (7, 4, 4, 64, 32, "gptj", "sections", None, "f16"),
    (33, 6, 2, 128, 128, "neox", "sections", [16, 24, 24], "bf16"),
    (50, 4, 1, 128, 128, "neox", "interleaved", [24, 20, 20], "f16"),
    (64, 3, 3, 96, 64, "gptj", "interleaved", [12, 10, 10], "bf16"),
    (300, 32, 8, 128, 128, "neox", "sections", [22, 21, 21], "bf16"),
    (129, 2, 2, 256, 256, "neox", "interleaved", [64, 64], "f16"),
    (40, 8, 2, 64, 64, "neox", "sections", [8, 8, 8, 8], "bf16"),
]
SHAPES16 = [
    (5, 3, 1, 80, 80, "neox", "sections", [20, 10, 10], "bf16"),
    (9, 2, 2, 72, 72, "neox", "sections", None, "f16"),      # halves of 36: 8-byte accesses
    (6, 3, 3, 10, 6, "neox", "sections", [1, 1, 1], "bf16"),  # single values
    (6, 1, 2, 34, 34, "gptj", "interleaved", [9, 8], "f16"),
    (11, 5, 2, 128, 2, "neox", "sections", None, "bf16"),
    (3, 2, 1, 256, 250, "gptj", "sections", None, "f16"),
]


@pytest.mark.parametrize("kv4", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotates_and_appends(shape, kv4):
    """q and k as views of a projection, results beside them."""
    torch = torch_cuda()
    tokens, hq, hkv, d, rot, mode, layout, sections, dtype = shape
    c = Case(tokens, hq, hkv, d, rot, mode=mode, layout=layout, sections=sections, dtype=dtype,
             kv4=kv4, seed=1)
    q, k, v = c.views(c.dev)
    q_out = torch.zeros(tokens, hq, d, dtype=q.dtype, device="cuda")
    k_out = torch.zeros(tokens, hkv, d, dtype=q.dtype, device="cuda")
    c.run(q, k, v, q_out, k_out)
    assert same(q_out.cpu(), c.want_q) and same(k_out.cpu(), c.want_k)
    assert same(c.dev.cpu(), c.qkv)  # the inputs stay
    c.check_cache()
    assert int(c.cache.status.item()) == 0
    c.cache.close()


# enough tokens for the append's tiles of whole units; the ends of the chunk go row by row
LONG = [
    # tokens, hq, hkv, d, rot, mode, layout, sections, dtype
    (1613, 2, 8, 128, 128, "neox", "sections", [22, 21, 21], "bf16"),
    (1613, 1, 8, 128, 64, "neox", "interleaved", [12, 10, 10], "f16"),
    (1600, 1, 8, 64, 64, "gptj", "sections", None, "bf16"),
    (1505, 0, 8, 96, 96, "neox", "sections", [16, 16, 16], "f16"),
    (1505, 1, 8, 256, 256, "neox", "sections", None, "bf16"),
    (1490, 1, 8, 160, 128, "neox", "sections", [32, 32], "bf16"),
    (3100, 1, 4, 32, 32, "neox", "sections", None, "f16"),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("shape", LONG)
def test_long_prompts_into_four_bits(shape, in_place):
    torch = torch_cuda()
    tokens, hq, hkv, d, rot, mode, layout, sections, dtype = shape
    c = Case(tokens, hq, hkv, d, rot, mode=mode, layout=layout, sections=sections, dtype=dtype,
             kv4=True, seed=12)
    q, k, v = c.views(c.dev)
    q_out = q if in_place else torch.zeros(tokens, hq, d, dtype=k.dtype, device="cuda")
    k_out = k if in_place else torch.zeros(tokens, hkv, d, dtype=k.dtype, device="cuda")
    kw = {} if hq else dict(q_ptr=0, q_out_ptr=0)
    c.run(q, k, v, q_out, k_out, **kw)
    assert same(q_out.cpu(), c.want_q) and same(k_out.cpu(), c.want_k) and same(v.cpu(), c.v)
    c.check_cache()
    assert int(c.cache.status.item()) == 0
    c.cache.close()


@pytest.mark.parametrize("d", [32, 96, 160, 192, 224, 256])
def test_in_place_of_every_row_size(d):
    """Rows of which a warp's lanes hold whole ones, and rows that they do not."""
    for tokens in (5, 64):
        c = Case(tokens, 2, 3, d, d, kv4=True, seed=13)
        q, k, v = c.views(c.dev)
        c.run(q, k, v, q, k)
        assert same(q.cpu(), c.want_q) and same(k.cpu(), c.want_k)
        c.check_cache()
        c.cache.close()


@pytest.mark.parametrize("shape", SHAPES16)
def test_odd_shapes(shape):
    torch = torch_cuda()
    tokens, hq, hkv, d, rot, mode, layout, sections, dtype = shape
    c = Case(tokens, hq, hkv, d, rot, mode=mode, layout=layout, sections=sections, dtype=dtype,
             seed=2)
    q, k, v = c.views(c.dev)
    q_out = torch.zeros(tokens, hq, d, dtype=q.dtype, device="cuda")
    c.run(q, k, v, q_out)
    assert same(q_out.cpu(), c.want_q)
    c.check_cache()
    c.cache.close()


@pytest.mark.parametrize("kv4", [False, True])
def test_in_place(kv4):
    c = Case(37, 8, 2, 64, 48, kv4=kv4, seed=3, sections=[8, 8, 8])
    q, k, v = c.views(c.dev)
    c.run(q, k, v, q, k)
    assert same(q.cpu(), c.want_q) and same(k.cpu(), c.want_k) and same(v.cpu(), c.v)
    c.check_cache()
    c.cache.close()


@pytest.mark.parametrize("kv4", [False, True])
def test_only_the_cache(kv4):
    """No queries and no k_out."""
    c = Case(20, 4, 2, 64, 64, kv4=kv4, seed=4)
    q, k, v = c.views(c.dev)
    c.run(q, k, v, q, num_q_heads=0, q_ptr=0, q_out_ptr=0)
    assert same(c.dev.cpu(), c.qkv)
    c.check_cache()
    c.cache.close()


@pytest.mark.parametrize("kv4,d,rot", [(False, 128, 128), (True, 128, 64), (False, 72, 40)])
def test_rows_off_their_alignment(kv4, d, rot):
    """Views that start on 2 bytes, token-minor queries, odd row strides."""
    torch = torch_cuda()
    tokens, hq, hkv = 19, 4, 2
    c = Case(tokens, hq, hkv, d, rot, kv4=kv4, seed=5, dtype="f16")
    row = hkv * d
    flat = torch.zeros(tokens, 2 * row + 13, dtype=c.qkv.dtype, device="cuda")
    k = flat[:, 3:3 + row].unflatten(1, (hkv, d))
    v = flat[:, 7 + row:7 + 2 * row].unflatten(1, (hkv, d))
    q = torch.zeros(hq, tokens, d, dtype=c.qkv.dtype, device="cuda").permute(1, 0, 2)
    for x, y in zip((q, k, v), c.views(c.dev)):
        x.copy_(y)
    q_out = torch.zeros(tokens, hq + 1, d + 1, dtype=q.dtype, device="cuda")
    k_out = torch.zeros(tokens, row + 5, dtype=q.dtype, device="cuda")
    c.run(q, k, v, q_out[:, 1:, 1:], k_out[:, 5:].unflatten(1, (hkv, d)))
    assert same(q_out[:, 1:, 1:].cpu(), c.want_q)
    assert same(k_out[:, 5:].unflatten(1, (hkv, d)).cpu(), c.want_k)
    assert (q_out[:, 0] == 0).all() and (q_out[:, :, 0] == 0).all() and (k_out[:, :5] == 0).all()
    c.check_cache()
    c.cache.close()


@pytest.mark.parametrize("kv4", [False, True])
def test_far_and_negative_positions(kv4):
    pos = np.array([[0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9, 123456789, -7, 2 ** 24 + 1, 65535]],
                   np.int32)
    c = Case(10, 4, 2, 64, 64, seed=6, pos=pos, kv4=kv4)
    q, k, v = c.views(c.dev)
    c.run(q, k, v, q, k)
    assert same(q.cpu(), c.want_q) and same(k.cpu(), c.want_k)
    c.check_cache()
    c.cache.close()


@pytest.mark.parametrize("kv4", [False, True])
@pytest.mark.parametrize("tokens", [6, 64, 200])
def test_skipped_and_bad_slots(kv4, tokens):
    """Padding slots, a block past the table, a free block and an offset past the region: their
    tokens' rows come out, nothing of theirs is written, the others' are."""
    torch = torch_cuda()
    for kind, status in (("pad", 0), ("block", 1), ("free", 2), ("offset", 1 if kv4 else 3)):
        c = Case(tokens, 4, 2, 64, 64, seed=7, kv4=kv4, blocks=tokens // 16 + 4)
        bad = np.zeros(tokens, bool)
        bad[[1, tokens - 1]] = True
        slots, kw = c.slots.copy(), {}
        offsets = c.cache.offsets.copy()
        valid = torch.ones(len(offsets), dtype=torch.uint8, device="cuda")
        if kind == "pad":
            slots[bad] = -1
        elif kind == "block":
            slots[bad] = len(offsets) * 16 + 3
        else:
            spare = [b for b in range(len(offsets)) if b not in set(slots // 16)][0]
            slots[bad] = spare * 16
            if kind == "free":
                valid[spare] = 0
                kw = dict(valid_blocks_ptr=valid.data_ptr())
            else:
                offsets[spare] = 1 << 40
        c.d_slots.copy_(torch.from_numpy(slots))
        d_off = torch.from_numpy(offsets).cuda()
        before = [c.cache.region(x).clone() for x in "kv"]
        q, k, v = c.views(c.dev)
        c.run(q, k, v, q, k, block_offsets_f16_ptr=d_off.data_ptr(), **kw)
        assert same(q.cpu(), c.want_q) and same(k.cpu(), c.want_k)
        assert int(c.cache.status.item()) == status
        c.check_cache(~bad)
        for x, y in zip("kv", before):  # as many words changed as rows were written, at most
            changed = int((c.cache.region(x) != y).sum())
            assert changed <= int((~bad).sum()) * 2 * c.cache.row
        c.cache.close()


def test_pages_of_other_sizes():
    for bs in (1, 8, 24, 64):
        c = Case(50, 4, 2, 64, 64, seed=8, bs=bs)
        q, k, v = c.views(c.dev)
        c.run(q, k, v, q)
        c.check_cache()
        c.cache.close()


@pytest.mark.parametrize("kv4", [False, True])
def test_side_stream_and_graph(kv4):
    torch = torch_cuda()
    c = Case(70, 4, 2, 128, 128, seed=9, kv4=kv4, sections=[24, 20, 20], layout="interleaved")
    q, k, v = c.views(c.dev)
    q_out = torch.zeros(70, 4, 128, dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        c.run(q, k, v, q_out)
    assert same(q_out.cpu(), c.want_q)
    c.check_cache()
    g = torch.cuda.CUDAGraph()
    rope, p = c.rope(), c.cache.pool
    with torch.cuda.graph(g):
        p.rope_append(0, rope=rope, head_dim=128, num_q_heads=4, q_ptr=q.data_ptr(),
                      q_stride_token=q.stride(0), q_out_ptr=q_out.data_ptr(), k_ptr=k.data_ptr(),
                      k_row_stride=k.stride(0), v_ptr=v.data_ptr(), v_row_stride=v.stride(0),
                      slot_mapping_ptr=c.d_slots.data_ptr(),
                      block_offsets_f16_ptr=c.cache.d_offsets.data_ptr(),
                      block_offsets_f16_len=len(c.cache.offsets), num_tokens=70,
                      cache_format=int(kv4), stream_ptr=torch.cuda.current_stream().cuda_stream)
    new = Case(70, 4, 2, 128, 128, seed=10, kv4=kv4, sections=[24, 20, 20], layout="interleaved")
    c.dev.copy_(new.dev)
    c.d_pos.copy_(new.d_pos)
    q_out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert same(q_out.cpu(), new.want_q)
    c.want_k, c.v = new.want_k, new.v
    c.check_cache()
    c.cache.close()
    new.cache.close()


def test_as_the_separate_calls_do():
    """In one call what the 4-bit append gives for the rotated rows: the same page bytes."""
    torch = torch_cuda()
    a = Case(90, 8, 2, 128, 128, seed=11, kv4=True)
    b = Case(90, 8, 2, 128, 128, seed=11, kv4=True)
    q, k, v = a.views(a.dev)
    a.run(q, k, v, q)
    b.cache.write(b.want_k.cuda().contiguous(), b.v.cuda().contiguous(), b.slots)
    for x in "kv":
        assert torch.equal(a.cache.region(x), b.cache.region(x))
    a.cache.close()
    b.cache.close()
