"""Cases of the prompt operators: rotation and append in one call, attention over packed prompts.

Each case is one pass through an operator as a serving step calls it.  With `own`
false `run` computes it in elementary torch operations in 32 bits; with `own` true it
calls the library (`lattice_b200`).  `exact` computes the same outputs in 64 bits from
the definitions.

Operators and their definitions
  rope_append  q and k rows rotated, k and v rows into the slots of a paged cache.  Pair i of a
               row is (2i, 2i+1) or (i, i + rotary_dim/2); its angle is p * inv_freq[i], p the
               token's position on the pair's axis (time, height, width; one axis for text).
               A pair's axis goes by sections in order, or interleaved: i mod axes where
               i < axes * sections[i mod axes], else the first.
                 x1' = x1 cos - x2 sin,  x2' = x2 cos + x1 sin,  rounded to 16 bits.
               The cache holds k' and v: in 16 bits, or in 4 with a scale per group of 32
               (s = bf16(max|x| / 7), code = round-half-even(x / s), value = code * s); the
               latter are read back as 16-bit rows, as attention over a longer prompt needs them.
  prompt_attn  packed sequences of different lengths: query i of the nq of a sequence attends to
               its keys j <= i + nk - nq (all of them where not causal),
               out = sum_j softmax_j(scale * q_i k_j) v_j, query heads grouped on kv heads.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16}
_SB_BYTES = 2 << 20  # the pool maps its regions in superblocks of this size
_BS = 16             # tokens per page in every case

# --- cases ---------------------------------------------------------------------------


def listed():
    return [
        # one decode step of the Llama-3-8B serving batch: 64 tokens at positions of their own
        {"name": "rope_step", "op": "rope_append", "dtype": "bf16", "tokens": 64, "hq": 32, "hkv": 8,
         "d": 128, "rot": 128, "mode": "neox", "axes": 1, "layout": "sections", "cache": "16"},
        # a step of a few sequences into a 4-bit cache, half of each head rotated, adjacent pairs
        {"name": "rope_kv4_step", "op": "rope_append", "dtype": "f16", "tokens": 7, "hq": 16,
         "hkv": 4, "d": 64, "rot": 32, "mode": "gptj", "axes": 1, "layout": "sections",
         "cache": "kv4"},
        # the prompt of a long video: three axes, 16384 tokens into the 16-bit cache
        {"name": "rope_video", "op": "rope_append", "dtype": "bf16", "tokens": 16384, "hq": 32,
         "hkv": 8, "d": 128, "rot": 128, "mode": "neox", "axes": 3, "layout": "sections",
         "cache": "16"},
        # a prompt chunk with images into a 4-bit cache, interleaved axes, an odd count of tokens
        {"name": "rope_kv4_images", "op": "rope_append", "dtype": "bf16", "tokens": 4099, "hq": 32,
         "hkv": 8, "d": 128, "rot": 128, "mode": "neox", "axes": 3, "layout": "interleaved",
         "cache": "kv4"},
        # one short question: latency counts
        {"name": "attn_question", "op": "prompt_attn", "dtype": "f16", "batch": 1, "hq": 16,
         "hkv": 4, "d": 64, "min_len": 37, "max_len": 37, "min_past": 0, "max_past": 0,
         "causal": True},
        # a serving step's new prompts for the Llama-3-8B heads, from one token to 2048
        {"name": "attn_8b", "op": "prompt_attn", "dtype": "bf16", "batch": 16, "hq": 32, "hkv": 8,
         "d": 128, "min_len": 1, "max_len": 2048, "min_past": 0, "max_past": 0, "causal": True},
        # one kv head of the Llama-3-70B shape: a whole prompt of 32768 tokens
        {"name": "attn_70b_long", "op": "prompt_attn", "dtype": "bf16", "batch": 1, "hq": 8,
         "hkv": 1, "d": 128, "min_len": 32768, "max_len": 32768, "min_past": 0, "max_past": 0,
         "causal": True},
        # chunks of prompts after a past that was read back from a 4-bit cache
        {"name": "attn_chunks", "op": "prompt_attn", "dtype": "bf16", "batch": 4, "hq": 32,
         "hkv": 8, "d": 128, "min_len": 300, "max_len": 512, "min_past": 2000, "max_past": 8192,
         "causal": True},
        # small heads, f16, ragged
        {"name": "attn_d64", "op": "prompt_attn", "dtype": "f16", "batch": 8, "hq": 16, "hkv": 4,
         "d": 64, "min_len": 511, "max_len": 4001, "min_past": 0, "max_past": 0, "causal": True},
        # heads of 256 values, 4 query heads on one kv head
        {"name": "attn_d256", "op": "prompt_attn", "dtype": "bf16", "batch": 3, "hq": 8, "hkv": 2,
         "d": 256, "min_len": 1025, "max_len": 5000, "min_past": 0, "max_past": 0, "causal": True},
        # image patches, which see each other both ways: heads of 80 values, no grouping
        {"name": "attn_images", "op": "prompt_attn", "dtype": "bf16", "batch": 12, "hq": 16,
         "hkv": 16, "d": 80, "min_len": 256, "max_len": 1369, "min_past": 0, "max_past": 0,
         "causal": False},
        # single tokens of a batch over packed pasts
        {"name": "attn_tokens", "op": "prompt_attn", "dtype": "bf16", "batch": 32, "hq": 32,
         "hkv": 8, "d": 128, "min_len": 1, "max_len": 1, "min_past": 0, "max_past": 4095,
         "causal": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope_append", "prompt_attn", "prompt_attn"])
    heads = rng.choice([(32, 8), (16, 4), (8, 1), (12, 2), (4, 4), (28, 4), (16, 16)])
    dtype = rng.choice(["bf16", "f16"])
    if op == "rope_append":
        cache = rng.choice(["16", "kv4"])
        d = rng.choice([64, 96, 128, 128, 256] if cache == "kv4" else [64, 72, 80, 128, 128, 256])
        axes = rng.choice([1, 1, 2, 3, 3])
        rot = rng.choice([d, d, d // 16 * 8])
        cap = min(16384, (16384 * 40 * 128) // ((heads[0] + heads[1]) * d))
        return {"op": op, "dtype": dtype, "tokens": _log_int(rng, 1, cap), "hq": heads[0],
                "hkv": heads[1], "d": d, "rot": rot, "mode": rng.choice(["neox", "neox", "gptj"]),
                "axes": axes, "layout": rng.choice(["sections", "interleaved"]), "cache": cache}
    d = rng.choice([64, 64, 72, 80, 96, 128, 128, 128, 192, 256])
    batch = _log_int(rng, 1, 32)
    # at most a quarter of the longest listed case's products, whose plain form costs the most
    cap = int(math.sqrt(0.25 * 32768 * 32768 * 8 * 128 / (batch * heads[0] * d)))
    hi = _log_int(rng, 1, min(8192, max(64, cap)))
    past = rng.choice([0, 0, 1])
    causal = past == 1 or rng.random() < 0.8
    most = max(1, min(16384, 3 * cap * cap // (4 * hi))) if past else 0
    past_hi = _log_int(rng, 1, most) if past else 0
    return {"op": op, "dtype": dtype, "batch": batch, "hq": heads[0], "hkv": heads[1], "d": d,
            "min_len": rng.choice([1, max(1, hi // 3), hi]), "max_len": hi,
            "min_past": rng.choice([0, past_hi // 2]), "max_past": past_hi, "causal": causal}


# --- inputs --------------------------------------------------------------------------


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + salt)


def _spread(lo, hi, n, seed, salt):
    """n lengths from lo to hi, evenly, in an order of the seed's; hi alone where n is 1."""
    x = np.full(1, hi) if n == 1 else np.round(np.linspace(lo, hi, n))
    return np.random.default_rng([int(seed), salt]).permutation(x.astype(np.int64))


def _lens(case, seed):
    new = _spread(case["min_len"], case["max_len"], case["batch"], seed, 17)
    return new, new + _spread(case["min_past"], case["max_past"], case["batch"], seed, 19)


def _keys(shape, seed, salt, dt):
    """Normal rows with some loud channels per head, as projections have them."""
    g = _gen(seed, salt)
    x = torch.randn(shape, device="cuda", generator=g)
    loud = torch.rand(shape[-2:], device="cuda", generator=g)
    return (x * (1.0 + 3.0 * (loud > 0.94).float())).to(dt)


def _values(shape, seed, salt, dt):
    g = _gen(seed, salt)
    x = torch.randn(shape, device="cuda", generator=g)
    return (x * (0.3 + torch.rand(shape[:-1], device="cuda", generator=g))[..., None]).to(dt)


def _rope_positions(case, seed):
    """int32 [axes][tokens]: runs of text, whose axes agree, between images or frames, whose
    tokens lie on a grid; a step's tokens belong to sequences of their own."""
    r = np.random.default_rng([int(seed), 23])
    n, axes = case["tokens"], case["axes"]
    if n <= 256:
        return np.tile(r.integers(0, 131072, n).astype(np.int32), (axes, 1))
    cols, at, done = [], int(r.integers(0, 4096)), 0
    while done < n:
        text = int(r.integers(8, 200))
        cols.append(np.tile(at + np.arange(text), (axes, 1)))
        at, done = at + text, done + text
        if axes > 1:
            size = [int(r.integers(1, 5))] + [int(r.integers(8, 40)) for _ in range(axes - 1)]
            grid = np.stack(np.meshgrid(*[np.arange(s) for s in size], indexing="ij"))
            cols.append(at + grid.reshape(axes, -1))
            at, done = at + max(size), done + int(np.prod(size))
    return np.concatenate(cols, axis=1)[:, :n].astype(np.int32)


def _sections(case):
    """How many of a row's pairs go to each axis: the first gets the odd ones."""
    half = case["rot"] // 2
    rest = [half // case["axes"]] * (case["axes"] - 1)
    return [half - sum(rest)] + rest


def _pair_axes(case):
    s, n = _sections(case), case["axes"]
    if case["layout"] == "sections":
        return np.repeat(np.arange(n), s)
    i = np.arange(case["rot"] // 2)
    return np.where(i < n * np.array(s)[i % n], i % n, 0)


def _inv_freq(case):
    """float32, of base 500000."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
    return (500000.0 ** (-2.0 * i / case["rot"])).float()


def _rope_inputs(case, seed):
    """q, k and v rows as views of one projection's output."""
    t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
    dt = _DT[case["dtype"]]
    qkv = torch.empty(t, hq + 2 * hkv, d, dtype=dt, device="cuda")
    qkv[:, : hq + hkv] = _keys((t, hq + hkv, d), seed, 7, dt)
    qkv[:, hq + hkv:] = _values((t, hkv, d), seed, 11, dt)
    return qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]


def _rope_slots(case, seed, pages):
    """Page number * _BS + place of each token: a step's tokens lie in pages of their own, a
    chunk's in consecutive slots of scattered pages."""
    r = np.random.default_rng([int(seed), 29])
    slots = (r.permutation(pages)[:, None] * _BS + np.arange(_BS)[None, :]).reshape(-1)
    if case["tokens"] <= 256:
        slots = r.permutation(slots)
    return slots[: case["tokens"]].copy()


def _attn_inputs(case, seed):
    """q as a view of a projection's output; k and v packed (with their pasts in front)."""
    new, total = _lens(case, seed)
    hq, hkv, d, dt = case["hq"], case["hkv"], case["d"], _DT[case["dtype"]]
    nq, nk = int(new.sum()), int(total.sum())
    qkv = torch.empty(nq, hq + 2 * hkv, d, dtype=dt, device="cuda")
    qkv[:, :hq] = 1.5 * torch.randn(nq, hq, d, device="cuda", generator=_gen(seed, 3))
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    rows_k, rows_v = _keys((nk, hkv, d), seed, 7, dt), _values((nk, hkv, d), seed, 11, dt)
    if nk != nq:
        return new, total, q, rows_k, rows_v
    k.copy_(rows_k)
    v.copy_(rows_v)
    return new, total, q, k, v


# --- the library's state -----------------------------------------------------------------


class _Pool:
    """A pool of `pages` pages whose page number p lies p-th in the region."""

    def __init__(self, hkv, row_elems, pages, max_batch):
        from lattice_b200 import kcmm, workloads

        max_pages = -(-pages // max_batch)
        self.pool = workloads.library().create_pool(kcmm.make_config(
            num_layers=1, kv_heads=hkv, head_dim=row_elems, max_batch=max_batch,
            max_seq_len=max_pages * _BS, block_size=_BS))
        ids = np.array(self.pool.alloc_blocks(pages), np.int64)
        offsets = np.array(self.pool.all_block_offsets_f16(), np.uint64).astype(np.int64)
        self.ids = ids[np.argsort(offsets[ids])]  # page number -> block id
        self.offsets = torch.from_numpy(offsets).cuda()

    def __del__(self):
        pool = getattr(self, "pool", None)
        if pool is not None:
            pool.destroy()

    def region(self, kind, pages, per, page_elems, dt):
        """The pages as a view [superblocks, pages per superblock, elements]."""
        base = self.pool.va_k(0) if kind == "k" else self.pool.va_v(0)
        n = pages // per * (_SB_BYTES // 2)

        class _View:
            __cuda_array_interface__ = {"shape": (n,), "typestr": "<i2", "data": (base, False),
                                        "version": 3}

        t = torch.as_tensor(_View(), device="cuda").view(dt)
        return t.as_strided((pages // per, per, page_elems), (_SB_BYTES // 2, page_elems, 1))


def _stream():
    return torch.cuda.current_stream().cuda_stream


def prepare(case, seed):
    return globals()["_prepare_" + case["op"]](case, seed)


def run(state):
    if own:
        return globals()["_own_" + state["op"]](state)
    return globals()["_plain_" + state["op"]](state)


# --- rope_append ---------------------------------------------------------------------------


def _rope_pages(case):
    """Pages rounded up to whole superblocks of the 16-bit cache, and how many one holds."""
    per = max(1, _SB_BYTES // (_BS * case["hkv"] * case["d"] * 2))
    return -(-(-(-case["tokens"] // _BS) + 8) // per) * per, per


def _prepare_rope_append(case, seed):
    q, k, v = _rope_inputs(case, seed)
    pages, per = _rope_pages(case)
    slots = _rope_slots(case, seed, pages)
    st = dict(case, q=q, k=k, v=v, inv_freq=_inv_freq(case),
              positions=torch.from_numpy(_rope_positions(case, seed)).cuda())
    elems = _BS * case["hkv"] * case["d"]
    if not own:
        st["pair_axes"] = torch.from_numpy(_pair_axes(case)).cuda()
        st["slots"] = torch.from_numpy(slots).cuda()
        if case["cache"] == "16":
            st["pages"] = [torch.zeros(pages // per, per, elems, dtype=k.dtype, device="cuda")
                           for _ in "kv"]
        else:
            st["codes"] = torch.zeros(2, pages * _BS, case["hkv"], case["d"] // 2,
                                      dtype=torch.uint8, device="cuda")
            st["scales"] = torch.zeros(2, pages * _BS, case["hkv"], case["d"] // 32,
                                       dtype=torch.bfloat16, device="cuda")
        return st
    from lattice_b200 import kcmm

    row = case["d"] if case["cache"] == "16" else kcmm.kv4_row_elems(case["d"])
    p = st["pool"] = _Pool(case["hkv"], row, pages, 1)
    st["slots"] = torch.from_numpy(p.ids[slots // _BS] * _BS + slots % _BS).cuda()
    st["rope"] = kcmm.make_rope(
        mode=case["mode"], rotary_dim=case["rot"], inv_freq_ptr=st["inv_freq"].data_ptr(),
        positions_ptr=st["positions"].data_ptr(), positions_row_stride=case["tokens"],
        sections=_sections(case), layout=case["layout"])
    st["q_out"] = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    st["k_out"] = torch.empty(k.shape, dtype=k.dtype, device="cuda")
    if case["cache"] == "16":
        st["pages"] = [p.region(x, pages, per, elems, k.dtype) for x in "kv"]
        for x in st["pages"]:
            x.zero_()
    else:
        st["read"] = [torch.empty(k.shape, dtype=k.dtype, device="cuda") for _ in "kv"]
    return st


def _plain_rotate(x, c, s, rot, mode):
    y = x.float()
    a, b = ((y[..., : rot // 2], y[..., rot // 2:rot]) if mode == "neox"
            else (y[..., 0:rot:2], y[..., 1:rot:2]))
    first, second = a * c - b * s, b * c + a * s
    turned = (torch.cat((first, second), -1) if mode == "neox"
              else torch.stack((first, second), -1).flatten(-2))
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _plain_quantise(x):
    """Codes + 8 packed two to a byte, and the groups' scales."""
    g = x.float().unflatten(-1, (-1, 32))
    s = (g.abs().amax(-1) / 7.0).to(torch.bfloat16)
    sf = s.float()[..., None]
    c = torch.where(sf > 0, torch.round(g / sf), torch.zeros_like(g)).clamp(-7, 7)
    c = (c + 8).to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), s


def _plain_dequantise(codes, scales):
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    return (c.unflatten(-1, (-1, 32)) * scales.float()[..., None]).flatten(-2)


def _plain_rope_append(st):
    p = st["positions"].T[:, st["pair_axes"]]            # [tokens, pairs]
    angle = p.double() * st["inv_freq"].double()          # positions lie far out: 64 bits
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    q = _plain_rotate(st["q"], c, s, st["rot"], st["mode"])
    k = _plain_rotate(st["k"], c, s, st["rot"], st["mode"])
    if st["cache"] == "16":
        for pages, x in zip(st["pages"], (k, st["v"])):
            pages.view(-1, st["hkv"], st["d"])[st["slots"]] = x
        return [q, k] + st["pages"]
    read = []
    for i, x in enumerate((k, st["v"])):
        codes, scales = _plain_quantise(x)
        st["codes"][i, st["slots"]], st["scales"][i, st["slots"]] = codes, scales
        read.append(_plain_dequantise(st["codes"][i, st["slots"]],
                                      st["scales"][i, st["slots"]]).to(x.dtype))
    return [q, k] + read


def _own_rope_append(st):
    p, stream = st["pool"], _stream()
    cache = dict(slot_mapping_ptr=st["slots"].data_ptr(), block_offsets_f16_ptr=p.offsets.data_ptr(),
                 block_offsets_f16_len=p.offsets.shape[0], num_tokens=st["tokens"],
                 head_dim=st["d"], dtype=st["dtype"], stream_ptr=stream)
    q, k, v, q_out, k_out = st["q"], st["k"], st["v"], st["q_out"], st["k_out"]
    p.pool.rope_append(
        0, rope=st["rope"], cache_format=0 if st["cache"] == "16" else 1,
        num_q_heads=st["hq"], q_ptr=q.data_ptr(), q_stride_token=q.stride(0),
        q_stride_head=q.stride(1), q_out_ptr=q_out.data_ptr(), k_ptr=k.data_ptr(),
        k_row_stride=k.stride(0), v_ptr=v.data_ptr(), v_row_stride=v.stride(0),
        k_out_ptr=k_out.data_ptr(), **cache)
    if st["cache"] == "16":
        return [q_out, k_out] + st["pages"]
    rk, rv = st["read"]
    p.pool.kv4_read(0, k_dst_ptr=rk.data_ptr(), v_dst_ptr=rv.data_ptr(), **cache)
    return [q_out, k_out, rk, rv]


def _exact_rotate(x, angle, rot, mode):
    y = x.double().clone()
    i = torch.arange(rot // 2, device="cuda")
    at, by = (i, i + rot // 2) if mode == "neox" else (2 * i, 2 * i + 1)
    a, b = y[..., at].clone(), y[..., by].clone()
    y[..., at] = a * torch.cos(angle) - b * torch.sin(angle)
    y[..., by] = b * torch.cos(angle) + a * torch.sin(angle)
    return y


def _exact_quantised(x):
    g = x.double().reshape(x.shape[0], x.shape[1], -1, 32)
    s = (g.abs().max(dim=-1, keepdim=True).values / 7).to(torch.bfloat16).double()
    safe = torch.where(s == 0, torch.ones_like(s), s)
    c = torch.minimum(torch.maximum((g / safe).round(), torch.full_like(g, -7)),
                      torch.full_like(g, 7))
    return torch.where(s == 0, torch.zeros_like(c), c * s).reshape(x.shape)


def _exact_rope_append(case, seed):
    q, k, v = _rope_inputs(case, seed)
    pos = _rope_positions(case, seed).astype(np.float64)[_pair_axes(case)].T
    angle = (torch.from_numpy(pos).cuda() * _inv_freq(case).double())[:, None]
    q, turned = (_exact_rotate(x, angle, case["rot"], case["mode"]) for x in (q, k))
    if case["cache"] == "kv4":  # the cache's groups are of the rounded rows
        return [q, turned, _exact_quantised(turned.to(k.dtype)), _exact_quantised(v)]
    pages, per = _rope_pages(case)
    slots = torch.from_numpy(_rope_slots(case, seed, pages)).cuda()
    out = []
    for x in (turned, v.double()):
        y = torch.zeros(pages * _BS, case["hkv"], case["d"], dtype=torch.float64, device="cuda")
        y[slots] = x
        out.append(y.view(pages // per, per, -1))
    return [q, turned] + out


# --- prompt_attn ---------------------------------------------------------------------------


def _starts(lens):
    return np.concatenate(([0], np.cumsum(lens)))


def _prepare_prompt_attn(case, seed):
    new, total, q, k, v = _attn_inputs(case, seed)
    st = dict(case, q=q, k=k, v=v, scale=1.0 / math.sqrt(case["d"]),
              new=new.tolist(), total=total.tolist())
    st["q_start"], st["k_start"] = (torch.from_numpy(_starts(x).astype(np.int32)).cuda()
                                    for x in (new, total))
    if own:
        st["pool"] = _Pool(1, 64, 8, 1)
        st["out"] = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    return st


def _plain_prompt_attn(st):
    """A sequence at a time, in blocks of queries whose scores take 2 GB at most."""
    hkv, out, q0, k0 = st["hkv"], [], 0, 0
    for nq, nk in zip(st["new"], st["total"]):
        k = st["k"][k0:k0 + nk].float().permute(1, 2, 0)
        v = st["v"][k0:k0 + nk].float().transpose(0, 1)
        step = max(1, (1 << 29) // (nk * st["hq"]))
        for i in range(0, nq, step):
            q = st["q"][q0 + i:q0 + min(nq, i + step)].float()
            n = q.shape[0]
            q = q.unflatten(1, (hkv, -1)).permute(1, 2, 0, 3).flatten(1, 2)  # [hkv, group * n, d]
            s = torch.matmul(q, k) * st["scale"]
            if st["causal"]:
                last = torch.arange(i, i + n, device="cuda")[:, None] + (nk - nq)
                s = s.unflatten(1, (-1, n)).masked_fill(
                    torch.arange(nk, device="cuda")[None, :] > last, -math.inf).flatten(1, 2)
            e = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
            out.append(o.unflatten(1, (-1, n)).permute(2, 0, 1, 3).flatten(1, 2))
        q0, k0 = q0 + nq, k0 + nk
    return torch.cat(out).to(st["q"].dtype)


def _own_prompt_attn(st):
    q, k, v, out = st["q"], st["k"], st["v"], st["out"]
    st["pool"].pool.prompt_attn(
        query_ptr=q.data_ptr(), q_stride_token=q.stride(0), q_stride_head=q.stride(1),
        key_ptr=k.data_ptr(), k_stride_token=k.stride(0), k_stride_head=k.stride(1),
        value_ptr=v.data_ptr(), v_stride_token=v.stride(0), v_stride_head=v.stride(1),
        out_ptr=out.data_ptr(), q_start_ptr=st["q_start"].data_ptr(),
        k_start_ptr=st["k_start"].data_ptr(), batch=st["batch"], num_q_tokens=q.shape[0],
        num_k_tokens=k.shape[0], num_q_heads=st["hq"], kv_heads=st["hkv"], head_dim=st["d"],
        scale=st["scale"], causal=st["causal"], dtype=st["dtype"], stream_ptr=_stream())
    return out


def _exact_prompt_attn(case, seed):
    new, total, q, k, v = _attn_inputs(case, seed)
    group = case["hq"] // case["hkv"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    qs, ks = _starts(new), _starts(total)
    for b in range(case["batch"]):
        n, m = int(new[b]), int(total[b])
        for h in range(case["hq"]):
            kh = k[ks[b]:ks[b + 1], h // group].double()
            vh = v[ks[b]:ks[b + 1], h // group].double()
            for i in range(0, n, 4096):
                rows = q[qs[b] + i:qs[b] + min(n, i + 4096), h].double()
                s = rows @ kh.T / math.sqrt(case["d"])
                if case["causal"]:
                    s += torch.full_like(s, -math.inf).triu(1 + i + m - n)
                out[qs[b] + i:qs[b] + i + len(rows), h] = torch.softmax(s, dim=1) @ vh
    return out


def exact(case, seed):
    return globals()["_exact_" + case["op"]](case, seed)


# --- work ----------------------------------------------------------------------------------


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "rope_append":
        t, row = case["tokens"], hkv * d
        held = 4 * row if case["cache"] == "16" else 2 * (row * 9 // 16)
        read = 0 if case["cache"] == "16" else held + 4 * row
        return {"bytes": t * (4 * hq * d + 6 * row + held + read + 4 * case["axes"] + 8),
                "flops": 3 * t * (hq + hkv) * case["rot"]}
    b = case["batch"]
    new, total = _lens(case, 0)
    pairs = 0.0
    for s in range(8):  # which past goes with which prompt is the seed's
        new, total = (x.astype(np.float64) for x in _lens(case, s))
        seen = new * (total - new) + new * (new + 1) / 2 if case["causal"] else new * total
        pairs += seen.sum() / 8
    return {"bytes": int(4 * new.sum() * hq * d + 4 * total.sum() * hkv * d + 8 * (b + 1)),
            "flops": int(4 * pairs * hq * d)}
