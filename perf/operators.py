"""Cases of the cache operators: the 4-bit KV cache, attention-weight eviction, beam selection.

Each case is one pass through an operator as a serving step calls it.  With `own`
false `run` computes it in elementary torch operations in 32 bits; with `own` true it
calls the library (`lattice_b200`).  `exact` computes the same outputs in 64 bits from
the definitions.

Operators and their definitions
  kv4_store    rows of K and V quantised into a paged 4-bit cache and read back.
               Groups of 32 along head_dim: s = bf16(max|x| / 7), code = round-half-even(x/s)
               clamped to [-7, 7] (0 where s is 0), value = code * s.
  kv4_decode   softmax(scale * q k) v of one query token per sequence over that cache;
               with "weights" also w_out[b, kv head, t] = w_in + sum of the softmax
               weights of the kv head's query heads at token t.
  weights      the same decode and weights over the 16-bit cache.
  evict        per sequence and kv head: of n > budget cached tokens the `sinks` first and
               `recent` last positions stay, and of the others those with the largest
               accumulated weight (ties: the lowest index); the kept rows past `budget`
               move, in order, into the freed slots below it.
  beam         the n best of beams x vocabulary by score + log_softmax(logits), ties to the
               lowest (beam, token), then the beams' token histories and block tables
               gathered by parent.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SB_BYTES = 2 << 20  # the pool maps its regions in superblocks of this size
_BS = 16             # tokens per page in every case

# --- cases ---------------------------------------------------------------------------


def listed():
    return [
        # one decode step of the Llama-3-8B serving batch: 64 new tokens into the cache
        {"name": "kv4_store_step", "op": "kv4_store", "dtype": "bf16", "tokens": 64,
         "hkv": 8, "d": 128},
        # a prompt chunk of 16384 tokens stored after prefill, f16 model
        {"name": "kv4_store_chunk", "op": "kv4_store", "dtype": "f16", "tokens": 16384,
         "hkv": 8, "d": 128},
        # interactive: a few short sequences, latency counts; odd lengths, one of one token
        {"name": "kv4_decode_few", "op": "kv4_decode", "dtype": "f16", "batch": 3, "hq": 16,
         "hkv": 4, "d": 64, "min_len": 1, "max_len": 777, "weights": False},
        # the Llama-3-8B decode batch of the benchmark over a 4-bit cache
        {"name": "kv4_decode_8b", "op": "kv4_decode", "dtype": "bf16", "batch": 64, "hq": 32,
         "hkv": 8, "d": 128, "min_len": 512, "max_len": 4096, "weights": False},
        # one kv head of the Llama-3-70B long-context batch: 8 sequences of up to 32768 tokens
        {"name": "kv4_decode_long", "op": "kv4_decode", "dtype": "bf16", "batch": 8, "hq": 8,
         "hkv": 1, "d": 128, "min_len": 30001, "max_len": 32768, "weights": False},
        # the 4-bit cache with accumulated weights, a mid-size batch
        {"name": "kv4_decode_weights", "op": "kv4_decode", "dtype": "bf16", "batch": 16, "hq": 32,
         "hkv": 8, "d": 128, "min_len": 900, "max_len": 2100, "weights": True},
        # the benchmark's decode batch over the 16-bit cache with accumulated weights
        {"name": "weights_8b", "op": "weights", "dtype": "bf16", "batch": 64, "hq": 32, "hkv": 8,
         "d": 128, "min_len": 512, "max_len": 4096},
        # a few short f16 sequences with accumulated weights
        {"name": "weights_few", "op": "weights", "dtype": "f16", "batch": 4, "hq": 16, "hkv": 4,
         "d": 64, "min_len": 1, "max_len": 600},
        # first eviction after prefill: contexts of up to 3700 tokens cut to 1024
        {"name": "evict_prefill", "op": "evict", "dtype": "bf16", "batch": 16, "hkv": 8, "d": 128,
         "min_len": 2900, "max_len": 3700, "budget": 1024, "sinks": 4, "recent": 256,
         "again": False},
        # long contexts that were cut before and have grown by up to 512 tokens since
        {"name": "evict_long", "op": "evict", "dtype": "f16", "batch": 4, "hkv": 4, "d": 64,
         "min_len": 16385, "max_len": 16895, "budget": 16384, "sinks": 1, "recent": 2048,
         "again": True},
        # one request with 4 beams over a small vocabulary in 32 bits
        {"name": "beam_one", "op": "beam", "dtype": "f32", "batch": 1, "beams": 4, "vocab": 32000,
         "select": 4, "history": 100, "pages": 16},
        # the benchmark's 16 requests of 4 beams over the Llama-3 vocabulary
        {"name": "beam_16x4", "op": "beam", "dtype": "bf16", "batch": 16, "beams": 4,
         "vocab": 128256, "select": 4, "history": 2176, "pages": 136},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["kv4_store", "kv4_decode", "weights", "evict", "beam"])
    heads = rng.choice([(32, 8), (16, 4), (8, 1), (12, 2), (4, 4), (28, 4), (16, 1)])
    d = rng.choice([64, 64, 96, 128, 128, 128, 256])
    dtype = rng.choice(["bf16", "f16"])
    row = heads[1] * d  # elements of a token's K row
    if op == "kv4_store":
        cap = min(16384, (16384 * 1024) // row)
        return {"op": op, "dtype": dtype, "tokens": _log_int(rng, 1, cap), "hkv": heads[1], "d": d}
    if op in ("kv4_decode", "weights"):
        batch = _log_int(rng, 1, 64)
        cap = (64 * 2304 * 1024) // (row * batch)
        hi = _log_int(rng, 17, max(18, min(32768, cap)))
        lo = rng.choice([1, max(1, hi // 3), max(1, hi - 7)])
        c = {"op": op, "dtype": dtype, "batch": batch, "hq": heads[0], "hkv": heads[1], "d": d,
             "min_len": lo, "max_len": hi}
        if op == "kv4_decode":
            c["weights"] = rng.random() < 0.4
        return c
    if op == "evict":
        batch = _log_int(rng, 1, 16)
        cap = min(16895, (16 * 3700 * 1024) // (row * batch))
        hi = _log_int(rng, 65, max(66, cap))
        budget = max(16, int(hi * rng.choice([0.25, 0.5, 0.9])))
        recent = rng.randint(0, budget // 2)
        return {"op": op, "dtype": dtype, "batch": batch, "hkv": heads[1], "d": d,
                "min_len": max(1, hi // 2), "max_len": hi, "budget": budget,
                "sinks": rng.randint(0, min(8, budget - recent)), "recent": recent,
                "again": rng.random() < 0.5}
    batch, beams = _log_int(rng, 1, 16), rng.choice([1, 2, 4, 4])
    return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "batch": batch, "beams": beams,
            "vocab": _log_int(rng, 1000, 128256 if batch <= 8 else 64128),
            "select": rng.choice([beams, beams, 2 * beams]),
            "history": _log_int(rng, 1, 2176), "pages": _log_int(rng, 1, 136)}


# --- inputs --------------------------------------------------------------------------


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + salt)


def _lens(case, seed):
    r = np.random.default_rng([int(seed), 17])
    n = r.integers(case["min_len"], case["max_len"] + 1, case["batch"])
    n[r.integers(case["batch"])] = case["max_len"]
    if case["batch"] > 1:
        n[(int(np.argmax(n)) + 1) % case["batch"]] = case["min_len"]
    return n.astype(np.int64)


def _keys(shape, seed, salt, dt):
    """Normal rows with some loud channels per head, as rotated keys have them."""
    g = _gen(seed, salt)
    x = torch.randn(shape, device="cuda", generator=g)
    loud = torch.rand(shape[-2:], device="cuda", generator=g)
    return (x * (1.0 + 3.0 * (loud > 0.94).float())).to(dt)


def _values(shape, seed, salt, dt):
    g = _gen(seed, salt)
    x = torch.randn(shape, device="cuda", generator=g)
    return (x * (0.3 + torch.rand(shape[:-1], device="cuda", generator=g))[..., None]).to(dt)


def _geometry(case, pages, page_bytes):
    """Pages rounded up to whole superblocks, and how many a superblock holds."""
    per = _SB_BYTES // page_bytes
    return -(-pages // per) * per, per


def _layout(case, seed, page_bytes):
    """Lengths, page counts and the table of page numbers of every sequence."""
    lens = _lens(case, seed)
    max_pages = -(-int(case["max_len"]) // _BS)
    need = [-(-int(n) // _BS) for n in lens]
    total, per = _geometry(case, sum(need) + 3, page_bytes)
    order = np.random.default_rng([int(seed), 23]).permutation(total)
    tables = np.zeros((case["batch"], max_pages), np.int64)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return lens, tables, total, per


def _queries(case, seed):
    x = torch.randn(case["batch"], case["hq"], case["d"], device="cuda", generator=_gen(seed, 3))
    return (1.5 * x).to(_DT[case["dtype"]])


def _start_weights(case, seed, stride):
    """Weights gathered so far: heavy-tailed, as attention leaves them."""
    u = torch.rand(case["batch"], case["hkv"], stride, device="cuda", generator=_gen(seed, 5))
    return 1e-3 / (u + 1e-4)


def _page_rows(case, seed, page_bytes):
    lens, tables, total, per = _layout(case, seed, page_bytes)
    shape = (total * _BS, case["hkv"], case["d"])
    dt = _DT[case["dtype"]]
    return lens, tables, total, per, _keys(shape, seed, 7, dt), _values(shape, seed, 11, dt)


def _kv_page_bytes(case):
    elems = case["d"] * 9 // 32 if case["op"].startswith("kv4") else case["d"]
    return _BS * case["hkv"] * elems * 2


def _evict_state(case, seed, lens):
    """Positions of the cached tokens: those of an earlier eviction, then fresh ones."""
    r = np.random.default_rng([int(seed), 31])
    b_n, h_n, stride = case["batch"], case["hkv"], int(case["max_len"])
    pos = np.zeros((b_n, h_n, stride), np.int32)
    kept = np.zeros(b_n, np.int32)
    nxt = lens.astype(np.int32)
    if case["again"]:
        for b in range(b_n):
            kept[b] = min(case["budget"], int(lens[b]))
            nxt[b] = lens[b] + 5 * kept[b] // 4
            gap = int(nxt[b] - lens[b])
            for h in range(h_n):
                p = np.sort(r.permutation(int(kept[b]) + gap)[: kept[b]])
                k = min(len(p), 64)  # some slots were refilled from the tail, out of order
                idx = r.choice(len(p), k, replace=False)
                p[idx] = r.permutation(p[idx])
                pos[b, h, : kept[b]] = p
    return pos, kept, nxt


def _logits(case, seed):
    shape = (case["batch"], case["beams"], case["vocab"])
    x = 2.5 * torch.randn(shape, device="cuda", generator=_gen(seed, 13))
    return x.to(_DT[case["dtype"]])


def _beam_inputs(case, seed):
    logits = _logits(case, seed)
    g = _gen(seed, 19)
    scores = -3.0 * torch.rand(case["batch"], case["beams"], device="cuda", generator=g) - 20.0
    hist = torch.randint(0, case["vocab"], (case["batch"], case["beams"], case["history"] + 1),
                         device="cuda", generator=g, dtype=torch.int32)
    tables = torch.randint(0, 40000, (case["batch"], case["beams"], case["pages"]), device="cuda",
                           generator=g, dtype=torch.int32)
    return logits, scores, hist, tables


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

    def tables(self, pages):
        return torch.from_numpy(self.ids[pages].astype(np.int32)).cuda()

    def slots(self, total):
        s = self.ids[:total, None] * _BS + np.arange(_BS)[None, :]
        return torch.from_numpy(s.reshape(-1)).cuda()

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


# --- kv4_store ---------------------------------------------------------------------------


def _store_inputs(case, seed):
    shape = (case["tokens"], case["hkv"], case["d"])
    dt = _DT[case["dtype"]]
    return _keys(shape, seed, 7, dt), _values(shape, seed, 11, dt)


def _prepare_kv4_store(case, seed):
    k, v = _store_inputs(case, seed)
    st = dict(case, k=k, v=v)
    if not own:
        st["codes"] = torch.zeros((2,) + tuple(k.shape[:-1]) + (case["d"] // 2,),
                                  dtype=torch.uint8, device="cuda")
        st["scales"] = torch.zeros((2,) + tuple(k.shape[:-1]) + (case["d"] // 32,),
                                   dtype=torch.bfloat16, device="cuda")
        return st
    from lattice_b200 import kcmm

    pages = -(-case["tokens"] // _BS) + 8
    st["pool"] = _Pool(case["hkv"], kcmm.kv4_row_elems(case["d"]), pages, 8)
    # a step's tokens lie in pages of their own, a chunk's in consecutive slots
    r = np.random.default_rng([int(seed), 29])
    order = st["pool"].ids[r.permutation(pages)]
    slots = (order[:, None] * _BS + np.arange(_BS)[None, :]).reshape(-1)
    if case["tokens"] <= 256:
        slots = r.permutation(slots)
    st["slots"] = torch.from_numpy(slots[: case["tokens"]].copy()).cuda()
    st["k_out"], st["v_out"] = torch.empty_like(k), torch.empty_like(v)
    return st


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


def _plain_kv4_store(st):
    out = []
    for i, x in enumerate((st["k"], st["v"])):
        st["codes"][i], st["scales"][i] = _plain_quantise(x)
        out.append(_plain_dequantise(st["codes"][i], st["scales"][i]).to(x.dtype))
    return out


def _own_kv4_store(st):
    p = st["pool"]
    args = dict(slot_mapping_ptr=st["slots"].data_ptr(),
                block_offsets_f16_ptr=p.offsets.data_ptr(),
                block_offsets_f16_len=p.offsets.shape[0], num_tokens=st["tokens"],
                head_dim=st["d"], dtype=st["dtype"], stream_ptr=_stream())
    p.pool.kv4_append(0, k_src_ptr=st["k"].data_ptr(), v_src_ptr=st["v"].data_ptr(), **args)
    p.pool.kv4_read(0, k_dst_ptr=st["k_out"].data_ptr(), v_dst_ptr=st["v_out"].data_ptr(), **args)
    return [st["k_out"], st["v_out"]]


def _exact_quantised(x):
    g = x.double().reshape(x.shape[0], x.shape[1], -1, 32)
    s = (g.abs().max(dim=-1, keepdim=True).values / 7).to(torch.bfloat16).double()
    safe = torch.where(s == 0, torch.ones_like(s), s)
    c = torch.minimum(torch.maximum((g / safe).round(), torch.full_like(g, -7)),
                      torch.full_like(g, 7))
    return torch.where(s == 0, torch.zeros_like(c), c * s).reshape(x.shape)


def _exact_kv4_store(case, seed):
    return [_exact_quantised(x) for x in _store_inputs(case, seed)]


# --- decode over the 4-bit and the 16-bit cache --------------------------------------------


def _prepare_decode(case, seed, kv4):
    lens, tables, total, per, k, v = _page_rows(case, seed, _kv_page_bytes(case))
    stride = int(case["max_len"])
    st = dict(case, q=_queries(case, seed), scale=1.0 / math.sqrt(case["d"]),
              lens=torch.from_numpy(lens.astype(np.int32)).cuda(), stride=stride)
    if not kv4 or case["weights"]:
        st["w_in"] = _start_weights(case, seed, stride)
        st["w_out"] = torch.zeros_like(st["w_in"])
    if not own:
        st["tables"] = torch.from_numpy(tables).cuda()
        for name, x in (("k", k), ("v", v)):
            x = x.view(total, _BS, case["hkv"], case["d"])
            st[name] = _plain_quantise(x) if kv4 else x
        return st
    row = case["d"]
    if kv4:
        from lattice_b200 import kcmm

        row = kcmm.kv4_row_elems(case["d"])
    p = _Pool(case["hkv"], row, total, case["batch"])
    st["pool"], st["tables"] = p, p.tables(tables)
    if kv4:
        slots = p.slots(total)
        p.pool.kv4_append(0, slot_mapping_ptr=slots.data_ptr(),
                          block_offsets_f16_ptr=p.offsets.data_ptr(),
                          block_offsets_f16_len=p.offsets.shape[0], num_tokens=total * _BS,
                          head_dim=case["d"], dtype=case["dtype"], stream_ptr=_stream(),
                          k_src_ptr=k.data_ptr(), v_src_ptr=v.data_ptr())
        torch.cuda.synchronize()
    else:
        elems = _BS * case["hkv"] * case["d"]
        for name, x in (("k", k), ("v", v)):
            p.region(name, total, per, elems, x.dtype).copy_(x.view(total // per, per, elems))
    st["out"] = torch.zeros_like(st["q"])
    return st


def _prepare_kv4_decode(case, seed):
    return _prepare_decode(case, seed, True)


def _prepare_weights(case, seed):
    return _prepare_decode(case, seed, False)


def _plain_rows(st, name):
    """[batch, max_len, kv heads, d] in 32 bits, read through the block tables."""
    t = st["tables"]
    if st["op"] == "kv4_decode":
        codes, scales = st[name]
        x = _plain_dequantise(codes[t], scales[t])
    else:
        x = st[name][t].float()
    return x.flatten(1, 2)[:, : st["stride"]]


def _plain_decode(st):
    b, hkv, d = st["batch"], st["hkv"], st["d"]
    live = torch.arange(st["stride"], device="cuda")[None, :] < st["lens"][:, None]
    q = st["q"].float().view(b, hkv, -1, d)
    s = torch.matmul(q, _plain_rows(st, "k").permute(0, 2, 3, 1)) * st["scale"]
    s = torch.where(live[:, None, None, :], s, torch.full_like(s, -math.inf))
    e = torch.exp(s - s.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    out = torch.matmul(w, _plain_rows(st, "v").transpose(1, 2))
    out = out.view(b, st["hq"], d).to(st["q"].dtype)
    if "w_in" not in st:
        return out
    st["w_out"].copy_(torch.where(live[:, None, :], st["w_in"] + w.sum(2), st["w_out"]))
    return [out, st["w_out"]]


_plain_kv4_decode = _plain_weights = _plain_decode


def _own_decode(st):
    pool = st["pool"].pool
    kw = {}
    if "w_in" in st:
        kw = dict(weights_in_ptr=st["w_in"].data_ptr(), weights_out_ptr=st["w_out"].data_ptr(),
                  weights_row_stride=st["stride"])
    call = pool.kv4_paged_attn_decode if st["op"] == "kv4_decode" else pool.paged_attn_decode_weights
    call(0, query_ptr=st["q"].data_ptr(), out_ptr=st["out"].data_ptr(),
         block_tables_ptr=st["tables"].data_ptr(), seq_lens_ptr=st["lens"].data_ptr(),
         block_offsets_f16_ptr=st["pool"].offsets.data_ptr(), batch=st["batch"],
         num_q_heads=st["hq"], kv_heads=st["hkv"], head_dim=st["d"], block_size=_BS,
         max_blocks_per_seq=st["tables"].shape[1], scale=st["scale"], dtype=st["dtype"],
         stream_ptr=_stream(), **kw)
    return [st["out"], st["w_out"]] if kw else st["out"]


_own_kv4_decode = _own_weights = _own_decode


def _exact_decode(case, seed):
    kv4 = case["op"] == "kv4_decode"
    lens, tables, _, _, k, v = _page_rows(case, seed, _kv_page_bytes(case))
    q = _queries(case, seed).double()
    group = case["hq"] // case["hkv"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    wants = not kv4 or case["weights"]
    if wants:
        w_in = _start_weights(case, seed, int(case["max_len"])).double()
        w_out = torch.zeros_like(w_in)
    for b, n in enumerate(lens):
        t = np.arange(int(n))
        rows = torch.from_numpy(tables[b, t // _BS] * _BS + t % _BS).cuda()
        kb, vb = ((_exact_quantised(x[rows]) if kv4 else x[rows].double()) for x in (k, v))
        for h in range(case["hkv"]):
            qh = q[b, h * group:(h + 1) * group]
            p = torch.softmax(qh @ kb[:, h].T / math.sqrt(case["d"]), dim=1)
            out[b, h * group:(h + 1) * group] = p @ vb[:, h]
            if wants:
                w_out[b, h, : int(n)] = w_in[b, h, : int(n)] + p.sum(dim=0)
    return [out, w_out] if wants else out


_exact_kv4_decode = _exact_weights = _exact_decode


# --- evict ---------------------------------------------------------------------------------


def _prepare_evict(case, seed):
    page_bytes = _kv_page_bytes(case)
    lens, tables, total, per, k, v = _page_rows(case, seed, page_bytes)
    stride = int(case["max_len"])
    pos, kept, nxt = _evict_state(case, seed, lens)
    st = dict(case, stride=stride, lens=torch.from_numpy(lens.astype(np.int32)).cuda(),
              w_in=_start_weights(case, seed, stride), pos_in=torch.from_numpy(pos).cuda(),
              kept=torch.from_numpy(kept).cuda(), next_pos=torch.from_numpy(nxt).cuda())
    st["w_out"], st["pos_out"] = torch.zeros_like(st["w_in"]), torch.zeros_like(st["pos_in"])
    st["new_lens"] = torch.zeros_like(st["lens"])
    elems = _BS * case["hkv"] * case["d"]
    if not own:
        st["tables"] = torch.from_numpy(tables).cuda()
        st["pages"] = [x.view(total // per, per, elems) for x in (k, v)]
        return st
    p = _Pool(case["hkv"], case["d"], total, case["batch"])
    st["pool"], st["tables"] = p, p.tables(tables)
    st["pages"] = [p.region(n, total, per, elems, x.dtype) for n, x in (("k", k), ("v", v))]
    for dst, x in zip(st["pages"], (k, v)):
        dst.copy_(x.view(dst.shape))
    return st


def _plain_evict(st):
    b_n, h_n, stride, budget = st["batch"], st["hkv"], st["stride"], st["budget"]
    idx = torch.arange(stride, device="cuda")
    lens, nxt = st["lens"].long()[:, None], st["next_pos"].long()[:, None]
    live = (idx[None, :] < lens)[:, None, :].expand(b_n, h_n, stride)
    fresh = (idx[None, :] + (nxt - lens))[:, None, :]
    pos = torch.where((idx[None, :] < st["kept"].long()[:, None])[:, None, :],
                      st["pos_in"].long(), fresh)
    held = live & ((pos < st["sinks"]) | (pos >= (nxt - st["recent"])[:, None, :]))
    w = st["w_in"]
    # rank: held first, then by weight, then by index; slots past the length last
    key = torch.where(live, w, torch.full_like(w, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    cls = torch.where(held, 2, torch.where(live, 1, 0))
    order = order.gather(-1, torch.sort(cls.gather(-1, order), dim=-1, descending=True,
                                        stable=True).indices)
    rank = torch.empty_like(order).scatter_(-1, order, idx.expand(b_n, h_n, stride).contiguous())
    keep = live & (rank < budget)
    hole = live & ~keep & (idx < budget)
    move = keep & (idx >= budget)
    b, h, src = move.nonzero(as_tuple=True)
    bd, hd, dst = hole.nonzero(as_tuple=True)
    # sequences no longer than the budget have neither; elsewhere the counts agree per row
    new_lens = torch.minimum(st["lens"], torch.full_like(st["lens"], budget))
    inside = (idx[None, :] < new_lens[:, None])[:, None, :]
    w_out = torch.where(inside, w, torch.zeros_like(w))
    p_out = torch.where(inside, pos, torch.zeros_like(pos))
    w_out[bd, hd, dst] = w[b, h, src]
    p_out[bd, hd, dst] = pos[b, h, src]
    st["w_out"].copy_(torch.where(live, w_out, st["w_out"]))
    st["pos_out"].copy_(torch.where(inside, p_out, st["pos_out"].long()))
    st["new_lens"].copy_(new_lens)
    t = st["tables"]
    rs, rd = t[b, src // _BS] * _BS + src % _BS, t[bd, dst // _BS] * _BS + dst % _BS
    for x in st["pages"]:
        rows = x.view(-1, h_n, st["d"])
        rows[rd, hd] = rows[rs, h]
    return [st["new_lens"], st["w_out"], st["pos_out"]] + st["pages"]


def _own_evict(st):
    st["pool"].pool.evict_tokens(
        0, head_dim=st["d"], block_tables_ptr=st["tables"].data_ptr(),
        seq_lens_ptr=st["lens"].data_ptr(),
        block_offsets_f16_ptr=st["pool"].offsets.data_ptr(), batch=st["batch"],
        max_blocks_per_seq=st["tables"].shape[1], budget=st["budget"], sinks=st["sinks"],
        recent=st["recent"], weights_in_ptr=st["w_in"].data_ptr(),
        weights_out_ptr=st["w_out"].data_ptr(), weights_row_stride=st["stride"],
        positions_in_ptr=st["pos_in"].data_ptr(), positions_out_ptr=st["pos_out"].data_ptr(),
        next_positions_ptr=st["next_pos"].data_ptr(), kept_lens_ptr=st["kept"].data_ptr(),
        new_lens_ptr=st["new_lens"].data_ptr(), stream_ptr=_stream())
    return [st["new_lens"], st["w_out"], st["pos_out"]] + st["pages"]


def _exact_evict(case, seed):
    lens, tables, total, per, k, v = _page_rows(case, seed, _kv_page_bytes(case))
    pos_in, kept_lens, nxt = _evict_state(case, seed, lens)
    w = _start_weights(case, seed, int(case["max_len"])).cpu().numpy().astype(np.float64)
    w_out, p_out = np.zeros_like(w), np.zeros_like(pos_in)
    src_rows, dst_rows, heads = [], [], []
    for b, n in enumerate(int(x) for x in lens):
        m = min(n, case["budget"])
        for h in range(case["hkv"]):
            pos = np.arange(n) + int(nxt[b]) - n
            pos[: kept_lens[b]] = pos_in[b, h, : kept_lens[b]]
            stay = (pos < case["sinks"]) | (pos >= int(nxt[b]) - case["recent"])
            best = np.lexsort((np.arange(n), -w[b, h, :n], ~stay))[:m]
            kept = np.zeros(n, bool)
            kept[best] = True
            src = np.arange(n)[:m].copy()
            free = np.flatnonzero(~kept[:m])
            src[free] = m + np.flatnonzero(kept[m:])
            w_out[b, h, :m], p_out[b, h, :m] = w[b, h, src], pos[src]
            slot = tables[b, np.arange(n) // _BS] * _BS + np.arange(n) % _BS
            src_rows.append(slot[src[free]])
            dst_rows.append(slot[free])
            heads.append(np.full(len(free), h))
    rs, rd, hh = (torch.from_numpy(np.concatenate(x)).cuda() for x in (src_rows, dst_rows, heads))
    pages = []
    for x in (k, v):  # rows move as they are, in the cache's own type
        moved = x.clone()
        moved[rd, hh] = x[rs, hh]
        pages.append(moved.view(total // per, per, -1))
    new = torch.from_numpy(np.minimum(lens, case["budget"]).astype(np.int32)).cuda()
    return [new, torch.from_numpy(w_out).cuda(), torch.from_numpy(p_out).cuda()] + pages


# --- beam ----------------------------------------------------------------------------------


def _prepare_beam(case, seed):
    logits, scores, hist, tables = _beam_inputs(case, seed)
    st = dict(case, logits=logits, scores=scores, hist=hist, tables=tables)
    if own:
        st["pool"] = _Pool(1, 64, 8, 1)
        b, n = case["batch"], case["select"]
        st["s_out"] = torch.empty(b, n, device="cuda")
        st["parents"] = torch.empty(b, n, dtype=torch.int32, device="cuda")
        st["tokens"] = torch.empty(b, n, dtype=torch.int32, device="cuda")
        st["hist_out"] = torch.empty(b, n, hist.shape[2], dtype=torch.int32, device="cuda")
        st["tables_out"] = torch.empty(b, n, tables.shape[2], dtype=torch.int32, device="cuda")
    return st


def _plain_beam(st):
    b_n, vocab, n = st["batch"], st["vocab"], st["select"]
    x = st["logits"].float()
    x = x - x.amax(-1, keepdim=True)
    x = x - torch.log(torch.exp(x).sum(-1, keepdim=True)) + st["scores"][..., None]
    x = x.view(b_n, -1)
    # 2n + 8 candidates, then their order by score and index
    s, i = torch.topk(x, min(2 * n + 8, x.shape[1]), dim=-1)
    i, by = torch.sort(i, dim=-1)
    s, by = torch.sort(s.gather(-1, by), dim=-1, descending=True, stable=True)
    s, i = s[:, :n], i.gather(-1, by)[:, :n]
    parents, tokens = i // vocab, i % vocab
    rows = torch.arange(b_n, device="cuda")[:, None]
    hist = st["hist"][rows, parents]
    hist[:, :, st["history"]] = tokens.int()
    return [s, parents.int(), tokens.int(), hist, st["tables"][rows, parents]]


def _own_beam(st):
    pool, stream = st["pool"].pool, _stream()
    pool.beam_select(logits_ptr=st["logits"].data_ptr(), dtype=st["dtype"],
                     scores_in_ptr=st["scores"].data_ptr(), batch=st["batch"], beams=st["beams"],
                     vocab=st["vocab"], n_select=st["select"], scores_out_ptr=st["s_out"].data_ptr(),
                     parents_out_ptr=st["parents"].data_ptr(), tokens_out_ptr=st["tokens"].data_ptr(),
                     stream_ptr=stream)
    pool.beam_gather(src_ptr=st["hist"].data_ptr(), dst_ptr=st["hist_out"].data_ptr(),
                     row_bytes=4 * st["hist"].shape[2], parents_ptr=st["parents"].data_ptr(),
                     batch=st["batch"], beams=st["beams"], n_select=st["select"],
                     tokens_ptr=st["tokens"].data_ptr(), token_index=st["history"],
                     stream_ptr=stream)
    pool.beam_gather(src_ptr=st["tables"].data_ptr(), dst_ptr=st["tables_out"].data_ptr(),
                     row_bytes=4 * st["tables"].shape[2], parents_ptr=st["parents"].data_ptr(),
                     batch=st["batch"], beams=st["beams"], n_select=st["select"],
                     stream_ptr=stream)
    return [st["s_out"], st["parents"], st["tokens"], st["hist_out"], st["tables_out"]]


def _exact_beam(case, seed):
    logits, scores, hist, tables = _beam_inputs(case, seed)
    n, vocab = case["select"], case["vocab"]
    s_out, parents, tokens = [], [], []
    for b in range(case["batch"]):
        x = torch.log_softmax(logits[b].double(), dim=1) + scores[b].double()[:, None]
        x = x.reshape(-1).cpu().numpy()
        top = np.argpartition(-x, min(4 * n + 64, x.size) - 1)[: 4 * n + 64]
        top = top[np.lexsort((top, -x[top]))][:n]
        s_out.append(x[top])
        parents.append((top // vocab).astype(np.int32))
        tokens.append((top % vocab).astype(np.int32))
    parents = torch.from_numpy(np.stack(parents)).cuda()
    tokens = torch.from_numpy(np.stack(tokens)).cuda()
    h = torch.stack([hist[b][parents[b].long()] for b in range(case["batch"])])
    h[:, :, case["history"]] = tokens
    t = torch.stack([tables[b][parents[b].long()] for b in range(case["batch"])])
    return [torch.from_numpy(np.stack(s_out)).cuda(), parents, tokens, h, t]


def exact(case, seed):
    return globals()["_exact_" + case["op"]](case, seed)


# --- work ----------------------------------------------------------------------------------


def _mean_tokens(case):
    """Tokens of the batch: the ends are always drawn, the others uniform between them."""
    lo, hi, b = case["min_len"], case["max_len"], case["batch"]
    return hi if b == 1 else hi + lo + (b - 2) * (lo + hi) / 2


def work(case):
    op = case["op"]
    if op == "beam":
        e = 4 if case["dtype"] == "f32" else 2
        rows = case["batch"] * case["beams"]
        sel = case["batch"] * case["select"]
        state = 4 * (case["history"] + 1 + case["pages"])
        return {"bytes": rows * (case["vocab"] * e + 4) + sel * (12 + 2 * state),
                "flops": 4 * rows * case["vocab"]}
    row = case["hkv"] * case["d"]  # elements of a K or V row
    row4 = row * 9 // 16           # its bytes in the 4-bit cache
    if op == "kv4_store":
        t = case["tokens"]
        return {"bytes": t * (2 * (2 * row + row4 + row4 + 2 * row) + 8), "flops": 2 * t * 4 * row}
    n = _mean_tokens(case)
    if op == "evict":
        cut, b = case["budget"], case["batch"]
        mean = n / b
        moved = 0.0
        if mean > cut:
            rest = mean - case["recent"] - case["sinks"]
            share = (cut - case["recent"] - case["sinks"]) / max(rest, 1)
            tail = mean - cut
            moved = min(tail, case["recent"]) + max(0.0, tail - case["recent"]) * share
        moved *= b
        kept = b * min(mean, cut)
        pos_in = kept if case["again"] else 0
        return {"bytes": int(case["hkv"] * 4 * (2 * n + kept + pos_in) + moved * row * 8 + 16 * b),
                "flops": int(case["hkv"] * n)}
    per_token = 2 * row4 if op == "kv4_decode" else 4 * row
    if op == "weights" or case["weights"]:
        per_token += 8 * case["hkv"]
    return {"bytes": int(n * per_token + 4 * case["batch"] * case["hq"] * case["d"] + n / 4),
            "flops": int(4 * n * case["hq"] * case["d"])}
