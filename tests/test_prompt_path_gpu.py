"""The prompt operators together, as a serving loop uses them: two packed prompts are rotated into
the cache and attended, one goes on with a chunk behind what was read back from the cache, and
decode steps rotate, append and attend single tokens; over a 16-bit and a 4-bit cache, on a stream
of their own, against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from kv_cases import Cache, attention, check_decode, quantised, torch_cuda
from test_prompt_attn_gpu import HALF, reference, starts
from test_rope_append_gpu import rotate, same

pytestmark = pytest.mark.gpu

HQ, HKV, D, ROT = 8, 2, 64, 64
SECTIONS = [12, 10, 10]


def bounded(got, ref, mass, dtype):
    over = (got.double() - ref).abs() - (HALF[dtype] * (ref.abs() + mass) + 2.0 ** -12 * mass + 1e-7)
    assert (over <= 0).all(), float(over.max())


class Loop:
    def __init__(self, dtype, kv4, lens):
        torch = torch_cuda()
        self.dtype, self.kv4 = dtype, kv4
        self.tdt = torch.bfloat16 if dtype == "bf16" else torch.float16
        self.cache = Cache(lens, HKV, D, kv4=kv4, dtype=dtype, seed=21)
        self.inv_freq = torch.from_numpy(
            (1e4 ** (-2.0 * np.arange(ROT // 2) / ROT)).astype(np.float32))
        self.d_freq = self.inv_freq.cuda()
        self.g = torch.Generator().manual_seed(22)
        self.scale = D ** -0.5
        self.held = [([], []) for _ in lens]  # rotated k and v rows of each sequence, 16 bits

    def rows(self, n):
        torch = torch_cuda()
        return (1.5 * torch.randn(n, HQ + 2 * HKV, D, generator=self.g)).to(self.tdt)

    def append(self, qkv, seqs, first, pos):
        """Rows of the sequences (count each) from the given positions on; q_out and k_out."""
        torch = torch_cuda()
        from lattice_b200 import kcmm

        dev = qkv.cuda()
        slots = np.concatenate([self.cache.slots(b, np.arange(f, f + n))
                                for (b, n), f in zip(seqs, first)])
        n = len(slots)
        self.keep = (dev, torch.from_numpy(slots).cuda(), torch.from_numpy(pos).cuda())
        q_out = torch.empty(n, HQ, D, dtype=self.tdt, device="cuda")
        k_out = torch.empty(n, HKV, D, dtype=self.tdt, device="cuda")
        rope = kcmm.make_rope(rotary_dim=ROT, inv_freq_ptr=self.d_freq.data_ptr(),
                              positions_ptr=self.keep[2].data_ptr(), sections=SECTIONS)
        row = dev.stride(0)
        self.cache.pool.rope_append(
            0, rope=rope, head_dim=D, num_q_heads=HQ, q_ptr=dev.data_ptr(), q_stride_token=row,
            q_out_ptr=q_out.data_ptr(), k_ptr=dev[:, HQ:].data_ptr(), k_row_stride=row,
            v_ptr=dev[:, HQ + HKV:].data_ptr(), v_row_stride=row, k_out_ptr=k_out.data_ptr(),
            slot_mapping_ptr=self.keep[1].data_ptr(),
            block_offsets_f16_ptr=self.cache.d_offsets.data_ptr(),
            block_offsets_f16_len=len(self.cache.offsets), num_tokens=n,
            cache_format=int(self.kv4), status_ptr=self.cache.status.data_ptr(), dtype=self.dtype,
            stream_ptr=torch.cuda.current_stream().cuda_stream)
        turned = rotate(qkv[:, :HQ + HKV], pos, self.inv_freq, ROT, SECTIONS, "neox", "sections")
        at = 0
        for b, m in seqs:
            self.held[b][0].append(turned[at:at + m, HQ:])
            self.held[b][1].append(qkv[at:at + m, HQ + HKV:])
            at += m
        assert same(q_out.cpu(), turned[:, :HQ]) and same(k_out.cpu(), turned[:, HQ:])
        return q_out, k_out, dev[:, HQ + HKV:]

    def attend(self, q, k, v, nq, nk):
        torch = torch_cuda()
        qs, ks = (torch.from_numpy(starts(x).astype(np.int32)).cuda() for x in (nq, nk))
        out = torch.full_like(q, 7.0)
        self.cache.pool.prompt_attn(
            query_ptr=q.data_ptr(), key_ptr=k.data_ptr(), k_stride_token=k.stride(0),
            value_ptr=v.data_ptr(), v_stride_token=v.stride(0), out_ptr=out.data_ptr(),
            q_start_ptr=qs.data_ptr(), k_start_ptr=ks.data_ptr(), batch=len(nq),
            num_q_tokens=q.shape[0], num_k_tokens=k.shape[0], num_q_heads=HQ, kv_heads=HKV,
            head_dim=D, scale=self.scale, dtype=self.dtype,
            stream_ptr=torch.cuda.current_stream().cuda_stream)
        torch.cuda.current_stream().synchronize()
        return out

    def held_values(self, b):
        """float64 rows that attention over the cache sees."""
        import torch

        k, v = (torch.cat(x).double().numpy() for x in self.held[b])
        return (quantised(k), quantised(v)) if self.kv4 else (k, v)


@pytest.mark.parametrize("kv4", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_prompts_chunk_and_decode(dtype, kv4):
    torch = torch_cuda()
    torch.cuda.synchronize()
    prompts, chunk, steps = [150, 41], 70, 3
    total = [prompts[0] + chunk + steps, prompts[1] + steps]
    r = np.random.default_rng(23)
    with torch.cuda.stream(torch.cuda.Stream()):
        loop = Loop(dtype, kv4, total)
        # prompts with image tokens: three positions a token
        pos = r.integers(0, 400, (3, sum(prompts))).astype(np.int32)
        qkv = loop.rows(sum(prompts))
        q, k, v = loop.append(qkv, list(enumerate(prompts)), [0, 0], pos)
        out = loop.attend(q, k, v, prompts, prompts)
        at = 0
        for n in prompts:
            ref, mass = reference(*(x[at:at + n].double() for x in (q, k, v)), loop.scale, True)
            bounded(out[at:at + n], ref, mass, dtype)
            at += n
        # a chunk of the first sequence: its past from the cache, its own rows as they are
        pos = np.tile(np.arange(400, 400 + chunk, dtype=np.int32), (3, 1))
        q, k, v = loop.append(loop.rows(chunk), [(0, chunk)], [prompts[0]], pos)
        past = loop.cache.read(loop.cache.slots(0, np.arange(prompts[0])))
        k, v = (torch.cat((x, y)) for x, y in zip(past, (k, v)))
        out = loop.attend(q, k, v, [chunk], [prompts[0] + chunk])
        ref, mass = reference(q.double(), k.double(), v.double(), loop.scale, True)
        bounded(out, ref, mass, dtype)
        # decode: a token of each sequence a step
        lens = [prompts[0] + chunk, prompts[1]]
        for step in range(steps):
            pos = np.tile(np.array([470 + step, 400 + step], np.int32), (3, 1))
            q, _, _ = loop.append(loop.rows(2), [(0, 1), (1, 1)], lens, pos)
            lens = [n + 1 for n in lens]
            loop.cache.lens = np.array(lens)
            loop.cache.d_lens.copy_(torch.from_numpy(np.array(lens, np.int32)))
            out = torch.zeros_like(q)
            rows = [loop.held_values(b) for b in range(2)]
            if kv4:
                loop.cache.decode(q, loop.scale, out)
                check_decode(loop.cache, rows, q, out, loop.scale)
            else:
                call = getattr(loop.cache.pool.lib, f"kcmm_paged_attn_decode_{dtype}_on_stream")
                assert call(loop.cache.pool.handle, 0, q.data_ptr(), out.data_ptr(),
                            loop.cache.d_tables.data_ptr(), loop.cache.d_lens.data_ptr(),
                            loop.cache.d_offsets.data_ptr(), 2, HQ, HKV, D, 16,
                            loop.cache.max_bps, loop.scale,
                            torch.cuda.current_stream().cuda_stream) == 0
                torch.cuda.current_stream().synchronize()
                for b in range(2):
                    ref, mass, _ = attention(q[b].double().cpu().numpy(), *rows[b], loop.scale)
                    err = np.abs(out[b].double().cpu().numpy() - ref)
                    assert (err <= HALF[dtype] * (np.abs(ref) + mass) + 2.0 ** -12 * mass).all()
        assert int(loop.cache.status.item()) == 0 and loop.cache.pool.kernel_status() == 0
    loop.cache.close()


def test_two_streams_at_once():
    """Prompts on two streams from two threads, each with its own scratch."""
    import threading

    torch = torch_cuda()
    loops, errors = [], []

    def work(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                loop = Loop("bf16", False, [1300])
                loops.append(loop)
                for i in range(8):
                    g = torch.Generator(device="cuda").manual_seed(seed + i)
                    n, m = (64, 1300) if i % 2 else (1300, 1300)  # in parts, and whole
                    q = torch.randn(n, HQ, D, device="cuda", generator=g).to(loop.tdt)
                    k, v = (torch.randn(m, HKV, D, device="cuda", generator=g).to(loop.tdt)
                            for _ in "kv")
                    out = loop.attend(q, k, v, [n], [m])
                    ref, mass = reference(q.double(), k.double(), v.double(), loop.scale, True)
                    bounded(out, ref, mass, "bf16")
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(100 * s,)) for s in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for loop in loops:
        loop.cache.close()
    assert not errors, errors
