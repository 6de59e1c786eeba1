"""Packed prompt attention at the ends of its ranges: values near the type's largest and smallest,
what an earlier call that failed leaves in the stream's scratch, and long items; against the
definition in 64 bits with the bound of `test_prompt_attn_gpu.py`."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from kv_cases import torch_cuda
from test_prompt_attn_gpu import HALF, call, inputs, pool, reference, starts  # noqa: F401

pytestmark = pytest.mark.gpu


def check_sequences(q, k, v, out, qs, ks, causal, dtype, scale):
    """As `check` there, without its absolute term: the values are of any size."""
    for b in range(len(qs) - 1):
        got = out[qs[b]:qs[b + 1]].double()
        ref, mass = reference(q[qs[b]:qs[b + 1]].double(), k[ks[b]:ks[b + 1]].double(),
                              v[ks[b]:ks[b + 1]].double(), scale, causal)
        bound = HALF[dtype] * (ref.abs() + mass) + 2.0 ** -12 * mass
        assert (got.isfinite() & ((got - ref).abs() <= bound)).all(), b


@pytest.mark.parametrize("size", [2e38, 1e-26])
@pytest.mark.parametrize("scores", ["equal", "flat", "peaked", "rising"])
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 4), (128, 8, 2), (80, 7, 1), (256, 3, 1)])
def test_large_and_small_values(pool, d, hq, hkv, scores, size):  # noqa: F811
    """bf16 values near the largest, of one sign by column or of both: the weighted mean is finite,
    the sum of the values is not.  Over one key, some and many, the last ones in parts."""
    torch = torch_cuda()
    nq, nk = [1, 3, 300, 130, 5], [1, 2, 300, 4000, 9000]
    qs, ks = starts(nq), starts(nk)
    q, k, v = inputs(sum(nq), sum(nk), hq, hkv, d, "bf16", 31, 12.0 if scores == "peaked" else 1.5)
    if scores == "equal":
        k.zero_()
    if scores == "rising":  # the running maximum lags behind every step's
        u = torch.ones(d, device="cuda") / d ** 0.5
        t = torch.cat([torch.linspace(0, 25 * n / 4000, n, device="cuda") for n in nk])
        k = (0.1 * k.float() + t[:, None, None] * u).to(k.dtype)
        q = (0.1 * q.float() + u * d ** 0.5).to(q.dtype)
    g = torch.Generator(device="cuda").manual_seed(32)
    v = size * (1 + 0.6 * torch.rand(v.shape, device="cuda", generator=g).double())
    v[..., d // 4:d // 2] *= -1
    v[..., 3 * d // 4:] *= torch.where(torch.arange(sum(nk), device="cuda") % 2 == 0, 1, -1)[
        :, None, None]
    v = v.to(q.dtype)
    for causal in (True, False):
        out = call(pool, q, k, v, torch.zeros_like(q), qs, ks, causal, "bf16", d ** -0.5)
        check_sequences(q, k, v, out, qs, ks, causal, "bf16", d ** -0.5)
    # few items: keys in parts
    out = call(pool, q[:1], k[:9000], v[:9000], torch.zeros_like(q[:1]), np.array([0, 1]),
               np.array([0, 9000]), True, "bf16", d ** -0.5)
    check_sequences(q[:1], k[:9000], v[:9000], out, np.array([0, 1]), np.array([0, 9000]), True,
                    "bf16", d ** -0.5)
    assert pool.kernel_status() == 0


class Scratch(ctypes.Structure):
    """`CallScratch` of `csrc/launch.hpp`: what a call holds of its stream's buffer."""
    _fields_ = [("ptr", ctypes.c_uint64), ("counters", ctypes.c_uint64),
                ("tickets", ctypes.c_uint64), ("ticket_base", ctypes.c_uint64),
                ("owned", ctypes.c_bool), ("mutex", ctypes.c_uint64), ("owns", ctypes.c_bool)]
    COUNTERS, TICKETS, RANGE = 65536, 2048, 32

    def __init__(self, lib, stream, nbytes):
        super().__init__()
        self.acquire = lib["_ZN4kcmm3dev11CallScratch7acquireEP11CUstream_stm"]
        self.release = lib["_ZN4kcmm3dev11CallScratch7releaseEP11CUstream_st"]
        for fn in (self.acquire, self.release):
            fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p] + [ctypes.c_size_t] * (
                fn is self.acquire)
        self.stream, self.nbytes = stream, nbytes

    def __enter__(self):
        assert self.acquire(ctypes.addressof(self), self.stream, self.nbytes) == 0
        assert not self.owned  # the stream's kept buffer
        return self

    def __exit__(self, *exc):
        assert self.release(ctypes.addressof(self), self.stream) == 0

    def words(self, at, count, dtype):
        """Device words as a tensor."""
        import torch

        class View:
            __cuda_array_interface__ = dict(shape=(count,), typestr=dtype, data=(at, False),
                                            version=2)

        return torch.as_tensor(View(), device="cuda")


def test_scratch_counts_start_anew_after_a_call_that_failed(pool):  # noqa: F811
    """Keys in parts, behind counts that an earlier call left where they stood when its waits ran
    out: every part is merged, whatever they were.  The earlier sums are NaN, so that one taken
    too early shows."""
    torch = torch_cuda()
    nq, nk, hq, hkv, d = [40, 1], [3000, 2500], 8, 1, 128
    qs, ks = starts(nq), starts(nk)
    stream = torch.cuda.current_stream().cuda_stream
    for left in (0, 1, 2, 7, 15, 16, Scratch.RANGE - 1):
        q, k, v = inputs(sum(nq), sum(nk), hq, hkv, d, "bf16", 40 + left)
        call(pool, q, k, v, torch.zeros_like(q), qs, ks, True, "bf16", 0.1)
        nbytes = sum(nq) * hq * 16 * (d + 2) * 4
        with Scratch(pool.lib, stream, nbytes) as held:
            assert not held.words(held.counters, held.COUNTERS, "<i4").any()
            tickets = held.words(held.tickets, held.TICKETS, "<i8")
            assert int(tickets.max()) < held.ticket_base
            tickets.fill_(held.ticket_base + left)
            held.words(held.ptr, nbytes // 4, "<i4").fill_(-1)
            torch.cuda.synchronize()
        for _ in range(2):
            out = call(pool, q, k, v, torch.zeros_like(q), qs, ks, True, "bf16", 0.1)
            check_sequences(q, k, v, out, qs, ks, True, "bf16", 0.1)
    assert pool.kernel_status() == 0


def test_an_item_that_takes_seconds(pool):  # noqa: F811
    """More items than are cut into parts, each over 200 million keys: some 1.5 million steps, of
    2000 to 3000 cycles.  The roles that wait for an item's end wait for longer than 2^31 cycles
    and do not give up.  The last keys outweigh all others by e^60."""
    torch = torch_cuda()
    nq, nk, last, d = 20480, 200_000_000, 100, 8
    q = torch.zeros(nq, 1, d, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1
    k = torch.zeros(nk, 1, d, dtype=torch.bfloat16, device="cuda")
    k[:-last, :, 0] = -60
    v = torch.ones_like(k)
    g = torch.Generator(device="cuda").manual_seed(51)
    v[-last:] = torch.randn(last, 1, d, device="cuda", generator=g).to(v.dtype)
    out = call(pool, q, k, v, torch.zeros_like(q), np.array([0, nq]), np.array([0, nk]), False,
               "bf16", 1.0)
    assert pool.kernel_status() == 0
    rows = v[-last:].double()
    ref, mass = rows.mean(0, keepdim=True), rows.abs().mean(0, keepdim=True)
    assert ((out.double() - ref).abs() <= HALF["bf16"] * (ref.abs() + mass)
            + 2.0 ** -12 * mass).all()
