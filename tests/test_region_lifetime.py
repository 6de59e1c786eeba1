"""A pool's regions stay mapped while an address of theirs, or a tensor over one, is held."""
from __future__ import annotations

import copy
import gc
import pickle

import numpy as np
import pytest

from lattice_b200 import KcmmError, kcmm


def mapped(address):
    with open("/proc/self/maps") as f:
        spans = [[int(x, 16) for x in line.split()[0].split("-")] for line in f]
    return any(a <= address < b for a, b in spans)


def test_destroy_waits_for_the_last_address(host_pool_factory):
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=2, max_seq_len=64)
    k, v = pool.va_k(0), pool.va_v(1)
    where = int(k)
    pool.destroy()
    assert mapped(where)
    with pytest.raises(KcmmError, match="destroyed"):
        pool.va_k(0)
    copies = [copy.deepcopy(k), pickle.loads(pickle.dumps(k))]
    assert copies == [where, where] and {type(x) for x in copies} == {int}
    del k
    assert mapped(where)  # a region's address holds them all
    del v
    assert not mapped(where)


def test_destroy_releases_at_once(host_pool_factory):
    """Nothing is held: by no address, by one that is gone, by a plain int, by a dead cycle."""
    pool = host_pool_factory(kv_heads=2, head_dim=64, max_batch=2, max_seq_len=64)
    where = pool.va_k(0) + 0

    class View:
        interface = {"data": (pool.va_k(0), False)}

    gc.disable()
    try:
        del View  # a class lies in a cycle of its own
        assert mapped(where)
        pool.destroy()
        assert not mapped(where)
    finally:
        gc.enable()
    pool.destroy()


@pytest.mark.gpu
def test_tensor_outlives_its_pool():
    import torch

    from lattice_b200 import workloads

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")

    class Owner:
        def __init__(self):
            self.pool = workloads.library().create_pool(kcmm.make_config(
                num_layers=1, kv_heads=2, head_dim=64, max_batch=1, max_seq_len=64))
            self.pool.alloc_blocks(4)

        def __del__(self):
            self.pool.destroy()

        def view(self):
            class View:
                __cuda_array_interface__ = {"shape": (4096,), "typestr": "<i2",
                                            "data": (self.pool.va_k(0), False), "version": 3}

            return torch.as_tensor(View(), device="cuda")

    owner = Owner()
    held = owner.pool._regions
    t = owner.view()
    t.copy_(torch.arange(4096, dtype=torch.int16))
    t = t.view(64, 64)[::2]  # a view of the tensor holds them as well
    del owner
    gc.collect()
    assert held.closed
    del held
    assert np.array_equal(t.cpu().numpy(), np.arange(4096, dtype=np.int16).reshape(64, 64)[::2])
