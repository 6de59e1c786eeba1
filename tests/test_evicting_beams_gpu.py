"""The example runs the cache operators together: its invariants."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest

from kv_cases import torch_cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams", [1, 4])
def test_example(beams):
    torch_cuda()
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import evicting_beams as ex

    r = ex.generate(steps=90, beams=beams)
    again = ex.generate(steps=90, beams=beams)
    assert r["kernel_status"] == 0 and r["cuts"] == (70 + 90 - 96 - 1) // 17
    assert r["position"] == 160 and r["cached"] == 96 + (160 - 112 - 1) % 17
    assert bool((r["tokens"] >= 0).all()) and bool((r["tokens"] < ex.VOCAB).all())
    # best first; beams are distinct continuations
    assert r["scores"].tolist() == sorted(r["scores"].tolist(), reverse=True)
    assert len({tuple(t) for t in r["tokens"].tolist()}) == beams
    # sinks and the recent window of the last cut stay, no position twice
    for row in r["positions"].reshape(-1, 96).tolist():
        assert len(set(row)) == 96 and set(range(4)) <= set(row)
        last = max(row)
        assert set(range(last - 31, last + 1)) <= set(row)
    used = {b for t in r["block_tables"] for b in t}
    assert r["blocks"] == len(used)  # nothing leaked
    assert (r["tokens"] == again["tokens"]).all() and (r["scores"] == again["scores"]).all()
