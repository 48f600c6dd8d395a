"""One lane's signal stands for its whole warp, read from the kernels' sources (nothing here runs on a GPU).

Where lane 0 alone arrives on a barrier that hands memory over (a place of a ring or of a list that the warp has read, a tile
that it has written), the other lanes' accesses have to be behind them: nothing but ``__syncwarp()`` orders them before
the arrival, since lanes that diverged need not have come together.
"""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "tiny-vllm_b200" / "csrc"
ARRIVAL = re.compile(r"if \(lane == 0(?: && \w+)?\) \{?\s*ptx::mbar_arrive\(ptx::smem_u32\((\w+)")
SOURCES = [p for p in sorted(CSRC.glob("*.cu*")) if ARRIVAL.search(p.read_text())]
OWN = {"want_bar"}      # a request: it hands no memory over


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_a_lane_signals_for_its_warp_behind_the_whole_warp(path):
    code = re.sub(r"//[^\n]*", "", path.read_text())
    for m in ARRIVAL.finditer(code):
        if m.group(1) in OWN:
            continue
        before = code[:m.start()].rstrip()
        statement = before[max(before.rfind(e, 0, len(before) - 1) for e in ";{}") + 1:].strip()
        assert statement == "__syncwarp();", f"{m.group(0)} ... stands behind: {statement}"


def test_the_attention_kernels_are_among_them():
    assert {"attn_prefill.cu", "attn_decode.cu"} <= {p.name for p in SOURCES}
