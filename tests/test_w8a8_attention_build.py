"""What the 8-bit operators' and attention's kernels rest on in the compiler's output, checked on the CPU (hipcc cross-compiles):

* No scratch memory, but for the epilogue of the 256 x 256 tiles; registers that leave two waves on a SIMD.
* The loop over the keys waits for memory where the source says so, in front of the barrier, and nowhere else: a wait that the compiler
  adds for another load would also be one for the copies just asked for, at every step.
* No condition code is kept across inline assembly, and no request is made in a loop over the lanes' values.
"""

import re
import tempfile
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_build_guard import compile_variant, lane_by_lane_requests, scc_live_across_asm

UNITS = ("attention.hip", "w8a8_gemm.hip", "w8a8_quantize.hip")


@pytest.fixture(scope="module")
def compiled():
    with tempfile.TemporaryDirectory(prefix="svdq_guard_") as tmp, ThreadPoolExecutor(max_workers=3) as pool:
        return dict(zip(UNITS, pool.map(lambda u: compile_variant(u, 0, tmp), UNITS)))


@pytest.mark.parametrize("unit", UNITS)
def test_registers(compiled, unit):
    usage, _ = compiled[unit]
    kernels = {k: u for k, u in usage.items() if "_kernel" in k}
    assert len(kernels) == {"attention.hip": 60, "w8a8_gemm.hip": 9, "w8a8_quantize.hip": 60}[unit], len(kernels)
    for name, u in kernels.items():
        whole = "w8a8_tiles_kernelILi256ELi256" in name
        assert u["ScratchSize"] <= (96 if whole else 0), (name, u)
        wide_keys = "attention_keys_kernel" in name and "Li128E" in name  # (a workgroup has the compute unit's LDS to itself there)
        assert u["Occupancy"] >= (1 if wide_keys else 2), (name, u)


def loop_around(lines, at):
    """The lines of the innermost loop that holds line ``at``."""
    labels = {m.group(1): i for i, t in enumerate(lines[:at]) if (m := re.match(r"^(\.LBB\w+):", t))}
    for i in range(at, len(lines)):
        m = re.match(r"^\ts_c?branch\w*\s+(\.LBB\w+)", lines[i])
        if m and m.group(1) in labels:
            return lines[labels[m.group(1)]: i]
    return []


def test_the_loop_over_the_keys_waits_where_it_says(compiled):
    _, lines = compiled["attention.hip"]
    starts = [i for i, t in enumerate(lines) if re.match(r"^_ZN\S*attention_rows_kernel\S*:", t)]
    seen = 0
    for first in starts:
        if not re.search(r"Li\d+ELb0ELb\dE", lines[first]):  # (with a mask: its bytes are loads of their own)
            continue
        body = lines[first:next(i for i in range(first, len(lines)) if lines[i].startswith(".Lfunc_end"))]
        barrier = [i for i, t in enumerate(body) if "s_barrier" in t and "s_waitcnt vmcnt(0) lgkmcnt(0)" in body[i - 1]]
        assert len(barrier) == 1, (lines[first], barrier)
        loop = loop_around(body, barrier[0])
        assert sum("global_load_lds" in t for t in loop) > 0 and sum("v_mfma" in t for t in loop) > 0
        waits = [t.strip() for t in loop if "s_waitcnt" in t and "vmcnt" in t]
        assert waits == ["s_waitcnt vmcnt(0) lgkmcnt(0)"], (lines[first], waits)
        seen += 1
    assert seen == 18  # five head sizes, two types, with a column of ones and (where the head ends on 32 columns) without


@pytest.mark.parametrize("unit", UNITS)
def test_inline_assembly(compiled, unit):
    _, lines = compiled[unit]
    assert scc_live_across_asm(lines) == []
    plain = [re.sub(r"global_(load|store)", r"buffer_\1", t) for t in lines]
    # (such a loop's branch follows the exclusive or that takes the lanes served out of the mask; the end of an `if` looks the same but for that)
    ends = [i for i, t in enumerate(plain) if "s_cbranch_execnz" in t and "s_xor_b64 exec" in plain[i - 1]]
    assert lane_by_lane_requests([t for i in ends for t in plain[i - 8: i + 1]]) == {}
