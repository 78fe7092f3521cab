"""What the kernels of gated norms, rotary positions and attention within sequences rest on in the compiler's output, checked on the CPU (hipcc cross-compiles):

* No scratch memory in any loop that every call runs: in the attention's main loops a spill would be a wait for memory at every step.  (The way for sums that hold a NaN may spill.)
* Those loops wait for copies where the source says so and nowhere else.
* Registers that leave three workgroups of heads up to 64 (rows form) and two waves on a SIMD.
* No condition code is kept across inline assembly, and no request is made in a loop over the lanes' values.
"""

import re
import tempfile
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_build_guard import compile_variant, lane_by_lane_requests, scc_live_across_asm

UNITS = ("self_attention.hip", "gated_norm.hip", "rotary_axes.hip")


@pytest.fixture(scope="module")
def compiled():
    with tempfile.TemporaryDirectory(prefix="svdq_guard_") as tmp, ThreadPoolExecutor(max_workers=3) as pool:
        return dict(zip(UNITS, pool.map(lambda u: compile_variant(u, 0, tmp), UNITS)))


def bodies(lines, kernel):
    for first in (i for i, t in enumerate(lines) if re.match(rf"^_ZN\S*{kernel}\S*:", t)):
        yield lines[first], lines[first:next(i for i in range(first, len(lines)) if lines[i].startswith(".Lfunc_end"))]


def innermost_loops(body):
    """Line ranges of the loops with matrix instructions that hold no other such loop."""
    labels = {m.group(1): i for i, t in enumerate(body) if (m := re.match(r"^(\.LBB\w+):", t))}
    loops = {(labels[m.group(1)], i) for i, t in enumerate(body) if (m := re.match(r"^\ts_c?branch\w*\s+(\.LBB\w+)", t)) and labels.get(m.group(1), i) < i}
    loops = {(a, b) for a, b in loops if any("v_mfma" in t for t in body[a:b])}
    return [body[a:b] for a, b in sorted(loops) if not any(a <= c and d <= b and (a, b) != (c, d) for c, d in loops)]


def test_registers(compiled):
    usage, _ = compiled["self_attention.hip"]
    kernels = {k: u for k, u in usage.items() if "_kernel" in k}
    # two types; keys: five head sizes; rows: those and a column of ones, of 80 always; turns: above 64; joins: of 32 and 128 rows
    assert len(kernels) == 2 * (5 + 9 + 5 + 2), len(kernels)
    for name, u in kernels.items():
        rows, narrow = "rows_kernel" in name, re.search(r"kernelILb\dELi(32|64)E", name)
        wide_keys = "keys_kernel" in name and not narrow
        assert u["Occupancy"] >= (1 if wide_keys else 3 if rows and narrow else 2), (name, u)
        assert u["ScratchSize"] <= (160 if rows or "turns_kernel" in name else 0), (name, u)
    for unit, count in (("gated_norm.hip", 16), ("rotary_axes.hip", 32)):
        kernels = {k: u for k, u in compiled[unit][0].items() if "_kernel" in k}
        assert len(kernels) == count, (unit, len(kernels))
        assert all(u["ScratchSize"] == 0 for u in kernels.values()), unit


def test_main_loops(compiled):
    _, lines = compiled["self_attention.hip"]
    seen = {"rows": 0, "turns": 0}
    for form, barriers, waits in (("rows", 1, {"s_waitcnt vmcnt(0) lgkmcnt(0)"}), ("turns", 2, {"s_waitcnt vmcnt(0)", "s_waitcnt vmcnt(3)", "s_waitcnt vmcnt(4)"})):
        for name, body in bodies(lines, f"self_attention_{form}_kernel"):
            mains = []
            for loop in innermost_loops(body):
                steps = sum("s_barrier" in t for t in loop)
                # (the careful way's steps wait for both barriers' copies in place: no request is on its way across one)
                if steps == barriers and any("global_load_lds" in t for t in loop) and not any("scratch_" in t for t in loop):
                    if {t.strip() for t in loop if "s_waitcnt" in t and "vmcnt" in t} <= waits:
                        mains.append(loop)
            assert mains, name
            seen[form] += 1
    assert seen == {"rows": 18, "turns": 10}


@pytest.mark.parametrize("unit", UNITS)
def test_inline_assembly(compiled, unit):
    _, lines = compiled[unit]
    assert scc_live_across_asm(lines) == []
    plain = [re.sub(r"global_(load|store)", r"buffer_\1", t) for t in lines]
    # (such a loop's branch follows the exclusive or that takes the lanes served out of the mask; the end of an `if` looks the same but for that)
    ends = [i for i, t in enumerate(plain) if "s_cbranch_execnz" in t and "s_xor_b64 exec" in plain[i - 1]]
    assert lane_by_lane_requests([t for i in ends for t in plain[i - 8: i + 1]]) == {}
