"""CPU: the gfx950 code of the microscaled 4-bit operators and of the norms, as the compiler made it: no spilled vector
registers, the LDS copies (inline assembly that sets M0) with their wait state, no packed fp32 instructions, products in
the scaled instructions, and in the products' loop a wait for the reads of a stage before it is written again."""

from __future__ import annotations

import re

import pytest

from test_codegen import _device_asm, m0_lds_dma_hazards


@pytest.mark.parametrize("name,copies", [("mx_linear.hip", True), ("mx_quantize.hip", False), ("block_norm.hip", False)])
def test_operator_code(tmp_path, name, copies):
    text = _device_asm(tmp_path, name)
    counts = [int(c) for c in re.findall(r"\.vgpr_spill_count:\s+(\d+)", text)]
    assert counts and not any(counts), counts
    assert not re.search(r"^\s*scratch_(load|store)", text, re.M)
    assert not re.search(r"^\s*v_pk_(add|mul|fma)_f32", text, re.M)
    assert (text.count("global_load_lds_dwordx4") > 0) == copies
    assert not m0_lds_dma_hazards(text)
    if copies:
        assert "v_mfma_scale_f32_32x32x64_f8f6f4" in text and "v_mfma_scale_f32_16x16x128_f8f6f4" in text
        # No read of LDS is under way at a barrier, behind which its place is written again.
        assert sum(reads_at_barriers(f) for f in re.split(r"^\.Lfunc_end", text, flags=re.M)) == 0


def reads_at_barriers(function: str) -> int:
    """The barriers that some path reaches with an LDS read that no lgkmcnt(0) has waited for."""
    code, label = [], {}
    for line in function.splitlines():
        x = line.split(";")[0].strip()
        if re.match(r"\.LBB\w+:", x):
            label[x[:-1]] = len(code)
        elif x and not x.startswith((".", "_")):
            code.append(x)
    pending, todo, found = set(), [], 0
    for i, x in enumerate(code):
        if x.startswith("ds_read"):
            todo.append(i + 1)
    while todo:
        i = todo.pop()
        if i in pending or i >= len(code):
            continue
        pending.add(i)
        x = code[i]
        if "lgkmcnt(0)" in x or x.startswith("s_endpgm"):
            continue
        found += x == "s_barrier"
        if x.startswith(("s_cbranch", "s_branch")):
            todo.append(label[x.split()[1]])
        if not x.startswith("s_branch"):
            todo.append(i + 1)
    return found


def test_the_check_of_barriers_sees_a_missing_wait():
    loop = [".LBB0_1:", "ds_read_b128 v[0:3], v4", "s_cbranch_scc1 .LBB0_2", "s_waitcnt lgkmcnt(0)", ".LBB0_2:", "s_barrier",
            "s_branch .LBB0_1"]
    assert reads_at_barriers("\n".join(loop)) == 1
    loop[2], loop[3] = loop[3], loop[2]
    assert reads_at_barriers("\n".join(loop)) == 0
