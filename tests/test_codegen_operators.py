"""CPU: the gfx950 code of the operators around the experts' products, as the compiler made it: no spilled vector
registers, the LDS copies (inline assembly that sets M0) with their wait state, no packed fp32 instructions."""

from __future__ import annotations

import re

import pytest

from test_codegen import _device_asm, m0_lds_dma_hazards


@pytest.mark.parametrize("name,copies", [("linear_act_tiles.hip", True), ("linear_act.hip", False), ("token_sort.hip", False)])
def test_operator_code(tmp_path, name, copies):
    text = _device_asm(tmp_path, name)
    counts = [int(c) for c in re.findall(r"\.vgpr_spill_count:\s+(\d+)", text)]
    assert counts and not any(counts), counts
    assert not re.search(r"^\s*scratch_(load|store)", text, re.M)
    assert not re.search(r"^\s*v_pk_(add|mul|fma)_f32", text, re.M)
    assert (text.count("global_load_lds_dwordx4") > 0) == copies
    assert not m0_lds_dma_hazards(text)
