"""shared_attn.hip's scalar inline assembly must not break the compiler's own use of SCC and m0 (the
checks of test_isa_carry.py), and nothing of it may be spilled to memory.  Compile only, no GPU."""
import re
import subprocess
from pathlib import Path

import pytest

from test_isa_carry import CSRC, FLAGS, HIPCC, carry_hazards, m0_hazards


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")
def test_shared_attention():
    asm = subprocess.run([HIPCC, *FLAGS, str(CSRC / "shared_attn.hip")], capture_output=True, text=True,
                         check=True, timeout=600).stdout
    assert "s_addc_u32" in asm and " lds" in asm
    assert carry_hazards(asm) == []
    assert m0_hazards(asm) == []
    for field in ("vgpr_spill_count", "private_segment_fixed_size"):
        assert set(re.findall(rf"\.{field}:\s+(\d+)", asm)) == {"0"}
    assert not re.search(r"v_pk_(add|mul|fma)_f32", asm)
