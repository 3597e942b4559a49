"""Rules that the kernels' sources keep and no compiler checks."""

import re
from pathlib import Path

KERNELS = Path(__file__).resolve().parent.parent / "llama-cuda-runtime_amd" / "csrc" / "kernels"


def test_scalar_addresses_of_inline_loads_are_waited_for():
    """A memory instruction may read a scalar register five wait states after a
    vector instruction wrote it (gfx9). The compiler keeps that distance for its
    own instructions only: inline assembly that reads an address from scalar
    registers begins with `s_nop 4`."""
    found = 0
    for path in sorted(KERNELS.iterdir()):
        for m in re.finditer(r'asm volatile\(\s*"([^;]*?)\);', path.read_text(), re.S):
            code, *operands = m.group(0).split(":")
            if re.search(r"(global|buffer|scratch|flat)_", code) and any(re.search(r'"s"\(', o) for o in operands):
                found += 1
                assert m.group(1).startswith("s_nop 4"), (path.name, m.group(0))
    assert found >= 1
