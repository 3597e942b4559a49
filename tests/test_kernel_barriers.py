"""Barriers that kernels keep and no compiler checks: read from the sources."""

import re
from pathlib import Path

KERNELS = Path(__file__).resolve().parent.parent / "llama-cuda-runtime_amd" / "csrc" / "kernels"


def function_body(text, name):
    """The braces of the function `name`, comments taken out."""
    text = re.sub(r"//[^\n]*", "", text)
    start = text.index("{", re.search(rf"\b{name}\([^;{{]*\)\s*(?={{)", text).end() - 1)
    depth = 0
    for i in range(start, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start:i + 1]
    raise AssertionError(name)


def test_a_draw_leaves_its_shared_memory_free():
    """draw_index is called again on the same shared memory where its first draw
    finds no weight, so each of its returns stands behind a barrier that no read
    of that memory follows."""
    body = function_body((KERNELS / "k_batch_verify.hip").read_text(), "draw_index")
    # the lambda's own return is none of the function's
    returns = [m.start() for m in re.finditer(r"\breturn\b", body)]
    assert len(returns) >= 2
    for at in returns:
        since = body[:at].rsplit("__syncthreads();", 1)
        assert len(since) == 2 and "lds." not in since[1], body[max(0, at - 200):at + 40]
