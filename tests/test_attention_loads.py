"""The prompt kernels' loads into LDS, read in the source: rows behind a sequence are kept out by the range check of the
buffer, which is certain to count a lane's own offset only.  No result can show a read past it (the mask hides the values)."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm_quantization-kernel_amd", "csrc")


def _arguments(text, at):
    """The arguments of the call whose opening bracket is at `at`."""
    depth, out, word = 0, [], ""
    for c in text[at:]:
        if c in "([{":
            depth += 1
            if depth == 1:
                continue
        elif c in ")]}":
            depth -= 1
            if depth == 0:
                return [*out, word.strip()]
        if c == "," and depth == 1:
            out.append(word.strip())
            word = ""
        else:
            word += c
    raise AssertionError("unbalanced call")


@pytest.mark.parametrize("name", ["prompt_attn.hip", "prompt_attn_f32.hip"])
def test_whole_offset_is_the_lanes(name):
    text = open(os.path.join(CSRC, name)).read()
    calls = [_arguments(text, m.end() - 1) for m in re.finditer(r"raw_ptr_buffer_load_lds\(", text)]
    assert calls
    for c in calls:                       # buffer, LDS, size, lane offset, scalar offset, constant offset, flags
        assert len(c) == 7 and c[4] == "0" and c[5] == "0", c
