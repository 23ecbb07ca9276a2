"""When a kernel lets the next one in: read from the sources, since a release that comes too early shows in a run by chance only."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "nano-vllm_b200", "csrc")


def code(name):
    """A source without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def body(text, function):
    """What stands between the braces of a function."""
    begin = text.index("{", text.index(function + "("))
    depth = 0
    for i in range(begin, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[begin + 1:i]
    raise AssertionError(function)


def test_a_release_of_results_waits_for_the_whole_cta():
    """One thread's release counts for its CTA: each thread's stores are fenced before a barrier, and the release comes behind that."""
    assert re.fullmatch(r"\s*__threadfence\(\);\s*__syncthreads\(\);\s*pdl_launch_dependents\(\);\s*", body(code("b2_common.cuh"), "void pdl_release_results"))


# kernels whose lengths and tables decode attention reads ahead of its dependency wait
@pytest.mark.parametrize("name, kernel", [("b2_batch.cu", "batch_inputs_kernel"), ("b2_elementwise.cu", "advance_decode_kernel")])
def test_what_is_read_ahead_is_released_at_the_end(name, kernel):
    text = body(code(name), kernel)
    assert "pdl_launch_dependents" not in text and "return;" not in text
    assert text.rstrip().endswith("b2::pdl_release_results();")
