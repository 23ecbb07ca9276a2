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


def kernels(text):
    return re.findall(r"__global__\s+void\s+(?:__launch_bounds__\([^;{]*?\)\s+)?(\w+)\(", text)


def test_columns_are_allocated_before_the_next_kernel_is_let_in():
    """A kernel that is let in early keeps its columns of tensor memory until this one has ended, so this one's CTA must have its own by then: the
    release stands behind a barrier that the allocating warp meets with its columns."""
    found = []
    for name in sorted(os.listdir(CSRC)):
        text = code(name)
        for kernel in kernels(text):
            inside = body(text, kernel)
            if "tmem_alloc" not in inside:
                continue
            found.append(kernel)
            before, after = inside.split("tmem_alloc", 1)
            assert "pdl_launch_dependents" not in before, kernel
            if "pdl_launch_dependents" in after:  # (or in a function that runs at the end)
                assert "__syncthreads();" in after[:after.index("pdl_launch_dependents")], kernel
    assert {"tree_attention_kernel", "prefill_attention_kernel", "gemm_kernel", "gemm_tile_kernel", "gemm_pair_kernel"} <= set(found), found


def test_reordered_tables_are_released_at_the_end():
    """Decode attention may follow beam_move_kernel, the last of the two that write tables and lengths; the first lets nothing but the second in, which waits for all of it."""
    text = body(code("b2_beam.cu"), "beam_move_kernel")
    assert "pdl_launch_dependents" not in text and "return;" not in text
    assert text.rstrip().endswith("b2::pdl_release_results();")
    assert text.index("b2::pdl_wait();") < text.index("a.counts")
