"""ops.reorder_beams on a B200: tokens of any negative value."""
import random

import pytest
import torch

import gpu_util
from tests.test_gpu_reorder_beams import Case, i32

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops(pkg):
    gpu_util.ensure_group()
    torch.cuda.set_device(0)
    pkg.init_runtime(max_tokens=512, hidden=1024, vocab=2048, max_seqs=64)
    from nanovllm_b200 import ops
    yield ops
    pkg.shutdown_runtime()


@pytest.mark.parametrize("width", [1, 9, 1025])
def test_a_negative_token_is_none_whatever_its_value(ops, width):
    """Behind a row's tokens there is -1, whatever negative number stood for "none"."""
    case = Case(4, 5, 40, 16, seed=width, history=width)
    r = random.Random(width)
    case.tokens = [[r.choice((-2, -100, -2 ** 31, -2 ** 40, -2 ** 63, 0, 2 ** 62)) for _ in range(5)] for _ in range(4)]
    assert min(min(t) for t in case.tokens) < -1
    case.check(*case.run(ops))
