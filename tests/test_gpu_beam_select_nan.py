"""ops.beam_select on a B200: chunks with a NaN among their logits, whose sums are formed in 64 bits, beside others whose sums are formed in 32, with log2(e) in 24 bits."""
import pytest
import torch

import gpu_util
from tests.test_gpu_beam_select import DEV, INF, NAN, check, draw

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    gpu_util.ensure_group()
    torch.cuda.set_device(0)
    pkg.init_runtime(max_tokens=512, hidden=1024, vocab=2048, max_seqs=64)
    from nanovllm_b200 import ops
    yield ops
    pkg.shutdown_runtime()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [40, 402, 9001])
@pytest.mark.parametrize("base, std", [(0.0, 3.0), (90.0, 3.0), (-500.0, 5.0), (0.0, 1e4), (60000.0, 100.0), (-60000.0, 100.0)])
def test_nan_among_logits_of_any_size(ops, dtype, vocab, base, std):
    """In no chunk, in one and in all of them; rows that differ by that alone have the same sum but for the token that it stands for."""
    logits, scores = draw(3, 4, vocab, torch.float32, seed=vocab, std=std)
    logits = (logits + base).to(dtype)
    check(ops, logits, scores, 8)
    logits[1::4, vocab // 2] = NAN
    logits[2::4, ::31] = NAN
    logits[3::4, 5] = -INF
    check(ops, logits, scores, 8)
    # beams that are alike: those whose forbidden token is a NaN come between the others by their places
    row = logits[:1].repeat(12, 1)
    row[:, 7] = -INF
    row[1::2, 7] = NAN
    check(ops, row, torch.full_like(scores, -1e-3), 8)


@pytest.mark.parametrize("gap", [0.0, 1e-6, 4.2e-6, 1e-5])
def test_beams_alike_but_for_a_nan(ops, gap):
    """Sums in 64 bits and in 32 of the same numbers are no further apart than two in 32 bits."""
    for base in (20.0, 200.0, 30000.0):
        row = torch.empty(30000, device=DEV).normal_(0, 2, generator=torch.Generator(device=DEV).manual_seed(3)) + base
        row[11] = -INF
        logits = row.repeat(8, 1)
        logits[[0, 3, 4, 6], 11] = NAN
        scores = torch.tensor([[-1e-3 - gap * i for i in (3, 1, 0, 2)], [-1e-3 - gap * i for i in (0, 3, 2, 1)]], device=DEV)
        check(ops, logits, scores, 6)
