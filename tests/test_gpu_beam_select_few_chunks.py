"""ops.beam_select on a B200 where the largest logits of the chunks of 2 KB give no bound near the best continuations: fewer chunks than picks, or chunks that hold many of the best."""
import pytest
import torch

import gpu_util
from tests.test_gpu_beam_select import DEV, INF, check, draw

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    gpu_util.ensure_group()
    torch.cuda.set_device(0)
    pkg.init_runtime(max_tokens=512, hidden=1024, vocab=2048, max_seqs=64)
    from nanovllm_b200 import ops
    yield ops
    pkg.shutdown_runtime()


SIZES = [(1, 1, 64, 50257, torch.bfloat16), (3, 1, 50, 50257, torch.bfloat16), (4, 1, 32, 32000, torch.bfloat16), (2, 1, 64, 30011, torch.float32), (2, 1, 4, 4096, torch.bfloat16),
         (2, 3, 64, 20000, torch.bfloat16), (1, 2, 64, 15000, torch.float32), (1, 1, 64, 1537, torch.float32)]


@pytest.mark.parametrize("n, beams, picks, vocab, dtype", SIZES)
def test_fewer_chunks_than_picks(ops, n, beams, picks, vocab, dtype):
    for seed, std in ((1, 3.0), (2, 0.01), (3, 200.0), (4, 1e5)):
        logits, scores = draw(n, beams, vocab, dtype, seed=seed, std=std)
        check(ops, logits, scores, picks)
        finished = torch.zeros(n, beams, dtype=torch.bool, device=DEV)
        finished[0, -1] = True
        check(ops, logits, scores, picks, finished, eos=vocab // 3)


@pytest.mark.parametrize("n, beams, picks, vocab, dtype", SIZES)
def test_orders_and_ties(ops, n, beams, picks, vocab, dtype):
    rows = n * beams
    scores = -1.0 - torch.arange(rows, device=DEV).view(n, beams).float() * 0.125
    rising = torch.arange(vocab, device=DEV, dtype=torch.float32) * (8.0 / vocab)
    g = torch.Generator(device=DEV).manual_seed(vocab)
    few = torch.randint(0, 9, (rows, vocab), generator=g, device=DEV).to(dtype)
    two = torch.where(torch.rand(rows, vocab, generator=g, device=DEV) < 1e-3, 2.0, -1.0).to(dtype)
    for logits in (rising.repeat(rows, 1).to(dtype), rising.flip(0).repeat(rows, 1).to(dtype), few, two, torch.full((rows, vocab), -3.0, dtype=dtype, device=DEV)):
        check(ops, logits, scores, picks)


@pytest.mark.parametrize("n, beams, picks, vocab, dtype", SIZES)
def test_masks_and_infinities(ops, n, beams, picks, vocab, dtype):
    logits, scores = draw(n, beams, vocab, dtype, seed=7)
    g = torch.Generator(device=DEV).manual_seed(vocab)
    half = logits.masked_fill(torch.rand(logits.shape, generator=g, device=DEV) < 0.5, -INF)
    check(ops, half, scores, picks)
    check(ops, logits.masked_fill(half == -INF, torch.finfo(dtype).min), scores, picks)
    half[:, 3::97] = float("nan")
    half[0, 5:900:7] = INF
    half[-1, 11] = torch.finfo(dtype).max
    check(ops, half, scores, picks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_few_chunks_allowed(ops, dtype):
    """Of a large vocabulary the tokens of four chunks are allowed, all of them or half."""
    per = 2048 // torch.empty(0, dtype=dtype).element_size()
    for beams, picks in ((1, 8), (4, 20), (8, 64)):
        logits, scores = draw(2, beams, 151936, dtype, seed=beams)
        allowed = torch.zeros(151936, dtype=torch.bool, device=DEV)
        allowed[40 * per:44 * per] = True
        check(ops, logits.masked_fill(~allowed, -INF), scores, picks)
        allowed[40 * per:44 * per:2] = False
        check(ops, logits.masked_fill(~allowed, -INF), scores, picks)


@pytest.mark.parametrize("gap", [3e-8, 1e-6, 4.2e-6])
def test_beams_nearly_alike_in_few_chunks(ops, gap):
    """Rows that are permutations of one another, so that the order of equal logits of different beams is that of the scores."""
    vocab, beams = 9001, 4
    g = torch.Generator(device=DEV).manual_seed(6)
    row = torch.empty(vocab, device=DEV).normal_(0, 3, generator=g).bfloat16()
    row[7] = 30.0
    logits = torch.stack([row[torch.randperm(vocab, generator=g, device=DEV)] for _ in range(beams)])
    scores = torch.tensor([[-1e-3 - gap * i for i in (3, 1, 0, 2)]], device=DEV)
    check(ops, logits, scores, 64)


def test_time(ops):
    """The first step of a search with many beams has one row a request.  With fewer chunks than picks it takes a few times as long as over a larger vocabulary, which has more, and not a hundred times."""
    def microseconds(vocab, picks):
        logits, scores = draw(1, 1, vocab, torch.bfloat16, seed=1)
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        best = INF
        for _ in range(5):
            ops.beam_select(logits, scores, picks)
            begin.record()
            for _ in range(10):
                ops.beam_select(logits, scores, picks)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end) * 100)
        return best

    ordinary = microseconds(151936, 64)
    for vocab, picks in ((50257, 64), (32000, 32), (50257, 50)):
        assert microseconds(vocab, picks) <= 10 * ordinary


@pytest.mark.parametrize("n, beams, picks, vocab, dtype", [(2, 32, 64, 151936, torch.float32), (1, 16, 5, 400003, torch.bfloat16), (1, 3, 64, 3000001, torch.bfloat16)])
def test_more_chunks_than_a_cta_keeps(ops, n, beams, picks, vocab, dtype):
    """Chunks whose largest logits a CTA reads again each time, since it has no registers for them; equal ones too, of which there are more than it lists."""
    logits, scores = draw(n, beams, vocab, dtype, seed=beams)
    check(ops, logits, scores, picks, eos=3)
    finished = torch.zeros(n, beams, dtype=torch.bool, device=DEV)
    finished[:, ::5] = True
    scores[0, 1] = -INF
    check(ops, logits, scores, picks, finished)
    logits.fill_(-1.5)
    logits[:, vocab - 1] = 4.0
    check(ops, logits, torch.full_like(scores, -2.0), picks)
