"""ops.beam_select on a B200 where a warp walks many chunks of the logits, over the ends of rows: the reference of a row's sum is raised, kept and left behind there.

The largest logits lie 20 to 26 above the first chunk's, on both sides of where the reference is raised, at the beginning, in the middle and at the end of the warps' ranges.  Scores are so near one another that the
order of the beams hangs on the sums: 4.2e-6 apart, a little more than what is decided in 64 bits, or less.  The definition is formed on the GPU in 64 bits; its own rounding, some
1e-14, is far below the gaps.  A row's sum may be off by 1.8e-6 (exponents 9.5e-7, exponential 2^-22, additions 6e-7), a score by 2^-24 of itself more."""
import pytest
import torch

import gpu_util

pytestmark = pytest.mark.gpu
DEV = "cuda"
SUM, ROUND = 1.8e-6, 2.0 ** -24


@pytest.fixture(scope="module")
def ops(pkg):
    gpu_util.ensure_group()
    torch.cuda.set_device(0)
    pkg.init_runtime(max_tokens=512, hidden=1024, vocab=2048, max_seqs=64)
    from nanovllm_b200 import ops
    yield ops
    pkg.shutdown_runtime()


def chunks_of_ranges(rows, vocab, size):
    """For each row the pieces that the warps' ranges leave of it: lists of (first chunk, chunks)."""
    chunks = -(-(vocab * size + 16 - size) // 2048)
    total = rows * chunks
    warps = min(total, torch.cuda.get_device_properties(0).multi_processor_count * 32)
    base, rem = divmod(total, warps)
    assert base > 5, "too few chunks a warp"
    starts = [x * base + min(x, rem) for x in range(warps + 1)]
    out = [[] for _ in range(rows)]
    for a, b in zip(starts, starts[1:]):
        while a < b:
            row, c = divmod(a, chunks)
            n = min(b - a, chunks - c)
            out[row].append((c, n))
            a += n
    return out


def check(ops, logits, scores, picks):
    n, beams = scores.shape
    vocab = logits.shape[1]
    got = ops.beam_select(logits, scores, picks)
    for r in range(n):
        x = logits[r * beams:(r + 1) * beams].double()
        top = x.amax(-1, keepdim=True)
        y = scores[r].double().view(-1, 1) + ((x - top) - (x - top).exp().sum(-1, keepdim=True).log())
        value, order = torch.sort(y.view(-1), descending=True, stable=True)
        value, order = value[:picks], order[:picks]
        assert torch.equal(got.parents[r].long(), order // vocab) and torch.equal(got.tokens[r], order % vocab), r
        error = (got.scores[r].double() - value).abs() - ROUND * value.abs()
        assert error.max().item() <= SUM, (r, error.max().item())


SHAPES = [(64, 8, 151936, torch.bfloat16), (16, 32, 50257, torch.float32), (61, 8, 151935, torch.bfloat16)]


@pytest.mark.parametrize("n, beams, vocab, dtype", SHAPES)
@pytest.mark.parametrize("gap", [4.2e-6, 1e-6])
@pytest.mark.parametrize("peaks", [1, 50])
def test_large_logits_behind_small_ones(ops, n, beams, vocab, dtype, gap, peaks):
    size = 2 if dtype == torch.bfloat16 else 4
    per = 2048 // size
    g = torch.Generator(device=DEV).manual_seed(peaks + vocab)
    r = torch.Generator().manual_seed(peaks)
    logits = torch.empty(n * beams, vocab, device=DEV).normal_(0, 0.5, generator=g)
    at = []
    for row, pieces in enumerate(chunks_of_ranges(n * beams, vocab, size)):
        c, count = pieces[torch.randint(len(pieces), (1,), generator=r).item()]
        inside = (0, 1, count // 2, count - 1)[row % 4]
        at.append(min(c + min(inside, count - 1), (vocab - 1) // per) * per)
    at = torch.tensor(at, device=DEV)
    first = logits.view(n * beams, -1)[:, :per].amax(-1, keepdim=True)
    place = (at.view(-1, 1) + torch.randint(0, per, (n * beams, peaks), generator=g, device=DEV)).clamp(max=vocab - 1)
    logits.scatter_(1, place, first + torch.empty(n * beams, peaks, device=DEV).uniform_(20, 26, generator=g))
    logits = logits.to(dtype)
    order = torch.stack([torch.randperm(beams, generator=r) for _ in range(n)]).to(DEV)
    scores = (-1e-3 - gap * order.double()).float()
    check(ops, logits, scores, 8)


@pytest.mark.parametrize("n, beams, vocab, dtype", SHAPES)
def test_rising_chunks(ops, n, beams, vocab, dtype):
    """Each chunk's largest logit is some 9 above the one's before for a while, so that the reference is raised again and again, and falls back."""
    g = torch.Generator(device=DEV).manual_seed(vocab)
    per = 2048 // (2 if dtype == torch.bfloat16 else 4)
    logits = torch.empty(n * beams, vocab, device=DEV).normal_(0, 0.5, generator=g)
    stairs = (torch.arange(vocab, device=DEV) // per).view(1, -1) + torch.arange(n * beams, device=DEV).view(-1, 1)
    logits = (logits + 9.0 * (stairs % 11) - 50.0).to(dtype)
    scores = torch.empty(n, beams, device=DEV).uniform_(-1e-3, 0, generator=g)
    check(ops, logits, scores, 8)
