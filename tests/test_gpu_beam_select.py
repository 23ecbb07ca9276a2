"""ops.beam_select on a B200 against its definition in 64 bits on the same inputs.

Parents, tokens and flags must be the definition's: pairs that are near each other are decided in 64 bits, and equal ones by their places.  Draws whose order hangs on less than 1e-11
(the definition's own rounding) do not occur here but for pairs that are equal by construction: equal logits of one row, rows that are copies.
Scores: a row's log of the sum comes from sums in 32 bits of exponentials.  An exponential's argument is off by at most 2^-24 of a size that is at most 32 for terms that count (the rest is less than
2^-32 of the sum), 2^-19 in all, its result by 2^-22, and the sums of 64 terms by 2^-18 of themselves at most: 2^-18 + 2^-19 + 2^-22 < 6e-6.  The result is rounded once, by
at most 2^-24 of itself."""
import random

import pytest
import torch

import beam_util as ref
import gpu_util

pytestmark = pytest.mark.gpu
DEV = "cuda"
SUM, ROUND = 6e-6, 2.0 ** -24
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ops(pkg):
    gpu_util.ensure_group()
    torch.cuda.set_device(0)
    pkg.init_runtime(max_tokens=512, hidden=1024, vocab=2048, max_seqs=64)
    from nanovllm_b200 import ops
    yield ops
    pkg.shutdown_runtime()


def draw(n, beams, vocab, dtype, seed, std=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = torch.empty(n * beams, vocab, device=DEV).normal_(0, std, generator=g).to(dtype)
    scores = torch.empty(n, beams, device=DEV).uniform_(-14, -10, generator=g)
    return logits, scores


def check(ops, logits, scores, picks, finished=None, eos=None):
    got = ops.beam_select(logits, scores, picks, finished=finished, eos_token=eos)
    n = scores.shape[0]
    for x, dtype in zip(got, (torch.float32, torch.int32, torch.int64, torch.bool)):
        assert x.shape == (n, picks) and x.dtype == dtype and x.is_contiguous()
    want = ref.beam_select(logits, scores, picks, finished, eos)
    assert got.parents.tolist() == want[1]
    assert got.tokens.tolist() == want[2]
    assert got.finished.tolist() == want[3]
    for a, b, t in zip(sum(got.scores.tolist(), []), sum(want[0], []), sum(want[2], [])):
        if b == -INF:
            assert a == -INF
        else:
            assert abs(a - b) <= (0 if t < 0 else SUM) + ROUND * abs(b), (a, b)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n, beams, picks, vocab", [(1, 1, 1, 1), (1, 1, 3, 2), (2, 4, 4, 7), (3, 2, 64, 5), (1, 32, 64, 1), (2, 32, 32, 999), (5, 3, 7, 1001), (1, 4, 4, 4096), (3, 5, 10, 4097),
                                                   (2, 8, 8, 32000), (33, 3, 7, 5027), (1, 32, 64, 20011), (1, 4, 8, 151936), (300, 1, 1, 513), (40, 6, 12, 2048)])
def test_sizes(ops, dtype, n, beams, picks, vocab):
    logits, scores = draw(n, beams, vocab, dtype, seed=n + beams + vocab)
    check(ops, logits, scores, picks)
    finished = torch.rand(n, beams, generator=torch.Generator().manual_seed(vocab)).to(DEV) < 0.4
    check(ops, logits, scores, picks, finished, eos=vocab // 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab, picks", [(5, 5), (1000, 64), (70000, 33)])
def test_ties(ops, dtype, vocab, picks):
    """Constant rows, copies of rows with equal scores, few values: the lowest beam, then the lowest token."""
    logits = torch.full((8, vocab), 1.25, dtype=dtype, device=DEV)
    scores = torch.tensor([[-3.0, -3.0, -2.5, -3.0], [-1.0, -1.0, -1.0, -1.0]], device=DEV)
    check(ops, logits, scores, picks)
    g = torch.Generator(device=DEV).manual_seed(vocab)
    row = torch.randint(0, 9, (1, vocab), generator=g, device=DEV).to(dtype)
    check(ops, row.expand(8, vocab).contiguous(), scores, picks)
    row = torch.empty(1, vocab, device=DEV).normal_(0, 3, generator=g).to(dtype)
    check(ops, row.expand(8, vocab).contiguous(), scores, picks)
    lone = torch.full((8, vocab), -2.0, dtype=dtype, device=DEV)
    lone[:, vocab - 1] = 4.0
    check(ops, lone, scores, picks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_orders_of_the_logits(ops, dtype):
    """Rising and falling rows: the best are in one chunk, and each chunk's largest is above the one's before."""
    vocab = 30011
    rising = torch.arange(vocab, device=DEV, dtype=torch.float32) * (8.0 / vocab)
    for row in (rising, rising.flip(0)):
        logits = row.repeat(6, 1).to(dtype)
        scores = torch.tensor([[-1.0, -1.5, -2.25], [-7.0, -7.0, -7.0]], device=DEV)
        check(ops, logits, scores, 48)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_nan_and_masks(ops, dtype):
    """Forbidden tokens (minus infinity, or the type's lowest value), NaN, plus infinity; rows with nothing left, or one token."""
    vocab = 3001
    logits, _ = draw(4, 6, vocab, dtype, seed=3)
    scores = torch.full((4, 6), -5.0, device=DEV) - torch.arange(24, device=DEV).view(4, 6) * 0.37
    g = torch.Generator(device=DEV).manual_seed(9)
    logits[0:6].masked_fill_(torch.rand(6, vocab, generator=g, device=DEV) < 0.95, -INF)
    logits[0] = -INF
    logits[1] = NAN
    logits[2, :-1] = -INF
    logits[6:12].masked_fill_(torch.rand(6, vocab, generator=g, device=DEV) < 0.5, NAN)
    logits[12:18].masked_fill_(torch.rand(6, vocab, generator=g, device=DEV) < 0.9, torch.finfo(dtype).min)
    logits[13] = torch.finfo(dtype).min
    logits[18, 5] = INF
    logits[19, 7:9] = INF
    logits[20, 3] = torch.finfo(dtype).max
    logits[21] = torch.finfo(dtype).max
    logits[21, 100:] = -torch.finfo(dtype).max
    check(ops, logits, scores, 12)
    check(ops, logits, scores, 64, eos=5)
    nothing = torch.full((6, vocab), -INF, dtype=dtype, device=DEV)
    got = check(ops, nothing, torch.zeros(2, 3, device=DEV), 5)
    assert (got.parents == -1).all() and not got.finished.any()


def test_scores_of_no_beam(ops):
    """-inf and NaN: no continuation, not even of a beam at its end; +-0, large and small ones."""
    logits, scores = draw(3, 5, 700, torch.bfloat16, seed=4)
    scores[0] = torch.tensor([-INF, NAN, -INF, -3.0, -INF])
    scores[1] = torch.tensor([-INF, NAN, -INF, -INF, NAN])
    scores[2] = torch.tensor([0.0, -0.0, -1e4, 1e3, -1e30])
    for finished in (None, torch.tensor([[True, True, False, False, True]] * 3, device=DEV)):
        check(ops, logits, scores, 9, finished, eos=4)


def test_all_at_their_end(ops):
    logits, scores = draw(2, 4, 321, torch.float32, seed=5)
    got = check(ops, logits, scores, 6, torch.ones(2, 4, dtype=torch.bool, device=DEV), eos=1)
    assert got.tokens.eq(-1).all() and got.finished.sum() == 8
    assert torch.equal(got.scores[:, :4], scores.sort(descending=True).values)  # (as they are, not rounded again)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gap", [3e-8, 1e-6, 1e-5])
def test_beams_nearly_alike(ops, dtype, gap):
    """Rows that are permutations of one another have the same sum, but for rounding, and scores a few roundings apart: the order is that of the scores' exact sums.  The
    definition's own sums of 64 bits differ by some 1e-15 between permutations; the gaps are 3e-8 and more, as far as 32 bits have them at scores of a thousandth."""
    vocab = 12007
    g = torch.Generator(device=DEV).manual_seed(6)
    row = torch.empty(vocab, device=DEV).normal_(0, 3, generator=g).to(dtype)
    row[77] = 30.0
    logits = torch.stack([row[torch.randperm(vocab, generator=g, device=DEV)] for _ in range(8)])
    scores = torch.tensor([[-1e-3 - gap * i for i in (3, 1, 0, 2)], [-2e-3 - gap * i for i in (0, 1, 2, 3)]], device=DEV)
    assert all(len(set(s)) == 4 for s in scores.tolist())
    check(ops, logits, scores, 4)
    check(ops, logits, scores, 20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("std", [0.01, 30.0, 1000.0, 1e5])
def test_magnitudes(ops, dtype, std):
    """Flat and steep rows, and logits beyond what the sums in 32 bits take (SUM's argument holds: terms that count are near the largest)."""
    logits, scores = draw(3, 4, 9001, dtype, seed=8, std=std)
    check(ops, logits, scores, 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(ops, dtype):
    """Columns of a wider tensor that begin anywhere, with odd strides; rows in another order of dimensions."""
    logits, scores = draw(3, 4, 5003, dtype, seed=10)
    want = check(ops, logits, scores, 8)
    for left, right in ((1, 0), (3, 2), (8, 5)):
        wide = torch.full((12, left + 5003 + right), 100.0, dtype=dtype, device=DEV)
        wide[:, left:left + 5003] = logits
        got = ops.beam_select(wide[:, left:left + 5003], scores, 8)
        assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))
    got = ops.beam_select(logits.t().contiguous().t(), scores, 8)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_picks_default_to_the_beams(ops):
    logits, scores = draw(2, 3, 99, torch.bfloat16, seed=11)
    assert ops.beam_select(logits, scores).parents.shape == (2, 3)
    assert ops.beam_select(logits[:0], scores[:0]).parents.shape == (0, 3)


def test_inputs_stay_and_calls_agree(ops):
    logits, scores = draw(20, 8, 20000, torch.bfloat16, seed=12)
    before = logits.clone(), scores.clone()
    first = ops.beam_select(logits, scores, 16)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(ops.beam_select(logits, scores, 16), first))
    assert torch.equal(before[0], logits) and torch.equal(before[1], scores)


def test_captured_and_on_two_streams(ops):
    work = [draw(8, 4, 30000, torch.bfloat16, seed=13), draw(2, 32, 9999, torch.float32, seed=14)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in work], [], []
    for (logits, scores), s in zip(work, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.beam_select(logits, scores, 8)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(ops.beam_select(logits, scores, 8))
        graphs.append(graph)
    for seed in (20, 21):
        for logits, scores in work:
            logits.copy_(draw(1, logits.shape[0], logits.shape[1], logits.dtype, seed)[0])
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        eager = [check(ops, logits, scores, 8) for logits, scores in work]
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_random_draws(ops):
    r = random.Random(15)
    for seed in range(25):
        n, beams, vocab = r.randint(1, 6), r.randint(1, 32), r.choice((r.randint(1, 50), r.randint(50, 5000), 40001))
        logits, scores = draw(n, beams, vocab, r.choice((torch.bfloat16, torch.float32)), seed, std=r.choice((0.5, 3.0)))
        g = torch.Generator(device=DEV).manual_seed(seed)
        if r.random() < 0.5:
            logits.masked_fill_(torch.rand(logits.shape, generator=g, device=DEV) < r.choice((0.3, 0.99, 0.9999)), -INF)
        finished = torch.rand(n, beams, generator=g, device=DEV) < 0.3 if r.random() < 0.5 else None
        check(ops, logits, scores, r.randint(1, 64), finished, r.choice((None, 0, vocab - 1)))
