"""ops.beam_select on a B200: beams whose score is +inf.  All their continuations have +inf, of equal ones the lowest beam and token come first, and the others' follow."""
import pytest
import torch

import gpu_util

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = float("inf")


@pytest.fixture(scope="module")
def ops(pkg):
    gpu_util.ensure_group()
    torch.cuda.set_device(0)
    pkg.init_runtime(max_tokens=512, hidden=1024, vocab=2048, max_seqs=64)
    from nanovllm_b200 import ops
    yield ops
    pkg.shutdown_runtime()


def definition(logits, scores, picks, finished):
    """(score, beam, token) of each request's picks, best first."""
    n, beams = scores.shape
    out = []
    for r in range(n):
        x = logits[r * beams:(r + 1) * beams].double().cpu()
        total, s = x.logsumexp(-1), scores[r].double().tolist()
        all_of = []
        for b in range(beams):
            if not s[b] > -INF:
                continue
            if finished[r][b]:
                all_of.append((s[b], b, -1))
                continue
            y = torch.where(x[b] > -INF, s[b] + (x[b].clamp(min=-1e30) - total[b]), -INF)  # (3e38 and more takes no notice of the logit: equal ones again)
            value, order = torch.sort(y, descending=True, stable=True)
            all_of += [(v, b, t) for v, t in zip(value[:picks].tolist(), order[:picks].tolist()) if v > -INF]
        all_of.sort(key=lambda c: (-c[0], c[1], c[2]))
        out.append((all_of + [(-INF, -1, -1)] * picks)[:picks])
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab, picks", [(5, 12), (151936, 8), (151936, 64), (700, 64), (40001, 1)])
def test_scores_of_plus_infinity(ops, dtype, vocab, picks):
    beams = 4
    g = torch.Generator(device=DEV).manual_seed(vocab + picks)
    scores = torch.tensor([[INF, -3.0, INF, -1.0], [-2.0, -1.0, -3.0, INF], [INF] * 4, [-INF, INF, -INF, -7.0], [-1.0, INF, -2.0, 3e38], [-1.0, -2.0, -3.0, -4.0]], device=DEV)
    logits = torch.empty(scores.numel(), vocab, device=DEV).normal_(0, 3, generator=g).to(dtype)
    logits[8:12, :vocab // 3] = -INF
    logits[13].masked_fill_(torch.rand(vocab, generator=g, device=DEV) < 0.5, -INF)
    for ended in ([[False] * beams] * 6, [[False, False, True, False]] * 3 + [[False, True, False, False]] * 3):
        got = ops.beam_select(logits, scores, picks, finished=torch.tensor(ended, device=DEV))
        for r, want in enumerate(definition(logits, scores, picks, ended)):
            assert got.parents[r].tolist() == [b for _, b, _ in want]
            assert got.tokens[r].tolist() == [t for _, _, t in want]
            for a, (b, _, _) in zip(got.scores[r].tolist(), want):  # (6e-6 of the row's sum, and the rounding to 32 bits)
                assert a == b or abs(a - b) <= 6e-6 + 2.0 ** -24 * abs(b), (a, b)
