"""What ModelRunner sends through the token broadcast, on two ranks on the host.  The kernel's inbox holds -1 until a value lands, so a negative value is one that never comes: the
other ranks wait for it until the time is up, take 0, and the runtime reports an expired wait.  The stand-in for the broadcast here does the same (without the wait)."""
import os
from datetime import timedelta

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _with_the_rule(runner, rank):
    """The runner with a broadcast that keeps the kernel's rule; the number of broadcasts so far."""
    from nanovllm_b200 import ops
    sent = []

    class Runtime:
        expired = False

        def check_status(self):
            if self.expired:
                self.expired = False
                raise RuntimeError("a wait expired")

    runner.runtime = Runtime()

    def broadcast_tokens(buf):
        assert buf.dtype == torch.int64 and buf.is_contiguous() and buf.numel() <= runner.max_num_seqs
        sent.append(buf.numel())
        landed = buf.clone()
        dist.broadcast(landed, 0)
        if rank != 0:
            runner.runtime.expired |= bool((landed < 0).any())
            buf.copy_(landed.clamp(min=0))
        return buf

    ops.broadcast_tokens = broadcast_tokens
    return sent


def _run(calls, sent):
    out = []
    for call in calls:
        before = len(sent)
        try:
            answer = call()
        except Exception as error:
            answer = f"{type(error).__name__}: {error}"
        out.append((answer, sent[before:]))
    return out


def _beam_searches(rank, world):
    from tests.test_beam_ranks import _runner
    r, Seq = _runner(rank, world)
    sent = _with_the_rule(r, rank)
    forced = dict(bias_ids=torch.tensor([[1], [2]]), bias_values=torch.tensor([[90.0], [80.0]]))
    none = dict(allowed_mask=torch.zeros(2, 2, dtype=torch.int32))  # nothing may follow: no beams, sums of -inf
    cases = [dict(), dict(eos_token=13), dict(rules=forced), dict(rules=none), dict()]
    return _run([lambda more=more: r.beam_search([Seq([4, 5, 6], [0]), Seq(list(range(20)), [1, 2])], 3, 5, list(range(10, 40)), **more) for more in cases], sent)


def _beam_errors(rank, world):
    from tests.test_beam_ranks import _runner
    r, Seq = _runner(rank, world)
    sent = _with_the_rule(r, rank)
    wrong = dict(no_such_rule=torch.zeros(2))
    late = dict(bias_ids=torch.tensor([[1], [2]]), bias_values=torch.tensor([[1.0], [1.0]]))
    cases = [dict(rules=wrong), dict(), dict(eos_token=13), dict(rules=late), dict()]
    from nanovllm_b200 import ops
    adjust, calls = ops.adjust_logits, []

    def adjust_logits(logits, **rules):  # the third step of the search whose rules are `late` fails
        if rules["bias_values"].numel() == 6:
            calls.append(0)
            if len(calls) == 2:
                raise ArithmeticError("on rank 0 only")
        return adjust(logits, **rules)

    ops.adjust_logits = lambda logits, **rules: adjust_logits(logits, **rules) if "bias_values" in rules else adjust(logits, **rules)
    return _run([lambda more=more: r.beam_search([Seq([4, 5, 6], [0]), Seq(list(range(20)), [1, 2])], 3, 5, list(range(10, 40)), **more) for more in cases], sent)


def _verify_steps(rank, world):
    from tests.test_verify_ranks import _runner
    r, Seq = _runner(rank, world)
    sent = _with_the_rule(r, rank)
    batch = [Seq([4, 5, 6], [0]), Seq(list(range(20)), [1, 2])], [[7, 8], [9]], [[0, 0], [0]]
    return _run([lambda rules=rules: r.verify(*batch, rules=rules) for rules in (None, dict(no_such_rule=1), None)], sent)


def _rank(rank, world, store, results):
    import sys
    if ROOT not in sys.path:
        sys.path.insert(0, ROOT)
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=world, timeout=timedelta(seconds=20))
    try:
        results[rank] = dict(beams=_beam_searches(rank, world), errors=_beam_errors(rank, world), verify=_verify_steps(rank, world))
    finally:
        dist.destroy_process_group()


@pytest.fixture(scope="module")
def answers(tmp_path_factory):
    with mp.Manager() as manager:
        results = manager.dict()
        mp.spawn(_rank, args=(2, str(tmp_path_factory.mktemp("ranks") / "store"), results), nprocs=2)
        return dict(results)


def test_a_searchs_sums_reach_every_rank(answers):
    """Sums of log-probabilities are negative, and -inf where there is no beam."""
    mine, others = answers[0]["beams"], answers[1]["beams"]
    assert mine == others
    for found, _ in mine:
        assert isinstance(found, list), found
    assert all(score < 0 for f in mine[0][0] for _, score in f) and all(len(f) == 3 for f in mine[0][0])
    assert mine[3][0] == [[], []] and mine[4] == mine[0]


def test_rank_0s_error_in_a_search_reaches_every_rank(answers):
    """As an error of its own, not as a wait that expired or a search without beams; all ranks have then made as many broadcasts, of which every other one goes to the other half of
    the inbox."""
    mine, others = answers[0]["errors"], answers[1]["errors"]
    assert [sent for _, sent in mine] == [sent for _, sent in others]
    for step, error, broadcasts in ((0, "TypeError", 1), (3, "ArithmeticError", 3)):
        assert mine[step][0].startswith(error) and others[step][0].startswith("RuntimeError: rank 0 could not"), (mine[step][0], others[step][0])
        assert len(mine[step][1]) == broadcasts
    for step, same in ((1, 0), (2, 1), (4, 0)):
        assert mine[step] == others[step] == answers[0]["beams"][same]


def test_rank_0s_error_in_a_verification_reaches_every_rank(answers):
    mine, others = answers[0]["verify"], answers[1]["verify"]
    assert [sent for _, sent in mine] == [sent for _, sent in others] == [[5]] * 3
    assert mine[0] == others[0] == mine[2] == others[2] and isinstance(mine[0][0], list)
    assert mine[1][0].startswith("TypeError") and others[1][0].startswith("RuntimeError: rank 0 could not")
