"""ModelRunner.beam_search on two ranks, on the host: gloo stands for the token broadcast, plain functions for the kernels and the model."""
import os
from datetime import timedelta

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
VOCAB = 50


def _runner(rank, world):
    """A runner without a GPU: beam_search and what it calls on the host, nothing else."""
    import sys
    for path in (ROOT, os.path.join(ROOT, "tests")):
        if path not in sys.path:
            sys.path.insert(0, path)
    import __graft_entry__ as entry
    entry.load_package()
    import beam_util
    import step_util
    from nanovllm_b200 import ops
    from nanovllm_b200.engine import model_runner
    from nanovllm_b200.utils.context import get_context

    def batch_inputs(tables, cached, wanted, free, num_free, bs, num_slots, max_tokens, tree_mask=None):
        t, f, *rest = step_util.batch_inputs(tables.tolist(), cached.tolist(), wanted.tolist(), free.tolist(), num_free.item(), bs, num_slots, max_tokens, tree_mask)
        tables.copy_(torch.tensor(t, dtype=torch.int32))
        free.copy_(torch.tensor(f, dtype=torch.int32))
        return ops.BatchInputs(*(torch.tensor(x, dtype=torch.int64 if i == 0 else torch.int32) for i, x in enumerate(rest)))

    def beam_select(logits, scores, picks, *, finished=None, eos_token=None):
        out = beam_util.beam_select(logits, scores, picks, finished, eos_token)
        return ops.BeamPicks(*(torch.tensor(x, dtype=t) for x, t in zip(out, (torch.float32, torch.int32, torch.int64, torch.bool))))

    def reorder_beams(parents, tables, lens, free, num_free, cache, *, first_blocks, history, history_lens, tokens):
        t, l, stack, height, copies = beam_util.reorder_beams(parents.tolist(), tables.tolist(), lens.tolist(), free.tolist(), num_free.item(), 16, 100, first_blocks.tolist())
        free.copy_(torch.tensor(stack, dtype=torch.int32))
        text, said = beam_util.append_history(parents.tolist(), history.tolist(), history_lens.tolist(), tokens.tolist(), history.shape[1])
        i = lambda x: torch.tensor(x, dtype=torch.int32)
        return ops.BeamState(i(t), i(l), i([height]), torch.tensor(text), i(said))

    class Model:
        """Token t at place p is followed by (3 t + p) and the two next tokens, with falling probability."""

        def __call__(self, ids, positions):
            ctx = get_context()
            if ctx.is_prefill:
                ids, positions = ids[ctx.last_token_index.long()], positions[ctx.last_token_index.long()]
            else:
                assert ctx.prefix_lens is not None and ctx.context_lens.numel() == ids.numel()
            out = torch.zeros(ids.numel(), VOCAB)
            for k in range(3):
                out[torch.arange(ids.numel()), (ids * 3 + positions + k) % VOCAB] = 6.0 - 0.7 * k
            return out

        def compute_logits(self, hidden):
            return hidden if rank == 0 else None

    class Runtime:
        def check_status(self):
            pass

    def adjust_logits(logits, *, out, **rules):
        out.copy_(step_util.adjust_logits(logits, **rules))
        return out

    ops.batch_inputs, ops.adjust_logits, ops.beam_select, ops.reorder_beams = batch_inputs, adjust_logits, beam_select, reorder_beams
    ops.broadcast_tokens = lambda picked: dist.broadcast(picked, 0)
    r = model_runner.ModelRunner.__new__(model_runner.ModelRunner)
    r.rank, r.world, r.device, r.block_size, r.num_kvcache_blocks, r.kv_cache = rank, world, torch.device("cpu"), 16, 100, torch.zeros(1)
    r.max_num_seqs, r.max_model_len, r.max_num_batched_tokens, r.model, r.runtime = 64, 128, 256, Model(), Runtime()
    r.config = model_runner.ModelConfig(64, 1, 1, 64, 64, 1, VOCAB)
    r._to_device = lambda *arrays: [torch.from_numpy(a.copy()) for a in arrays]
    return r, model_runner.Seq


SEARCHES = [dict(), dict(rules=dict(no_such_rule=torch.zeros(2))), dict(eos_token=13), dict(rules=dict(bias_ids=torch.tensor([[1], [2]]), bias_values=torch.tensor([[90.0], [80.0]]))), dict()]


def _steps(rank, world):
    r, Seq = _runner(rank, world)
    from_host = []
    for more in SEARCHES:
        try:
            from_host.append(r.beam_search([Seq([4, 5, 6], [0]), Seq(list(range(20)), [1, 2])], 3, 5, list(range(10, 40)), **more))
        except Exception as error:
            from_host.append(type(error).__name__)
    return from_host


def _rank(rank, world, store, results):
    # (a rank that waits for one that never comes ends with an error after this time, and not with the other's answer)
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=world, timeout=timedelta(seconds=20))
    try:
        results[rank] = _steps(rank, world)
    finally:
        dist.destroy_process_group()


@pytest.fixture(scope="module")
def answers(tmp_path_factory):
    with mp.Manager() as manager:
        results = manager.dict()
        mp.spawn(_rank, args=(2, str(tmp_path_factory.mktemp("ranks") / "store"), results), nprocs=2)
        return dict(results)


def test_the_same_continuations_on_both_ranks(answers):
    for step in (0, 2, 3, 4):
        assert answers[0][step] == answers[1][step] and isinstance(answers[0][step], list)
    assert answers[0][0] == answers[0][4]
    best = []
    t, p = 6, 2
    for _ in range(5):  # the most probable token each time is the best path here
        t, p = (3 * t + p) % VOCAB, p + 1
        best.append(t)
    (tokens, score), *others = answers[0][0][0]
    row = torch.zeros(VOCAB, dtype=torch.float64)
    row[:3] = torch.tensor([6.0, 5.3, 4.6])
    assert tokens == best and abs(score - 5 * row.log_softmax(0)[0].item()) < 1e-5 and len(others) == 2
    assert answers[0][3][0][0][0] == [1] * 5 and answers[0][3][1][0][0] == [2] * 5
    assert all(t[-1] == 13 or len(t) == 5 for f in answers[0][2] for t, _ in f) and any(t[-1] == 13 and len(t) < 5 for f in answers[0][2] for t, _ in f)


def test_a_bad_rule_is_an_error_on_both_ranks_and_the_next_search_runs(answers):
    assert (answers[0][1], answers[1][1]) == ("TypeError", "RuntimeError")
