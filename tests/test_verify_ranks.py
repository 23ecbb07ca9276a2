"""ModelRunner.verify on two ranks, on the host: gloo stands for the token broadcast, plain functions for the kernels and the model."""
import os
from datetime import timedelta

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
VOCAB = 50


def _runner(rank, world):
    """A runner without a GPU: verify and what it calls on the host, nothing else."""
    import sys
    for path in (ROOT, os.path.join(ROOT, "tests")):
        if path not in sys.path:
            sys.path.insert(0, path)
    import __graft_entry__ as entry
    entry.load_package()
    import step_util as ref
    from nanovllm_b200 import ops
    from nanovllm_b200.engine import model_runner

    def batch_inputs(tables, cached, wanted, free, num_free, bs, num_slots, max_tokens, tree_mask=None):
        t, f, *rest = ref.batch_inputs(tables.tolist(), cached.tolist(), wanted.tolist(), free.tolist(), num_free.item(), bs, num_slots, max_tokens, tree_mask)
        return ops.BatchInputs(*(torch.tensor(x, dtype=torch.int64 if i == 0 else torch.int32) for i, x in enumerate(rest)))

    class Model:
        def __call__(self, ids, positions):
            return torch.nn.functional.one_hot((ids * 3 + positions) % VOCAB, VOCAB).float()

        def compute_logits(self, hidden):
            return hidden if rank == 0 else None

    class Runtime:
        def check_status(self):
            pass

    def adjust_logits(logits, *, out, cu_seqlens, draft_tokens, tree_mask, **rules):
        out.copy_(ref.adjust_logits(logits, cu_seqlens=cu_seqlens, draft_tokens=draft_tokens, tree_mask=tree_mask, **rules))
        return out

    ops.batch_inputs, ops.adjust_logits = batch_inputs, adjust_logits
    ops.argmax = lambda logits, out: out.copy_(logits.argmax(-1))
    ops.broadcast_tokens = lambda picked: dist.broadcast(picked, 0)
    r = model_runner.ModelRunner.__new__(model_runner.ModelRunner)
    r.rank, r.world, r.device, r.block_size, r.num_kvcache_blocks = rank, world, torch.device("cpu"), 16, 8
    r.max_num_seqs, r.max_model_len, r.model, r.runtime = 64, 128, Model(), Runtime()
    r.config = model_runner.ModelConfig(64, 1, 1, 64, 64, 1, VOCAB)
    r._to_device = lambda *arrays: [torch.from_numpy(a.copy()) for a in arrays]
    return r, model_runner.Seq


def _steps(rank, world):
    from_host = []
    r, Seq = _runner(rank, world)
    batch = [Seq([4, 5, 6], [0]), Seq(list(range(20)), [1, 2])], [[7, 8], [9]], [[0, 0], [0]]
    for rules in (None, dict(history=torch.zeros(3, 2, dtype=torch.int64)), dict(no_such_rule=1), dict(bias_ids=torch.tensor([[1], [2]]), bias_values=torch.tensor([[9.0], [8.0]])), None):
        try:
            from_host.append(r.verify(*batch, rules=rules))
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


def test_the_same_picks_on_both_ranks(answers):
    for step in (0, 3, 4):
        assert answers[0][step] == answers[1][step]
    # node n: the token of its one-hot row; the biased ones where a rule says so
    assert answers[0][0] == [[(6 * 3 + 2) % VOCAB, (7 * 3 + 3) % VOCAB, (8 * 3 + 3) % VOCAB], [(19 * 3 + 19) % VOCAB, (9 * 3 + 20) % VOCAB]]
    assert answers[0][3] == [[1] * 3, [2] * 2] and answers[0][4] == answers[0][0]


def test_a_bad_rule_is_an_error_on_both_ranks_and_the_next_step_runs(answers):
    """Rules are applied where the logits are, on rank 0: its error reaches the other rank through the broadcast that both take."""
    for step in (1, 2):
        assert (answers[0][step], answers[1][step]) == ("TypeError", "RuntimeError")
