"""ModelRunner.verify on a small random-init Qwen3, one B200: the picks after a tree's nodes are those of plain decoding along each path."""
import pytest
import torch

from tests.gpu_util import ensure_group
from tests.test_gpu_model import _attention_backend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def runner(pkg):
    ensure_group()
    from nanovllm_b200.engine.model_runner import ModelConfig, ModelRunner
    _attention_backend()
    cfg = ModelConfig(hidden_size=1024, num_attention_heads=8, num_key_value_heads=4, head_dim=128, intermediate_size=2048, num_hidden_layers=3, vocab_size=2048,
                      max_position_embeddings=2048)
    runner = ModelRunner(cfg, max_num_seqs=64, max_model_len=1024, max_num_batched_tokens=2048, num_kvcache_blocks=32, enforce_eager=True, oneshot_tokens=128, seed=3)
    yield runner
    runner.exit()


def sequences(runner, lens, seed):
    from nanovllm_b200.engine.model_runner import Seq, sequential_block_tables
    g = torch.Generator().manual_seed(seed)
    seqs = [Seq(torch.randint(0, 2048, (n,), generator=g).tolist()) for n in lens]
    for s, bt in zip(seqs, sequential_block_tables([n + 64 for n in lens], 256)):
        s.block_table = bt
    for s, t in zip(seqs, runner.step(seqs, True)):
        s.token_ids.append(t)
    return seqs


def margins(runner, seqs):
    """The decode step's logits: picks, and by how much they lead."""
    ids, pos = runner.prepare_decode(seqs)
    top = runner.run_model(ids, pos, False).float().topk(2, dim=-1)
    return top.indices[:, 0].tolist(), (top.values[:, 0] - top.values[:, 1]).tolist()


def test_picks_along_every_path(runner):
    """Two branches per sequence, one of which follows the model's own picks.  A pick may differ where the decode step's two best logits are closer than
    bf16 keeps them apart (2 units of 2^-8 at their size)."""
    from nanovllm_b200.engine.model_runner import Seq
    seqs = sequences(runner, [30, 255, 256, 400], seed=5)
    follow = [[] for _ in seqs]
    work = [Seq(list(s.token_ids), s.block_table) for s in seqs]
    for _ in range(4):
        for w, f, t in zip(work, follow, runner.step(work, False)):
            w.token_ids.append(t)
            f.append(t)
    # nodes: 0 = last token, 1..3 the picks, 4 and 5 a branch from node 1
    drafts = [[f[0], f[1], f[2], (f[1] + 7) % 2048, (f[2] + 9) % 2048] for f in follow]
    parents = [[0, 1, 2, 1, 4]] * len(seqs)
    got = runner.verify(seqs, drafts, parents)
    agreed = total = 0
    for path, node in (([], 0), ([0], 1), ([0, 1], 2), ([0, 1, 2], 3), ([0, 3], 4), ([0, 3, 4], 5)):
        # the path's tokens put into the cache one after the other, as plain decoding does
        work = [Seq(list(s.token_ids), s.block_table) for s in seqs]
        for k in path:
            runner.step(work, False)
            for w, d in zip(work, drafts):
                w.token_ids.append(d[k])
        want, lead = margins(runner, work)
        for i, (w, l) in enumerate(zip(want, lead)):
            total += 1
            agreed += got[i][node] == w
            assert got[i][node] == w or l <= 0.05, f"sequence {i}, node {node}: {got[i][node]}, decoding picks {w} with a lead of {l}"
    assert agreed >= 0.9 * total


def test_rules_reach_the_picks(runner):
    seqs = sequences(runner, [20, 70], seed=6)
    drafts, parents = [[5, 9], [11]], [[0, 0], [0]]
    plain = runner.verify(seqs, drafts, parents)
    banned = torch.tensor([[p for p in picks] + [-1] * (3 - len(picks)) for picks in plain], device="cuda")
    got = runner.verify(seqs, drafts, parents, rules=dict(bias_ids=banned, bias_values=torch.full(banned.shape, -1e4, device="cuda")))
    assert all(g not in picks for gs, picks in zip(got, plain) for g in gs)
    allowed = torch.zeros(5, 64, dtype=torch.int32, device="cuda")
    allowed[:, 3] = 1 << 7
    assert runner.verify(seqs, drafts, parents, rules=dict(allowed_mask=allowed)) == [[3 * 32 + 7] * 3, [3 * 32 + 7] * 2]


def test_refusals(runner):
    seqs = sequences(runner, [20], seed=7)
    for drafts, parents in (([[1]], [[1]]), ([[1, 2]], [[0]]), ([], []), ([[1] * 64], [[0] * 64])):
        with pytest.raises(ValueError):
            runner.verify(seqs, drafts, parents)
    with pytest.raises(ValueError, match="room"):
        from nanovllm_b200.engine.model_runner import Seq
        runner.verify([Seq(list(range(250)), [0])], [[1] * 10], [[0] * 10])


def test_no_sequences_and_an_error_inside_a_step(runner):
    from nanovllm_b200.utils.context import get_context
    assert runner.verify([], [], []) == []
    seqs = sequences(runner, [20], seed=8)
    with pytest.raises(ValueError):
        runner.verify(seqs, [[1]], [[0]], rules=dict(bias_ids=torch.zeros(2, 1, dtype=torch.int64, device="cuda"), bias_values=torch.zeros(2, 1, device="cuda")))
    assert get_context().tree_mask is None
    assert len(runner.step(seqs, False)) == 1
    assert runner.verify(seqs, [[]], [[]]) == runner.verify(seqs, [[]], [[]])


def test_nodes_past_the_longest_context_are_refused(runner):
    from nanovllm_b200.engine.model_runner import Seq
    with pytest.raises(ValueError, match="max_model_len"):
        runner.verify([Seq(list(range(1020)), list(range(5)))], [[1] * 5], [[0] * 5])
