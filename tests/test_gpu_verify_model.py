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


def keep(runner, seq, path, drafts, pick):
    """The path's keys and values behind the sequence's, its tokens and the pick after it appended: what a program does with a step's result."""
    bs = runner.block_size

    def slots(places):
        return torch.tensor([seq.block_table[p // bs] * bs + p % bs for p in places], device="cuda")

    first = len(seq) - 1
    rows = runner.kv_cache.view(2, runner.kv_cache.shape[1], -1, *runner.kv_cache.shape[4:])
    rows[:, :, slots(first + j for j in range(len(path)))] = rows[:, :, slots(first + node for node in path)]
    seq.token_ids += [drafts[node - 1] for node in path[1:]] + [pick]


@pytest.mark.parametrize("path", [[0, 1, 2], [0, 2, 4], [0, 3], [0]])
def test_a_kept_path_is_the_next_steps_context(runner, path):
    """Trees with two branches, across a block's end: after a kept path, wherever its nodes lay, the next step's picks are those of plain decoding over the same tokens."""
    from nanovllm_b200.engine.model_runner import Seq
    seqs = sequences(runner, [40, 253], seed=9)
    drafts, parents = [[11, 12, 13, 14], [21, 22, 23, 24]], [[0, 0, 0, 2], [0, 0, 0, 2]]
    if path == [0, 1, 2]:
        parents = [[0, 1, 2, 3]] * 2
    plain = [Seq(list(s.token_ids), [b + 8 for b in s.block_table]) for s in seqs]  # the same requests in blocks of their own
    for p in plain:
        p.token_ids.pop()
    runner.step(plain, True)
    for p, s in zip(plain, seqs):
        p.token_ids.append(s.token_ids[-1])
    picked = runner.verify(seqs, drafts, parents)
    for node in path[1:]:
        runner.step(plain, False)
        for p, d in zip(plain, drafts):
            p.token_ids.append(d[node - 1])
    runner.step(plain, False)
    for s, p, d, picks in zip(seqs, plain, drafts, picked):
        keep(runner, s, path, d, picks[path[-1]])
        p.token_ids.append(picks[path[-1]])
        assert s.token_ids == p.token_ids
    # (plain decoding rounds its keys in launches of other shapes: the logits are held to the path's tolerance, not to the bit)
    ids, pos = runner.prepare_decode(plain)
    want = runner.run_model(ids, pos, False).float().clone()
    ids, pos = runner.prepare_decode(seqs)
    got = runner.run_model(ids, pos, False).float()
    assert ((got - want).abs() <= 2e-2 + 1e-2 * want.abs()).all(), (got - want).abs().max().item()
