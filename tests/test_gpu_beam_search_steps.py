"""ModelRunner.beam_search on one B200, one step after the other: the beams after t tokens are those of the search for t tokens, and each step is compared with what the model says in one prefill of every beam.

A logit is off by two roundings to bf16 of its size between the paths (2^-8 each, sizes up to 4 here), the log of the sum by as much: STEP for a token's log-probability.  A context of which a part is another one's
moves the log-probabilities by more: the tests show it for 16 tokens."""
import pytest
import torch

from tests.gpu_util import ensure_group
from tests.test_gpu_beam_search import STEP, sequences
from tests.test_gpu_model import _attention_backend

pytestmark = pytest.mark.gpu


def make_runner(block_size, num_blocks):
    ensure_group()
    from nanovllm_b200.engine.model_runner import ModelConfig, ModelRunner
    _attention_backend()
    cfg = ModelConfig(hidden_size=1024, num_attention_heads=8, num_key_value_heads=4, head_dim=128, intermediate_size=2048, num_hidden_layers=3, vocab_size=2048, max_position_embeddings=2048)
    return ModelRunner(cfg, max_num_seqs=64, max_model_len=1024, max_num_batched_tokens=2048, kvcache_block_size=block_size, num_kvcache_blocks=num_blocks, enforce_eager=True, oneshot_tokens=128, seed=3)


def log_probs(runner, texts, blocks):
    """The model's log-probabilities after each of the texts, a prefill each (float64, on the host)."""
    from nanovllm_b200.engine.model_runner import Seq
    from nanovllm_b200.utils.context import reset_context
    out = []
    for text in texts:
        ids, pos = runner.prepare_prefill([Seq(list(text), blocks[:-(-len(text) // runner.block_size)])])
        out.append(runner.run_model(ids, pos, True).double().cpu().log_softmax(-1)[0])
        reset_context()
    return torch.stack(out)


def check_steps(runner, seqs, beams, new, free, spare):
    """Each step of a search against the model; spare: blocks for the prefills."""
    before = [[([], 0.0)] for _ in seqs]
    for t in range(1, new + 1):
        found = runner.beam_search(seqs, beams, t, free)
        for s, now, last in zip(seqs, found, before):
            prompt = list(s.token_ids)
            assert len(now) == min(beams, len(last) * 2048) and len({tuple(tokens) for tokens, _ in now}) == len(now)
            assert [x for _, x in now] == sorted((x for _, x in now), reverse=True)
            at = {tuple(tokens): i for i, (tokens, _) in enumerate(last)}
            rows = log_probs(runner, [prompt + tokens for tokens, _ in last], spare)
            sums = rows + torch.tensor([x for _, x in last], dtype=torch.float64)[:, None]
            picked = []
            for tokens, score in now:
                assert len(tokens) == t
                parent = at[tuple(tokens[:-1])]  # (a continuation of one of the beams before)
                assert abs(sums[parent, tokens[-1]].item() - score) <= STEP
                picked.append((parent, tokens[-1]))
            worst = min(sums[p].item() for p in picked)
            for p in picked:
                sums[p] = float("-inf")
            assert sums.max().item() <= worst + 2 * STEP  # none that was left out is better
        before = found
    return before


@pytest.mark.parametrize("lens, beams, new", [([20, 37], 4, 5), ([16], 1, 4), ([100, 3, 31], 8, 3), ([48], 32, 2)])
def test_steps_of_a_search(pkg, lens, beams, new):
    runner = make_runner(16, 400)
    try:
        check_steps(runner, sequences(lens, seed=len(lens) + beams), beams, new, list(range(100, 350)), list(range(350, 400)))
    finally:
        runner.exit()


def test_steps_of_a_search_behind_cached_prompts(pkg):
    """Prompts whose first 256 tokens are in the cache; a block of other tokens in their place would be seen."""
    runner = make_runner(256, 40)
    try:
        seqs = sequences([300, 530], seed=12)
        for s, table in zip(seqs, ([0, 1], [2, 3, 4])):
            s.block_table = table
        free, spare = list(range(5, 30)), list(range(30, 40))
        runner.beam_search(seqs, 4, 1, free)  # (fills the cache)
        for s in seqs:
            s.num_cached_tokens = 256
        found = check_steps(runner, seqs, 4, 5, free, spare)
        for s, beams in zip(seqs, found):
            tokens = beams[0][0]
            prompt = list(s.token_ids)
            other = torch.randint(0, 2048, (16,), generator=torch.Generator().manual_seed(7)).tolist() + prompt[16:]
            moved = (log_probs(runner, [other + tokens], spare) - log_probs(runner, [prompt + tokens], spare)).abs()
            assert moved.max().item() > 4 * STEP, "the model does not see what it should"
    finally:
        runner.exit()
