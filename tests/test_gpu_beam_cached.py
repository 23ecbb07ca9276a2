"""ModelRunner.beam_search behind prompts that are partly in the cache, on one B200."""
import pytest

from tests.gpu_util import ensure_group
from tests.test_gpu_beam_search import STEP, sequences
from tests.test_gpu_model import _attention_backend

pytestmark = pytest.mark.gpu


def test_cached_prompts(pkg):
    """Prompts whose first tokens are in the cache already, in the blocks of 256 tokens that a prefill over the cache reads."""
    ensure_group()
    from nanovllm_b200.engine.model_runner import ModelConfig, ModelRunner
    _attention_backend()
    cfg = ModelConfig(hidden_size=1024, num_attention_heads=8, num_key_value_heads=4, head_dim=128, intermediate_size=2048, num_hidden_layers=3, vocab_size=2048, max_position_embeddings=2048)
    runner = ModelRunner(cfg, max_num_seqs=64, max_model_len=1024, max_num_batched_tokens=2048, num_kvcache_blocks=40, enforce_eager=True, oneshot_tokens=128, seed=3)
    try:
        seqs = sequences([300, 530], seed=12)
        for s, table in zip(seqs, ([0, 1], [2, 3, 4])):
            s.block_table = table
        want = runner.beam_search(seqs, 4, 5, list(range(5, 40)))
        for s in seqs:
            s.num_cached_tokens = 256
        got = runner.beam_search(seqs, 4, 5, list(range(5, 40)))
        for f, w in zip(got, want):
            assert abs(f[0][1] - w[0][1]) <= 2 * STEP * 5
    finally:
        runner.exit()
