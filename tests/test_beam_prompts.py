"""Which prompts ModelRunner.beam_search refuses, before anything reaches a GPU: a block that a search writes to (a prompt's last one, where it has room left) belongs to one place of one prompt."""
import pytest
import torch


@pytest.fixture
def search(pkg):
    from nanovllm_b200.engine.model_runner import ModelConfig, ModelRunner, Seq

    class Reached(Exception):
        pass

    def to_device(*arrays):
        raise Reached  # (the first thing after the checks)

    r = ModelRunner.__new__(ModelRunner)
    r.rank, r.world, r.device, r.block_size, r.num_kvcache_blocks = 0, 1, torch.device("cpu"), 16, 100
    r.max_num_seqs, r.max_model_len, r.max_num_batched_tokens = 64, 128, 256
    r._to_device = to_device
    r.config = ModelConfig(64, 1, 1, 64, 64, 1, 50)

    def call(*prompts, free=range(40, 100)):
        """(tokens, table) of each prompt: whether the search is on its way."""
        try:
            r.beam_search([Seq([1] * n, list(table)) for n, table in prompts], 3, 5, list(free))
        except Reached:
            return True
        raise AssertionError("neither an error nor a search")

    return call


@pytest.mark.parametrize("prompts", [
    [(20, [0, 1]), (40, [0, 1, 2])],      # open for the first, full for the second
    [(40, [0, 1, 2]), (20, [0, 1])],
    [(20, [0, 1]), (20, [0, 1])],         # open for both
    [(20, [5, 5])],                       # full and open in one table
    [(40, [3, 4, 3])],
    [(7, [0]), (7, [1]), (33, [2, 1, 6])],
    [(9, [4]), (32, [3, 4])],
])
def test_open_blocks_that_are_not_alone(search, prompts):
    with pytest.raises(ValueError, match="share full blocks only"):
        search(*prompts)


@pytest.mark.parametrize("prompts", [
    [(20, [0, 1]), (40, [0, 2, 3])],      # a full block of both
    [(32, [0, 1]), (32, [0, 1])],         # all of them full
    [(32, [0, 1]), (40, [0, 1, 2])],
    [(20, [0, 1, 7]), (7, [7])],          # (behind a prompt's tokens its table may hold anything)
    [(20, [0, 1, 1]), (16, [9, 9])],
    [(1, [0])],
])
def test_prompts_that_fit(search, prompts):
    assert search(*prompts)
